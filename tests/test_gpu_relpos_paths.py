"""GPU: attention with a relative position bias (csrc/relpos.hip) -- what its launches hand to one another, and what offsets that do not rise leave
alone."""
import numpy as np
import pytest
import torch

from oracle import tower_ops as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def dev():
    if not torch.cuda.is_available():
        pytest.skip('needs a GPU')
    from creamfl_amd import _lib
    _lib.load()
    return torch.device('cuda:0')


def launched(fn):
    """What fn() gives, and the names of the framework's kernels that ran in it."""
    from creamfl_amd import _lib
    _lib.prof_reset()
    _lib.prof_enable(True)
    try:
        out = fn()
        torch.cuda.synchronize()
        return out, {n.replace('cfl_', '').replace('_kernel', '') for n, (k, _) in _lib.prof_query().items() if k}
    finally:
        _lib.prof_enable(False)


@pytest.mark.parametrize('B,L,heads', [(600, 40, 2), (3, 300, 4), (1100, 5, 1)])
def test_the_tables_shares_meet_in_a_launch_of_their_own(dev, B, L, heads):
    """Sums of many texts and distances are formed by many workgroups; what orders their stores before the last sum is the end of their launch."""
    from creamfl_amd import ops
    g = torch.Generator().manual_seed(B)
    H = heads * 64
    qkv, do = torch.randn(B, L, 3 * H, generator=g).to(torch.bfloat16), torch.randn(B, L, H, generator=g).to(torch.bfloat16)
    table, buckets = torch.randn(32, heads, generator=g), ops.relpos_buckets(32, 128)
    leaves = [qkv.to(dev).requires_grad_(True), table.to(dev).requires_grad_(True)]

    def run():
        return torch.autograd.grad(ops.relpos_attention(leaves[0], leaves[1], buckets.to(dev), heads), leaves, do.to(dev))[1]
    first, names = launched(run)
    assert {'relpos_dtable', 'relpos_dtable_join'} <= names, names
    for _ in range(20):
        assert torch.equal(run(), first)
    dt, et = torch.zeros(32, heads, dtype=torch.float64), torch.zeros(32, heads, dtype=torch.float64)
    for b in range(B):
        q, k, v = (t.reshape(L, heads, 64) for t in qkv[b].split(H, 1))
        w = ref.relpos_attention_text(q, k, v, table, buckets, None, 0.125, do[b].view(L, heads, 64))['dtable']
        dt, et = dt + w[0], et + w[1]
    off = (first.double().cpu() - dt).abs()
    assert bool((off <= et + 2.0 ** -24 * (dt.abs() + et) + 1e-30).all()), float((off / et).max())
