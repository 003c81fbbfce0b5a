"""The encoder towers' operators on the CPU: sizes that their kernels' counters do not hold are refused before anything is launched."""
import torch

EINVAL, EALIGN, ELIMIT = -1, -2, -3


def test_gn_entries_refuse_maps_beyond_their_row_counters():
    """A sample's positions are counted in 32 bits: 2^30 of them are taken, one more is refused, forward and backward."""
    from creamfl_amd import _lib
    lib = _lib.load()
    P, most = 4096, 1 << 30
    assert lib.cfl_gn_ws_bytes(1, most, 8, 1) > 0
    for hw in (most + 1, (1 << 31) - 1):
        assert lib.cfl_gn_ws_bytes(1, hw, 8, 1) == 0
        assert lib.cfl_gn_fwd(P, None, P, P, 1, 1, hw, 8, 1, 1e-5, 0, P, P, P, P, None) == ELIMIT
        assert lib.cfl_gn_bwd(P, None, P, None, P, P, P, P, 1, 1, hw, 8, 1, 0, 0, P, None, P, P, P, None) == ELIMIT


def test_gn_act_refuses_maps_beyond_its_row_counters():
    """[1, 8, 65536, 65537] bf16 fits the card's memory; its positions would reach the entry modulo 2^32 (as 65536)."""
    import pytest
    from torch._subclasses.fake_tensor import FakeTensorMode
    from creamfl_amd import _lib, ops
    with FakeTensorMode():
        def fmap(h, w):
            return torch.empty_strided((1, 8, h, w), (8 * h * w, 1, 8 * w, 8), dtype=torch.bfloat16, device='cuda')
        assert ops.gn_act_supported(fmap(1 << 15, 1 << 15), 8, 1)
        for h, w in ((1 << 15, (1 << 15) + 1), (46340, 46341), (65536, 65537), (1, (1 << 30) + 1)):
            x = fmap(h, w)
            assert not ops.gn_act_supported(x, 8, 1), (h, w)
            with pytest.raises(_lib.CreamflHipError, match='H W'):
                ops.gn_act(x, x, x, 1)


def test_gn_ways_are_all_tested():
    """Every way that csrc/gnorm.hip's rule can choose stands in the GPU tests' list, and the rule still sends the listed shapes there: the kinds, both
    types, both directions, groups of whole records and others, the two-pass kernels' three sizes of a workgroup -- and what the server's and the
    clients' trunks take at their batches."""
    import sys
    import os
    sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
    from test_gpu_gn_paths import PATHS, way
    seen = set()
    for shape, dtype, fwd, bwd in PATHS:
        assert way(shape, dtype, False) == fwd and way(shape, dtype, True) == bwd, (shape, dtype, way(shape, dtype, False), way(shape, dtype, True))
        seen |= {(dtype, 'fwd', fwd), (dtype, 'bwd', bwd)}

    def kinds(got):
        return {(d, way_, w[0] if w[0] != 'two' else w[:2], w[2:]) for d, way_, w in got}
    for d in ('bf16', 'fp32'):
        assert {(d, 'fwd', ('chunks',)), (d, 'bwd', ('chunks',))} <= seen
        for t in (256, 512, 1024):
            assert (d, 'bwd', ('two', t)) in seen and {(d, 'fwd', ('two', t, True)), (d, 'fwd', ('two', t, False))} <= seen, (d, t)
        for k in ('one', 'few'):
            assert any(x[:2] == (d, 'bwd') and x[2][0] == k for x in seen), (d, k)
            for whole in (False, True):
                assert any(x[:2] == (d, 'fwd') and x[2][0] == k and x[2][2] == whole for x in seen), (d, k, whole)
    trunk = [(64, 112), (64, 56), (256, 56), (128, 56), (128, 28), (512, 28), (256, 28), (256, 14), (1024, 14), (512, 14), (512, 7), (2048, 7)]
    client = [(64, 112), (64, 56), (128, 28), (256, 14), (512, 7)]
    for d, batches, maps in (('bf16', (128, 256), trunk), ('fp32', (128,), client)):
        for n in batches:
            for c, s in maps:
                got = {(d, 'fwd', way((n, c, s, s, 32), d, False)), (d, 'bwd', way((n, c, s, s, 32), d, True))}
                assert kinds(got) <= kinds(seen), (n, c, s, got)


def test_pack_plan_lists_the_real_tokens():
    """The packed run's indexes against their definition, token by token; lengths that do not fit give no plan."""
    import random
    from creamfl_amd.networks.backbones import BertModel
    r = random.Random(3)
    for B, L, longest in ((1, 1, 32), (7, 24, 32), (256, 32, 32), (33, 300, 1 << 30), (5, 700, 1 << 30)):
        lens = [r.randint(1, min(L, longest)) for _ in range(B)]
        plan = BertModel.pack_plan(lens, L, 'cpu', longest)
        pairs = [(b, t) for b, n in enumerate(lens) for t in range(n)]
        assert (plan.B, plan.L, plan.T) == (B, L, len(pairs))
        assert plan.tok_idx.dtype == torch.int64 and plan.tok_idx.tolist() == [b * L + t for b, t in pairs]
        assert plan.pos_ids.dtype == torch.int64 and plan.pos_ids.tolist() == [t for _, t in pairs]
        assert plan.cu.dtype == torch.int32 and plan.cu.tolist() == [sum(lens[:i]) for i in range(B + 1)]
        assert plan.cls_rows.dtype == torch.int64 and plan.cls_rows.tolist() == plan.cu.tolist()[:-1] and plan.cls_rows.is_contiguous()
    assert BertModel.pack_plan([3, 33], 40, 'cpu') is None and BertModel.pack_plan([3, 33], 40, 'cpu', 1 << 30) is not None
    assert BertModel.pack_plan([], 40, 'cpu') is None and BertModel.pack_plan([0, 3], 40, 'cpu') is None and BertModel.pack_plan([41], 40, 'cpu', 1 << 30) is None
