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


# A sentinel before and behind every buffer that the entries write, in elements
GUARD = 4096


class Guarded:
    """A buffer between two stretches of a known value."""
    def __init__(self, dev, n, dtype):
        self.whole = torch.full((n + 2 * GUARD,), 7, dtype=dtype, device=dev)
        self.n = n

    def ptr(self):
        return self.whole.data_ptr() + GUARD * self.whole.element_size()

    def untouched(self):
        return bool((self.whole[:GUARD] == 7).all()) and bool((self.whole[GUARD + self.n:] == 7).all())


@pytest.mark.parametrize('cu', [[0, 30, 7, 12, -5], [5, -3, 1 << 30, 2], [-2 ** 31, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31, 9, 9], [25, 25, 25], [19, 3, 20, 0, 1]], ids=str)
@pytest.mark.parametrize('T,longest,cls', [(20, 20, False), (20, 20, True), (70, 70, False), (700, 700, False), (700, 700, True)])
def test_offsets_of_any_kind_leave_everything_else_alone(dev, cu, T, longest, cls):
    """Offsets that fall or lie outside the rows: the kernels clip them to the rows there are, so that nothing beside the buffers is written, forward
    and backward, short and long texts, split or not.  (Which values overlapping texts give is undefined.)"""
    from creamfl_amd import _lib, ops
    lib = _lib.load()
    B, H = len(cu) - 1, 64
    g = torch.Generator(device=dev).manual_seed(T)
    off = torch.tensor(cu, dtype=torch.int32, device=dev)
    rows, lq = (B, 1) if cls else (T, 0)
    q, k, v = (torch.randn(n, H, device=dev, generator=g).to(torch.bfloat16) for n in (rows, T, T))
    do = torch.randn(rows, H, device=dev, generator=g).to(torch.bfloat16)
    table, buckets = torch.randn(32, 1, device=dev, generator=g), ops.relpos_buckets(32, 128, dev)
    o, lse, dsum = Guarded(dev, rows * H, torch.bfloat16), Guarded(dev, rows, torch.float32), Guarded(dev, rows, torch.float32)
    nf = lib.cfl_relpos_fwd_ws_bytes(B, lq, longest, T, 1)
    nb = lib.cfl_relpos_bwd_ws_bytes(B, lq, longest, T, 1, 32, 128)
    wf, wb = Guarded(dev, max(nf, 256), torch.uint8), Guarded(dev, nb, torch.uint8)
    dq, dk, dv, dt = Guarded(dev, rows * H, torch.bfloat16), Guarded(dev, T * H, torch.bfloat16), Guarded(dev, T * H, torch.bfloat16), Guarded(dev, 32, torch.float32)
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(lib.cfl_relpos_fwd(q.data_ptr(), H, k.data_ptr(), v.data_ptr(), H, None, off.data_ptr(), B, lq, longest, T, 1, 64, 0.125, table.data_ptr(), 0, 32,
                                  buckets.data_ptr(), 128, o.ptr(), H, lse.ptr(), wf.ptr(), stream), 'fwd')
    _lib.check(lib.cfl_relpos_bwd(q.data_ptr(), H, k.data_ptr(), v.data_ptr(), H, None, off.data_ptr(), B, lq, longest, T, 1, 64, 0.125, table.data_ptr(), 0, 32,
                                  buckets.data_ptr(), 128, o.ptr(), do.data_ptr(), H, lse.ptr(), dsum.ptr(), dq.ptr(), H, dk.ptr(), dv.ptr(), H, dt.ptr(),
                                  wb.ptr(), stream), 'bwd')
    torch.cuda.synchronize()
    for name, t in dict(o=o, lse=lse, dsum=dsum, wf=wf, wb=wb, dq=dq, dk=dk, dv=dv, dt=dt).items():
        assert t.untouched(), name


@pytest.mark.parametrize('B,L,heads,form', [(5, 1, 2, 'padded'), (3, 17, 4, 'padded'), (9, 32, 12, 'padded'), (7, 31, 3, 'packed'), (4, 32, 2, 'cls'), (3, 513, 3, 'cls'),
                                            (2, 2100, 1, 'cls'), (300, 200, 12, 'cls')])
def test_few_queries_are_off_by_the_outputs_rounding_alone(dev, B, L, heads, form):
    """p enters its product with v in two bf16 terms where a text has at most 32 queries: what they leave is 2^-16 of it."""
    from creamfl_amd import ops
    g = torch.Generator().manual_seed(B * 100 + L)
    H = heads * 64
    qkv = torch.randn(B, L, 3 * H, generator=g).to(torch.bfloat16)
    table, buckets = torch.randn(32, heads, generator=g), ops.relpos_buckets(32, 128)
    keep = torch.rand(B, L, generator=g) < 0.8
    if form == 'packed':
        cu = torch.arange(0, (B + 1) * L, L, dtype=torch.int32, device=dev)
        o = ops.relpos_attention_varlen(qkv.view(B * L, 3 * H).to(dev), cu, L, table.to(dev), buckets.to(dev), heads).view(B, L, H)
    elif form == 'cls':
        o = ops.relpos_attention_cls(qkv[:, 0, :H].contiguous().to(dev), qkv[:, :, H:].contiguous().to(dev), table.to(dev), buckets.to(dev), heads,
                                     key_mask=keep.to(dev)).view(B, 1, H)
    else:
        o = ops.relpos_attention(qkv.to(dev), table.to(dev), buckets.to(dev), heads, key_mask=keep.to(dev))
    for b in range(min(B, 9)):
        q, k, v = (t.reshape(L, heads, 64) for t in qkv[b].split(H, 1))
        value, bound = ref.relpos_attention_text(q[:o.shape[1]], k, v, table, buckets, None if form == 'packed' else keep[b], 0.125, terms=2)['o']
        off = (o[b].double().cpu().view(-1, heads, 64) - value).abs()
        assert bool((off <= bound).all()), (b, float((off / bound).max()))


@pytest.mark.parametrize('lq,lk', [(40, 100), (100, 40), (5, 300), (300, 5), (33, 32), (32, 33), (20, 7), (1000, 64), (64, 1000), (1500, 33), (3, 1300)])
@pytest.mark.parametrize('packed', [False, True], ids=['padded', 'packed'])
def test_queries_and_keys_of_different_lengths(dev, lq, lk, packed):
    """The entries' own form: Lq query rows a text against other numbers of keys, both counted from position 0; padded with a mask, or packed keys with an
    empty text among them and rows behind the last one."""
    from creamfl_amd import _lib, ops
    lib = _lib.load()
    B, heads = 3, 2
    H = heads * 64
    g = torch.Generator().manual_seed(lq * 7 + lk)
    lens = [lk, 0, max(lk - 3, 1)] if packed else [lk] * 3
    T = sum(lens) + 2 if packed else 0
    keep = torch.rand(B, lk, generator=g) < 0.7
    keep[:, 0] = True
    rows = T if packed else B * lk
    q, k, v = (torch.randn(n, H, generator=g).to(torch.bfloat16) for n in (B * lq, rows, rows))
    do = torch.randn(B * lq, H, generator=g).to(torch.bfloat16)
    table, buckets = torch.randn(32, heads, generator=g), ops.relpos_buckets(32, 128)
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32)
    dq_, dk_, dv_, do_, dt_, db_ = (t.to(dev) for t in (q, k, v, do, table, buckets))
    dm, dc = keep.to(torch.uint8).to(dev), cu.to(dev)
    mask, off = (None, dc.data_ptr()) if packed else (dm.data_ptr(), None)
    o = torch.full((B * lq, H), 7, dtype=torch.bfloat16, device=dev)
    lse, dsum = torch.empty(heads, B * lq, device=dev), torch.empty(heads, B * lq, device=dev)
    gq, gk, gv, gt = torch.full_like(o, 7), torch.full_like(dk_, 7), torch.full_like(dk_, 7), torch.full_like(dt_, 7)
    wf = torch.empty(max(lib.cfl_relpos_fwd_ws_bytes(B, lq, lk, T, heads), 256), dtype=torch.uint8, device=dev)
    wb = torch.empty(lib.cfl_relpos_bwd_ws_bytes(B, lq, lk, T, heads, 32, 128), dtype=torch.uint8, device=dev)
    s = torch.cuda.current_stream().cuda_stream
    _lib.check(lib.cfl_relpos_fwd(dq_.data_ptr(), H, dk_.data_ptr(), dv_.data_ptr(), H, mask, off, B, lq, lk, T, heads, 64, 0.125, dt_.data_ptr(), 0, 32,
                                  db_.data_ptr(), 128, o.data_ptr(), H, lse.data_ptr(), wf.data_ptr(), s), 'fwd')
    _lib.check(lib.cfl_relpos_bwd(dq_.data_ptr(), H, dk_.data_ptr(), dv_.data_ptr(), H, mask, off, B, lq, lk, T, heads, 64, 0.125, dt_.data_ptr(), 0, 32,
                                  db_.data_ptr(), 128, o.data_ptr(), do_.data_ptr(), H, lse.data_ptr(), dsum.data_ptr(), gq.data_ptr(), H, gk.data_ptr(),
                                  gv.data_ptr(), H, gt.data_ptr(), wb.data_ptr(), s), 'bwd')
    torch.cuda.synchronize()

    def ok(got, want, name):
        value, bound = want
        off_ = (got.double().cpu().view(value.shape) - value).abs()
        assert bool((off_ <= bound).all()), (name, float((off_ / bound).nan_to_num(nan=np.inf).max()))
    dt, et = torch.zeros(32, heads, dtype=torch.float64), torch.zeros(32, heads, dtype=torch.float64)
    for b in range(B):
        a, n = (int(cu[b]), lens[b]) if packed else (b * lk, lk)
        qs = slice(b * lq, (b + 1) * lq)
        if n == 0:
            assert not o[qs].any() and not gq[qs].any()
            continue
        w = ref.relpos_attention_text(q[qs].view(lq, heads, 64), k[a:a + n].view(n, heads, 64), v[a:a + n].view(n, heads, 64), table, buckets,
                                      None if packed else keep[b], 0.125, do[qs].view(lq, heads, 64))
        for t, name in ((o[qs], 'o'), (gq[qs], 'dq'), (gk[a:a + n], 'dk'), (gv[a:a + n], 'dv')):
            ok(t, w[name], '%s of text %d' % (name, b))
        dt, et = dt + w['dtable'][0], et + w['dtable'][1]
    ok(gt, (dt, et + 2.0 ** -24 * (dt.abs() + et) + 1e-30), 'dtable')
    if packed:
        assert not gk[T - 2:].any() and not gv[T - 2:].any()


@pytest.mark.parametrize('L,B,heads', [(20, 3, 2), (32, 2, 2), (70, 2, 2), (300, 2, 2), (1000, 1, 1), (1300, 1, 1), (600, 8, 12)])
@pytest.mark.parametrize('kind', ['x30', 'x1000', 'rising', 'falling'])
def test_sharp_scores(dev, L, B, heads, kind):
    """Scores up to 10^8: rows that one key takes whole; maxima that rise with every tile, or stand in the first one."""
    from creamfl_amd import ops
    g = torch.Generator().manual_seed(L + B)
    H = heads * 64
    x = torch.randn(B, L, 3 * H, generator=g)
    if kind[0] == 'x':
        x[:, :, :2 * H] *= float(kind[1:])
    else:
        x[:, :, :H] = x[:, :, :H].abs() * 4
        x[:, :, H:2 * H] = torch.linspace(-20, 20, L)[None, :, None] * (1 if kind == 'rising' else -1) + 0.1 * x[:, :, H:2 * H]
    qkv, do = x.to(torch.bfloat16), torch.randn(B, L, H, generator=g).to(torch.bfloat16)
    table, buckets = torch.randn(32, heads, generator=g), ops.relpos_buckets(32, 128)
    leaves = [qkv.to(dev).requires_grad_(True), table.to(dev).requires_grad_(True)]
    o = ops.relpos_attention(leaves[0], leaves[1], buckets.to(dev), heads)
    dqkv, dtable = torch.autograd.grad(o, leaves, do.to(dev))
    dt, et = torch.zeros(32, heads, dtype=torch.float64), torch.zeros(32, heads, dtype=torch.float64)
    for b in range(B):
        q, k, v = (t.reshape(L, heads, 64) for t in qkv[b].split(H, 1))
        w = ref.relpos_attention_text(q, k, v, table, buckets, None, 0.125, do[b].view(L, heads, 64))
        for t, name in ((o[b], 'o'), *zip(dqkv[b].split(H, 1), ('dq', 'dk', 'dv'))):
            off = (t.double().cpu().reshape(L, heads, 64) - w[name][0]).abs()
            assert bool((off <= w[name][1]).all()), (b, name, float((off / w[name][1]).nan_to_num(nan=np.inf).max()))
        dt, et = dt + w['dtable'][0], et + w['dtable'][1]
    # (a block's sums over diagonals hold to 2^-24 of the largest of them, over at most 2 x 16 additions and the difference of two)
    off, bound = (dtable.double().cpu() - dt).abs(), et + 64 * 2.0 ** -24 * (et.max(0).values + dt.abs().max(0).values) + 1e-30
    assert bool((off <= bound).all()), float((off / bound).max())
