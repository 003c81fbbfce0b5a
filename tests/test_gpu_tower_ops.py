"""GPU: the encoder towers' operators (csrc/gnorm.hip, dropout.hip, relpos.hip) against their 64-bit restatement (oracle/tower_ops.py),
within bounds that count the kernels' roundings."""
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


def within(got, want, name):
    value, bound = want
    off = (got.detach().double().cpu() - value).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), '%s: %d of %d outside, worst %.3g of its bound at %s' % (
        name, int(bad.sum()), bad.numel(), float((off / bound).nan_to_num(nan=np.inf).max()), tuple(bad.nonzero()[0].tolist()))


def cl(t):
    return t.contiguous(memory_format=torch.channels_last)


# ------------------------------------------------------------------------------------------------ group norm
GN_SHAPES = [  # n, c, h, w, groups
    (1, 8, 1, 1, 8), (1, 8, 1, 1, 1), (3, 8, 1, 2, 4), (2, 16, 7, 7, 2), (1, 24, 5, 3, 3), (2, 40, 9, 11, 8), (5, 64, 13, 17, 32), (2, 320, 8, 8, 32),
    (3, 72, 30, 31, 9), (2, 512, 7, 7, 32), (1, 2048, 7, 7, 32), (2, 2048, 2, 3, 2048), (1, 1000, 4, 4, 5), (2, 64, 56, 56, 32), (1, 64, 112, 111, 16),
    (130, 8, 3, 3, 2), (2, 256, 28, 28, 1), (1, 1608, 12, 12, 67),
    (2, 512, 95, 97, 32), (1, 1000, 41, 40, 5), (1, 2048, 24, 23, 2048), (3, 64, 57, 94, 1), (1, 2048, 9, 11, 1)]             # (more than 64 chunks of rows, a ragged last one)


@pytest.mark.parametrize('shape', GN_SHAPES, ids=str)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
@pytest.mark.parametrize('act,res', [('none', False), ('relu', True), ('silu', False), ('silu', True)])
def test_gn_act_matches_oracle(dev, shape, dtype, act, res):
    from creamfl_amd import ops
    n, c, h, w, groups = shape
    g = torch.Generator().manual_seed(n * 7919 + c * 31 + h)
    x, r, dy = (cl(torch.randn(n, c, h, w, generator=g).to(dtype)) for _ in range(3))
    x = cl((x.float() * 1.5 + 0.5).to(dtype))
    ga, be = 1 + 0.3 * torch.randn(c, generator=g), 0.3 * torch.randn(c, generator=g)
    leaves = [t.to(dev).requires_grad_(True) for t in (x, ga, be)] + ([cl(r.to(dev)).requires_grad_(True)] if res else [])
    assert ops.gn_act_supported(leaves[0], c, groups)
    y = ops.gn_act(leaves[0], leaves[1], leaves[2], groups, act=act, residual=leaves[3] if res else None)
    assert y.dtype == dtype and y.is_contiguous(memory_format=torch.channels_last)
    grads = torch.autograd.grad(y, leaves, cl(dy.to(dev)))
    want = ref.group_norm_act(x, ga, be, groups, act=act, residual=r if res else None, dy=dy, bf16=dtype == torch.bfloat16)
    within(y, want['y'], 'y')
    for name, t in zip(('dx', 'dgamma', 'dbeta', 'dres'), grads):
        within(t, want[name], name)
    with torch.no_grad():                                  # the forward alone: the same bits
        y2 = ops.gn_act(leaves[0], leaves[1], leaves[2], groups, act=act, residual=leaves[3] if res else None)
    assert torch.equal(y, y2)


def test_gn_act_large_mean_costs_no_digits(dev):
    """A mean of 300 deviations: sums of squares would lose the variance's digits; here xh keeps the precision of x - mu."""
    from creamfl_amd import ops
    g = torch.Generator().manual_seed(1)
    x = cl(300 + torch.randn(2, 32, 40, 40, generator=g))
    ga, be = torch.ones(32), torch.zeros(32)
    y = ops.gn_act(x.to(dev), ga.to(dev), be.to(dev), 8)
    within(y, ref.group_norm_act(x, ga, be, 8)['y'], 'y')
    x[0, :, 0, 0] = 3e4                                    # and a corner far from everything else
    y = ops.gn_act(x.to(dev), ga.to(dev), be.to(dev), 8)
    within(y, ref.group_norm_act(x, ga, be, 8)['y'], 'y')


def test_gn_act_two_gradients_and_expanded_gradient(dev):
    from creamfl_amd import ops
    g = torch.Generator().manual_seed(2)
    x, r, d1, d2 = (cl(torch.randn(3, 16, 6, 5, generator=g)) for _ in range(4))
    ga, be = 1 + 0.1 * torch.randn(16, generator=g), torch.zeros(16)
    for act in ('relu', 'none'):
        xs, rs = x.to(dev).requires_grad_(True), r.to(dev).requires_grad_(True)
        a, b = ops.gn_act(xs, ga.to(dev), be.to(dev), 4, act=act, residual=rs, two=True)
        assert a.data_ptr() == b.data_ptr()
        ((a * d1.to(dev)).sum() + (b * d2.to(dev)).sum()).backward()
        want = ref.group_norm_act(x, ga, be, 4, act=act, residual=r, dy=d1.double() + d2.double())
        within(xs.grad, want['dx'], 'dx')
        within(rs.grad, want['dres'], 'dres')
        xs.grad = rs.grad = None
        _, b = ops.gn_act(xs, ga.to(dev), be.to(dev), 4, act=act, residual=rs, two=True)
        b.sum().backward()                                 # one alias unused; the gradient is an expanded scalar
        want = ref.group_norm_act(x, ga, be, 4, act=act, residual=r, dy=torch.ones_like(x))
        within(xs.grad, want['dx'], 'dx')
        within(rs.grad, want['dres'], 'dres')


def test_gn_act_views_and_refusals(dev):
    from creamfl_amd import _lib, ops
    g = torch.Generator().manual_seed(5)
    ga, be = torch.ones(16), torch.zeros(16)
    big = torch.randn(3 * 5 * 4 * 16 + 1, generator=g).to(dev)
    x = big[1:].view(3, 5, 4, 16).permute(0, 3, 1, 2)      # channels last, first element off the 16-byte border
    y = ops.gn_act(x, ga.to(dev), be.to(dev), 4, act='silu')
    within(y, ref.group_norm_act(x, ga, be, 4, act='silu')['y'], 'y')
    res = torch.randn(3, 16, 5, 4, generator=g).to(dev)    # NCHW, another type: brought into x's
    y = ops.gn_act(x, ga.to(dev), be.to(dev), 4, residual=res.double())
    within(y, ref.group_norm_act(x, ga, be, 4, residual=res)['y'], 'y')
    nan = x.clone(memory_format=torch.channels_last)
    nan[1, 3, 2, 2] = float('nan')                         # a group's NaN stays in its group
    y = ops.gn_act(nan, ga.to(dev), be.to(dev), 4, act='relu')
    assert bool(torch.isnan(y[1, :4]).all()) and int(torch.isnan(y).sum()) == 4 * 20
    ok = dict(x=x, weight=ga.to(dev), bias=be.to(dev), groups=4)
    for kw in (dict(x=x.contiguous()), dict(groups=3), dict(groups=0), dict(act='gelu'), dict(weight=ga[:8].to(dev)), dict(bias=be), dict(eps=-1.0),
               dict(residual=res[:2]), dict(x=x.half()), dict(x=x[0])):
        with pytest.raises(_lib.CreamflHipError):
            ops.gn_act(**{**ok, **kw})


# ------------------------------------------------------------------------------------------------ dropout
@pytest.fixture(autouse=True)
def tick_at_zero():
    """The oracle's flags are those of the seed alone: a tick that captured steps of the same process have moved on stands at 0 meanwhile."""
    from creamfl_amd import ops
    t = ops._DROPOUT_TICK[0]
    was = None if t is None else t.clone()
    if t is not None:
        t.zero_()
    yield
    if t is not None:
        t.copy_(was)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['fp32', 'bf16', 'fp16'])
@pytest.mark.parametrize('shape', [(1,), (2,), (7,), (8,), (1023,), (3, 5, 7), (33, 256), (257, 1001), (1 << 20,), (4099, 768)], ids=str)
@pytest.mark.parametrize('p', [0.1, 0.5, 1.0])
def test_dropout_matches_oracle(dev, dtype, shape, p):
    from creamfl_amd import ops
    g = torch.Generator().manual_seed(len(shape) + shape[0])
    x, dy = (torch.randn(*shape, generator=g).to(dtype) for _ in range(2))
    xs = x.to(dev).requires_grad_(True)
    y = ops.dropout(xs, p, seed=0xDEADBEEF)
    dx, = torch.autograd.grad(y, [xs], dy.to(dev))
    keep = ref.keep_flags(0xDEADBEEF, p, x.numel()).view(shape)
    thr = round(65536 * p)
    f = 65536 / (65536 - thr) if thr < 65536 else 0.0
    half = torch.finfo(dtype).eps / 2
    # (below the smallest normal number m the steps no longer shrink: they are eps m wide, so a rounding there is off by up to eps m / 2
    # whatever the value -- in fp16 2^-10 2^-14 / 2 = 2^-25, which values of this size reach; it is nothing in fp32 and bf16)
    floor = half * torch.finfo(dtype).smallest_normal
    for got, t in ((y, x), (dx, dy)):
        want = torch.where(keep, t.double() * f, torch.zeros_like(t, dtype=torch.float64))
        within(got, (want, want.abs() * (half + 2.0 ** -23) + floor), 'value')      # (the factor's rounding, the product's, the output's)
    if x.numel() % 4 == 0 and p < 1:
        assert torch.equal(ops.dropout_keep_mask(0xDEADBEEF, p, shape, dev).cpu(), keep)


def test_dropout_manner(dev):
    from creamfl_amd import _lib, ops
    x = torch.randn(64, 33, device=dev)
    assert ops.dropout(x, 0.0) is x
    assert ops.dropout(x[:0], 0.3).shape == (0, 33)
    assert torch.equal(ops.dropout(x.t(), 0.3, seed=5), ops.dropout(x.t().contiguous(), 0.3, seed=5))
    odd = torch.randn(1001, device=dev, dtype=torch.bfloat16)
    assert torch.equal(ops.dropout(odd[1:], 0.3, seed=5), ops.dropout(odd[1:].clone(), 0.3, seed=5))     # any alignment
    bad = torch.full((4096,), float('nan'), device=dev)
    y = ops.dropout(bad, 0.5, seed=9)
    assert bool((y[~ref.keep_flags(9, 0.5, 4096).to(dev)] == 0).all())                                    # a dropped NaN is gone
    torch.manual_seed(11)
    a = ops.dropout(x, 0.5)
    b = ops.dropout(x, 0.5)
    assert not torch.equal(a, b)                           # each call draws the next seed
    for kw in (dict(p=-0.1), dict(p=1.1), dict(p=float('nan')), dict(x=x.double()), dict(x=x.cpu())):
        with pytest.raises(_lib.CreamflHipError):
            ops.dropout(**{**dict(x=x, p=0.5), **kw})


def test_dropout_refuses_a_tick_of_another_device(dev, monkeypatch):
    from creamfl_amd import _lib, ops
    monkeypatch.setattr(ops, '_DROPOUT_TICK', [torch.zeros(1, dtype=torch.int32)])
    with pytest.raises(_lib.CreamflHipError, match='tick'):
        ops.dropout(torch.ones(4, device=dev), 0.5)


def test_dropout_backward_uses_the_forwards_tick(dev):
    """The tick moves on between forward and backward: the gradient still follows the mask that the forward drew."""
    from creamfl_amd import ops
    x = torch.randn(512, 40, device=dev, requires_grad=True)
    tick = ops.dropout_tick(dev)
    before = int(tick)
    try:
        tick.add_(3)
        y = ops.dropout(x, 0.4, seed=77)
        tick.add_(1)
        dx, = torch.autograd.grad(y, [x], torch.ones_like(y))
        assert torch.equal(dx != 0, y != 0)
        z = ops.dropout(x, 0.4, seed=77)
        assert not torch.equal(z != 0, y != 0)
    finally:
        tick.fill_(before)


# ------------------------------------------------------------------------------------------------ attention
def attn_inputs(seed, B, L, heads, nb=32, far=128, dtype=torch.bfloat16, lq=None):
    from creamfl_amd import ops
    g = torch.Generator().manual_seed(seed)
    H = heads * 64
    t = dict(qkv=torch.randn(B, L, 3 * H, generator=g).to(torch.bfloat16), do=torch.randn(B, L, H, generator=g).to(torch.bfloat16),
             table=torch.randn(nb, heads, generator=g).to(dtype), buckets=ops.relpos_buckets(nb, far))
    return t


def text_oracle(qkv, table, buckets, keep, do, scale=0.125):
    L, H3 = qkv.shape
    q, k, v = (t.reshape(L, -1, 64) for t in qkv.split(H3 // 3, 1))
    return ref.relpos_attention_text(q, k, v, table, buckets, keep, scale, do.view(L, -1, 64))


def check_padded(dev, t, mask, scale=None, heads=None):
    from creamfl_amd import ops
    B, L, H3 = t['qkv'].shape
    H, heads = H3 // 3, H3 // 192
    qkv, table = t['qkv'].to(dev).requires_grad_(True), t['table'].to(dev).requires_grad_(True)
    o = ops.relpos_attention(qkv, table, t['buckets'].to(dev), heads, key_mask=None if mask is None else mask.to(dev), scale=scale)
    dqkv, dtable = torch.autograd.grad(o, [qkv, table], t['do'].to(dev))
    dt, et = torch.zeros(t['table'].shape, dtype=torch.float64), torch.zeros(t['table'].shape, dtype=torch.float64)
    for b in range(B):
        w = text_oracle(t['qkv'][b], t['table'], t['buckets'], None if mask is None else mask[b], t['do'][b], 0.125 if scale is None else scale)
        within(o[b].view(L, heads, 64), w['o'], 'o of text %d' % b)
        for i, name in enumerate(('dq', 'dk', 'dv')):
            within(dqkv[b, :, i * H:(i + 1) * H].reshape(L, heads, 64), w[name], '%s of text %d' % (name, b))
        dt, et = dt + w['dtable'][0], et + w['dtable'][1]
    within(dtable, (dt, et + (torch.finfo(t['table'].dtype).eps / 2) * (dt.abs() + et) + 1e-30), 'dtable')
    with torch.no_grad():
        o2 = ops.relpos_attention(qkv, table, t['buckets'].to(dev), heads, key_mask=None if mask is None else mask.to(dev), scale=scale)
    assert torch.equal(o, o2)
    again = torch.autograd.grad(ops.relpos_attention(qkv, table, t['buckets'].to(dev), heads, key_mask=None if mask is None else mask.to(dev),
                                                     scale=scale), [qkv, table], t['do'].to(dev))
    assert torch.equal(again[0], dqkv) and torch.equal(again[1], dtable)       # the same bits on every run


@pytest.mark.parametrize('B,L,heads', [(1, 1, 1), (3, 2, 2), (2, 17, 3), (2, 31, 4), (3, 32, 12), (2, 33, 2), (2, 63, 1), (2, 64, 2), (1, 65, 3), (2, 96, 2),
                                       (1, 127, 1), (2, 128, 2), (2, 129, 2), (2, 197, 3), (1, 300, 2), (1, 513, 1), (9, 24, 12), (1, 1025, 1), (40, 160, 8), (1100, 3, 1), (260, 70, 1)])
def test_relpos_attention_matches_oracle(dev, B, L, heads):
    check_padded(dev, attn_inputs(B * 1000 + L, B, L, heads), None)


@pytest.mark.parametrize('B,L,heads,kind', [(4, 24, 2, 'prefix'), (5, 100, 2, 'prefix'), (3, 40, 3, 'holes'), (3, 197, 2, 'holes'), (2, 260, 1, 'tile'),
                                            (3, 9, 1, 'empty'), (3, 150, 2, 'empty')])
@pytest.mark.parametrize('poison', [False, True], ids=['', 'poison'])
def test_relpos_attention_masks(dev, B, L, heads, kind, poison):
    """Prefix lengths, scattered holes, whole dropped tiles, texts without a key; NaN and infinities in the k and v of dropped keys."""
    t = attn_inputs(B * 77 + L, B, L, heads)
    g = torch.Generator().manual_seed(L)
    mask = torch.ones(B, L, dtype=torch.bool)
    if kind == 'prefix':
        mask = torch.arange(L)[None] < torch.randint(1, L + 1, (B, 1), generator=g)
    elif kind == 'holes':
        mask = torch.rand(B, L, generator=g) < 0.6
    elif kind == 'tile':
        mask[:, 64:192] = False
        mask[1, :64] = False
    else:
        mask[1] = False
        mask[2, 1:] = False
    if poison:
        bad = torch.tensor([float('nan'), float('inf'), -float('inf')])
        H = heads * 64
        t['qkv'][:, :, H:] = torch.where(mask[:, :, None], t['qkv'][:, :, H:], bad[torch.arange(2 * H) % 3].to(torch.bfloat16))
    check_padded(dev, t, mask)


@pytest.mark.parametrize('nb,far,dtype', [(4, 2, torch.float32), (32, 128, torch.float32), (64, 512, torch.bfloat16), (8, 20, torch.float16)])
def test_relpos_attention_tables(dev, nb, far, dtype):
    check_padded(dev, attn_inputs(nb + far, 2, 170, 2, nb, far, dtype), None)


@pytest.mark.parametrize('B,L,heads,cut', [(3, 1, 2, False), (64, 1, 12, False), (3, 9, 2, True), (2, 32, 1, True)])
def test_relpos_attention_of_one_key_has_no_score_gradient(dev, B, L, heads, cut):
    """p = 1 in a row of one key: the gradients of q, k and the table are zero to the bit, in every kernel for short texts."""
    from creamfl_amd import ops
    t = attn_inputs(B * 31 + L, B, L, heads)
    qkv, table = t['qkv'].to(dev).requires_grad_(True), t['table'].to(dev).requires_grad_(True)
    mask = None
    if cut:
        mask = torch.zeros(B, L, dtype=torch.bool, device=dev)
        mask[torch.arange(B), torch.arange(B) * 5 % L] = True
    o = ops.relpos_attention(qkv, table, t['buckets'].to(dev), heads, key_mask=mask)
    dqkv, dtable = torch.autograd.grad(o, [qkv, table], t['do'].to(dev))
    H = heads * 64
    assert not dqkv[:, :, :2 * H].any() and not dtable.any()
    check_padded(dev, t, None if mask is None else mask.cpu())


@pytest.mark.parametrize('B,L,heads', [(3, 20, 2), (2, 33, 2), (2, 200, 3), (1, 900, 1), (40, 300, 8)])
@pytest.mark.parametrize('low', [-float('inf'), torch.finfo(torch.float32).min, -1e30])
def test_relpos_attention_bias_that_drops_keys(dev, B, L, heads, low):
    """A window by the bias: far buckets at -inf or the type's lowest value, so that a query's first tiles leave it nothing; scores far below zero in
    what is left (2^-s would underflow if the waiting rows' maximum stayed at zero); one head without any key; NaN gradients in a text that the mask
    empties."""
    t = attn_inputs(B * 3 + L, B, L, heads, 32, 16)
    t['table'] = t['table'] - 300.0
    far = t['buckets'][[0, -1]].long()
    t['table'][far] = low
    t['table'][t['buckets'][t['buckets'].numel() // 2 + 9].long()] = low
    if heads > 1:
        t['table'][:, 1] = low
    mask = torch.ones(B, L, dtype=torch.bool)
    mask[:, 4:7] = False
    if B > 1:
        mask[1] = False
    check_padded(dev, t, mask)


def test_relpos_attention_nan_gradient_of_a_text_without_keys(dev):
    from creamfl_amd import ops
    for L in (20, 70):
        t = attn_inputs(L, 2, L, 2)
        mask = torch.ones(2, L, dtype=torch.bool, device=dev)
        mask[0] = False
        qkv, table = t['qkv'].to(dev).requires_grad_(True), t['table'].to(dev).requires_grad_(True)
        do = t['do'].to(dev)
        want = torch.autograd.grad(ops.relpos_attention(qkv, table, t['buckets'].to(dev), 2, key_mask=mask), [qkv, table], do)
        do[0] = float('nan')
        got = torch.autograd.grad(ops.relpos_attention(qkv, table, t['buckets'].to(dev), 2, key_mask=mask), [qkv, table], do)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and not got[0][0].any()


def test_relpos_attention_scale_and_maps(dev):
    t = attn_inputs(5, 2, 70, 2, 32, 128)
    t['table'] = t['table'] * 8                            # (a strong bias: far distances win)
    check_padded(dev, t, None, scale=0.5)
    t['buckets'] = torch.zeros(1, dtype=torch.int32)       # R = 0: one bucket for every distance, the bias cancels
    check_padded(dev, t, None, scale=0.03)
    check_padded(dev, t, None, scale=-0.2)
    t['buckets'] = torch.randint(-3, 40, (41,), generator=torch.Generator().manual_seed(1)).to(torch.int32)    # any map; ends are clipped
    check_padded(dev, t, None)


@pytest.mark.parametrize('lens,max_len,tail', [([1], 1, 0), ([5, 0, 32, 1, 17], 32, 0), ([5, 0, 32, 1, 17], 32, 3), ([40, 0, 7, 129, 64], 129, 0),
                                               ([0, 70, 0], 70, 9), ([300, 20], 20, 0), ([33, 90, 128], 17, 1), ([9, 40, 3], 32, 2),
                                               ([700, 0, 1300], 1300, 5), ([700, 0, 1300], 900, 5)])
@pytest.mark.parametrize('lead', [0, 4])
def test_relpos_attention_varlen(dev, lens, max_len, tail, lead):
    """Packed texts, empty ones among them, rows before the first and behind the last one, texts longer than max_len (cut)."""
    from creamfl_amd import ops
    heads, H = 2, 128
    T = lead + sum(lens) + tail
    t = attn_inputs(T, 1, T, heads)
    cu = torch.tensor([lead] + [lead + int(v) for v in np.cumsum(lens)], dtype=torch.int32)
    qkv, table = t['qkv'][0].to(dev).requires_grad_(True), t['table'].to(dev).requires_grad_(True)
    idle = torch.ones(T, dtype=torch.bool)
    for b, n in enumerate(lens):
        idle[int(cu[b]):int(cu[b]) + min(n, max_len)] = False
    with torch.no_grad():
        qkv[idle.to(dev)] = float('nan')
    o = ops.relpos_attention_varlen(qkv, cu.to(dev), max_len, table, t['buckets'].to(dev), heads)
    dqkv, dtable = torch.autograd.grad(o, [qkv, table], t['do'][0].to(dev))
    dt, et = torch.zeros(32, heads, dtype=torch.float64), torch.zeros(32, heads, dtype=torch.float64)
    for b, n in enumerate(lens):
        n = min(n, max_len)
        if n == 0:
            continue
        at = slice(int(cu[b]), int(cu[b]) + n)
        w = text_oracle(t['qkv'][0, at], t['table'], t['buckets'], None, t['do'][0, at])
        within(o[at].view(n, heads, 64), w['o'], 'o')
        for i, name in enumerate(('dq', 'dk', 'dv')):
            within(dqkv[at, i * H:(i + 1) * H].reshape(n, heads, 64), w[name], name)
        dt, et = dt + w['dtable'][0], et + w['dtable'][1]
    within(dtable, (dt, et + 2.0 ** -8 * (dt.abs() + et) + 1e-30), 'dtable')
    assert bool((o.cpu()[idle] == 0).all()) and bool((dqkv.cpu()[idle] == 0).all())


@pytest.mark.parametrize('lens,packed', [([1], False), ([24, 7, 0, 31], False), ([24, 7, 0, 31], True), ([200, 0, 65, 129], False), ([200, 0, 65, 129], True),
                                         ([1000], False), ([3, 1], True), ([2100, 0, 5], True), ([600, 0, 37, 1500], False)])
def test_relpos_attention_cls(dev, lens, packed):
    from creamfl_amd import ops
    heads, H, B, L = 3, 192, len(lens), max(max(lens), 1)
    T = sum(lens)
    t = attn_inputs(T + B, B, L, heads)
    kvp, q0, do0 = t['qkv'][:, :, H:], t['qkv'][:, 0, :H], t['do'][:, 0]
    keep = torch.arange(L)[None] < torch.tensor(lens)[:, None]
    kv = kvp[keep] if packed else kvp
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32).to(dev)
    leaves = [x.contiguous().to(dev).requires_grad_(True) for x in (q0, kv, t['table'])]
    extra = dict(cu_seqlens=cu, max_len=L) if packed else dict(key_mask=keep.to(dev))
    o = ops.relpos_attention_cls(leaves[0], leaves[1], leaves[2], t['buckets'].to(dev), heads, **extra)
    dq, dkv, dtable = torch.autograd.grad(o, leaves, do0.contiguous().to(dev))
    dt, et = torch.zeros(32, heads, dtype=torch.float64), torch.zeros(32, heads, dtype=torch.float64)
    full = torch.zeros(B, L, 2 * H, dtype=torch.float64)
    full[keep] = dkv.double().cpu() if packed else dkv.double().cpu()[keep]
    if not packed:
        assert bool((dkv.cpu()[~keep] == 0).all())
    for b in range(B):
        k, v = (x.reshape(L, heads, 64) for x in kvp[b].split(H, 1))
        w = ref.relpos_attention_text(q0[b].view(1, heads, 64), k, v, t['table'], t['buckets'], keep[b], 0.125, do0[b].view(1, heads, 64))
        within(o[b].view(1, heads, 64), w['o'], 'o')
        within(dq[b].view(1, heads, 64), w['dq'], 'dq')
        within(full[b, :, :H].reshape(L, heads, 64), w['dk'], 'dk')
        within(full[b, :, H:].reshape(L, heads, 64), w['dv'], 'dv')
        dt, et = dt + w['dtable'][0], et + w['dtable'][1]
    within(dtable, (dt, et + 2.0 ** -8 * (dt.abs() + et) + 1e-30), 'dtable')


def test_relpos_attention_views_and_refusals(dev):
    from creamfl_amd import _lib, ops
    t = attn_inputs(3, 2, 20, 2)
    b = t['buckets'].to(dev)
    table = t['table'].to(dev)
    qkv = t['qkv'].to(dev)
    want = ops.relpos_attention(qkv, table, b, 2)
    wide = torch.zeros(2, 20, 400, dtype=torch.bfloat16, device=dev)
    wide[..., 5:389] = qkv
    assert torch.equal(ops.relpos_attention(wide[..., 5:389], table, b, 2), want)                 # strided, off the 16-byte border
    assert torch.equal(ops.relpos_attention(qkv.float(), table, b, 2), want)                      # another type: rounded to bf16 first
    assert torch.equal(ops.relpos_attention(qkv, table.t().contiguous().t(), b, 2), want)
    m = torch.ones(2, 20, dtype=torch.int64, device=dev)
    assert torch.equal(ops.relpos_attention(qkv, table, b, 2, key_mask=m), want)
    ok = dict(qkv=qkv, table=table, buckets=b, heads=2)
    for kw in (dict(heads=3), dict(heads=0), dict(table=table[:, :1]), dict(table=table[0]), dict(buckets=b[:-1]), dict(buckets=b.long()),
               dict(buckets=b.cpu()), dict(qkv=qkv[0]), dict(key_mask=m[:1]), dict(key_mask=m[:, :-1]), dict(key_mask=m.cpu()), dict(key_mask=m.float()), dict(qkv=qkv[:0]),
               dict(table=table.cpu())):
        with pytest.raises(_lib.CreamflHipError):
            ops.relpos_attention(**{**ok, **kw})
    cu = torch.tensor([0, 20, 40], dtype=torch.int32, device=dev)
    ok = dict(qkv=qkv.view(40, 384), cu_seqlens=cu, max_len=20, table=table, buckets=b, heads=2)
    assert torch.equal(ops.relpos_attention_varlen(**ok), want.view(40, 128))
    for kw in (dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu.cpu()), dict(max_len=0), dict(qkv=qkv), dict(cu_seqlens=cu[:1]), dict(heads=1)):
        with pytest.raises(_lib.CreamflHipError):
            ops.relpos_attention_varlen(**{**ok, **kw})
    q, kv = qkv[:, 0, :128].contiguous(), qkv[..., 128:].contiguous()
    ok = dict(q=q, kv=kv, table=table, buckets=b, heads=2)
    for kw in (dict(q=q[:1]), dict(kv=kv.view(40, 256), cu_seqlens=[0, 20, 40], max_len=20), dict(kv=kv[..., :128]), dict(kv=kv[0]), dict(cu_seqlens=cu), dict(kv=kv.view(40, 256), cu_seqlens=cu),
               dict(kv=kv.view(40, 256), cu_seqlens=cu, max_len=20, key_mask=m)):
        with pytest.raises(_lib.CreamflHipError):
            ops.relpos_attention_cls(**{**ok, **kw})


def test_relpos_attention_wild_offsets_stay_in_bounds(dev):
    """Offsets that run backwards or past the rows are clipped to the rows there are (the kernel's own bounds)."""
    from creamfl_amd import ops
    t = attn_inputs(3, 1, 20, 1)
    cu = torch.tensor([0, 30, 7, 12, -5], dtype=torch.int32, device=dev)      # text 0: rows 0 .. 19, the others: none
    qkv = t['qkv'][0].to(dev)
    o = ops.relpos_attention_varlen(qkv, cu, 20, t['table'].to(dev), t['buckets'].to(dev), 1)
    assert o.shape == (20, 64)


# ------------------------------------------------------------------------------------------------ streams, graphs
def _chain(dev):
    """The three operators as a tower step would chain them, on static buffers."""
    from creamfl_amd import ops
    g = torch.Generator().manual_seed(8)
    t = attn_inputs(8, 3, 50, 2)
    x = cl(torch.randn(3, 32, 5, 7, generator=g)).to(dev).requires_grad_(True)
    ga, be = torch.ones(32, device=dev, requires_grad=True), torch.zeros(32, device=dev, requires_grad=True)
    qkv, table = t['qkv'].to(dev).requires_grad_(True), t['table'].to(dev).requires_grad_(True)
    buckets = t['buckets'].to(dev)
    leaves = [x, ga, be, qkv, table]

    def step():
        f = ops.gn_act(x, ga, be, 8, act='silu')
        o = ops.relpos_attention(ops.dropout(qkv, 0.1, seed=21), table, buckets, 2)
        out = ops.dropout(f, 0.2, seed=22).float().sum() * 0.5 + (o.float() * torch.linspace(-1, 1, 128, device=dev)).sum()
        return [out.detach()] + [v.clone() for v in torch.autograd.grad(out, leaves)]
    return step, leaves


def test_other_stream_matches(dev):
    step, _ = _chain(dev)
    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_two_captured_graphs_replay(dev):
    """Forward and backward captured twice (each graph with workspaces of its own), replayed in turn with eager work between: every replay
    gives the eager bits for the inputs it finds."""
    def captured():
        step, leaves = _chain(dev)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        return step, leaves, g, out
    one, two = captured(), captured()
    gen = torch.Generator(device=dev).manual_seed(4)
    for k in range(4):
        for step, leaves, g, out in (one, two):
            with torch.no_grad():
                leaves[0].normal_(generator=gen)
                leaves[3].normal_(generator=gen)
            g.replay()
            got = [v.clone() for v in out]
            torch.cuda.synchronize()
            for a, b in zip(got, step()):
                assert torch.equal(a, b), k


# ------------------------------------------------------------------------------------------------ offsets past 32 bits
def test_relpos_attention_rows_past_32_bits(dev):
    """2.2e9 elements of qkv: the last texts' rows, a text of nearly all rows cut to 40, and the rest zero."""
    from creamfl_amd import ops
    T, heads, L = 950_000, 12, 40
    t = attn_inputs(3, 1, 1, heads)
    qkv = torch.zeros(T, 192 * heads, dtype=torch.bfloat16, device=dev)
    assert qkv.numel() > 1 << 31
    g = torch.Generator().manual_seed(6)
    cu = torch.tensor([0, 30, T - 75, T - 40, T], dtype=torch.int32)
    ends = [(0, 30), (30, 70), (T - 75, T - 40), (T - 40, T)]      # (what takes part of each text)
    parts = [torch.randn(b - a, 192 * heads, generator=g).to(torch.bfloat16) for a, b in ends]
    dos = [torch.randn(b - a, 64 * heads, generator=g).to(torch.bfloat16) for a, b in ends]
    do = torch.zeros(T, 64 * heads, dtype=torch.bfloat16, device=dev)
    for (a, b), x, d in zip(ends, parts, dos):
        qkv[a:b], do[a:b] = x.to(dev), d.to(dev)
    qkv.requires_grad_(True)
    o = ops.relpos_attention_varlen(qkv, cu.to(dev), L, t['table'].to(dev), t['buckets'].to(dev), heads)
    dqkv, = torch.autograd.grad(o, [qkv], do)
    H = heads * 64
    for (a, b), x, d in zip(ends, parts, dos):
        w = text_oracle(x, t['table'], t['buckets'], None, d)
        within(o[a:b].view(-1, heads, 64), w['o'], 'o from %d' % a)
        for i, name in enumerate(('dq', 'dk', 'dv')):
            within(dqkv[a:b, i * H:(i + 1) * H].reshape(-1, heads, 64), w[name], '%s from %d' % (name, a))
    assert not o[70:T - 75].any() and not dqkv[70:T - 75].any()


def test_gn_act_maps_past_32_bits(dev):
    """2.2e9 elements: the last sample's values and gradients against 64 bits."""
    from creamfl_amd import ops
    N, C, G, S = 33, 256, 32, 512
    x = torch.empty(N, C, S, S, dtype=torch.bfloat16, device=dev, memory_format=torch.channels_last)
    assert x.numel() > 1 << 31
    gen = torch.Generator(device=dev).manual_seed(3)
    for n in range(N):
        x[n] = torch.randn(C, S, S, device=dev, generator=gen) + n
    dy = torch.zeros_like(x)
    dy[-1] = torch.randn(C, S, S, device=dev, generator=gen)
    ga = (1 + 0.1 * torch.randn(C, device=dev, generator=gen)).requires_grad_(True)
    be = torch.zeros(C, device=dev, requires_grad=True)
    y = ops.gn_act(x.requires_grad_(True), ga, be, G)
    dx, dga, dbe = torch.autograd.grad(y, [x, ga, be], dy)
    v, d, w = x.detach()[-1].double().reshape(G, -1), dy[-1].double().reshape(G, C // G, -1), ga.detach().double().reshape(G, C // G, 1)
    mu = v.mean(1, keepdim=True)
    r = ((v - mu).square().mean(1, keepdim=True) + 1e-5).rsqrt()
    xh = (v - mu) * r
    # one rounding of the output, and in 32 bits what a mean of N adds to a deviation of 1: x - mu is exact to 2^-24 of the mean
    e = 2.0 ** -8
    want = (xh.reshape(G, C // G, -1) * w).reshape(C, S, S)
    assert bool(((y.detach()[-1].double() - want).abs() <= e * want.abs() + 64 * N * 2.0 ** -24).all())
    gg = (d * w).reshape(G, -1)
    want = (r * (gg - gg.mean(1, keepdim=True) - xh * (gg * xh).mean(1, keepdim=True))).reshape(C, S, S)
    assert bool(((dx[-1].double() - want).abs() <= e * want.abs() + 64 * N * 2.0 ** -24).all())
    assert not dx[:-1].any()
    # sums of 262144 products of about 1: pairwise over threads, at most sqrt(262144) ulps of the largest partial sum
    want = (d * xh.reshape(G, C // G, -1)).sum(2).reshape(-1)
    assert bool(((dga.double() - want).abs() <= 2.0 ** -24 * 512 * 64 * (1 + want.abs().max())).all())
    want = d.sum(2).reshape(-1)
    assert bool(((dbe.double() - want).abs() <= 2.0 ** -24 * 512 * 64 * (1 + want.abs().max())).all())


def test_dropout_elements_past_33_bits(dev):
    """Elements are counted in pairs by a 64-bit number: behind 2^33 its upper half changes the flags."""
    from creamfl_amd import ops
    n, p, seed = (1 << 33) + 5001, 0.25, 77
    y = ops.dropout(torch.ones(n, dtype=torch.bfloat16, device=dev), p, seed=seed)
    f = float(torch.tensor(4 / 3).to(torch.bfloat16))
    for start, s in ((0, seed), (1 << 33, seed + 0x632BE5AB)):
        got = y[start:start + 5001].float().cpu()
        assert torch.equal(got, torch.where(ref.keep_flags(s, p, 5001), torch.full_like(got, f), torch.zeros_like(got))), start
    assert not torch.equal(y[:5001], y[1 << 33:])
