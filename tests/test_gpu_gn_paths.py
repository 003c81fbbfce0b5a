"""GPU: group norm in each of the ways csrc/gnorm.hip runs it -- one pass over registers, two passes over a slice, chunks of rows -- against
its 64-bit restatement (oracle/tower_ops.py), on maps as large as the ways' rules ask for.  The statistics are per sample, so the oracle
takes a few samples of a large batch; the gradient of the others is zero, and so are their shares of dgamma and dbeta."""
import numpy as np
import pytest
import torch

from oracle import tower_ops as ref

pytestmark = pytest.mark.gpu
DT = {'fp32': torch.float32, 'bf16': torch.bfloat16}


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


def fmap(shape, dtype, dev, gen, scale=1.0, shift=0.0):
    return torch.empty(shape, dtype=DT[dtype], device=dev, memory_format=torch.channels_last).normal_(shift, scale, generator=gen)


def sample_oracle(x, ga, be, groups, picks, act, res, dy, dtype):
    p = torch.tensor(picks, device=x.device)
    return ref.group_norm_act(x[p], ga, be, groups, act=act, residual=None if res is None else res[p], dy=None if dy is None else dy[p],
                              bf16=dtype == 'bf16')


# one pass, one pass of few records, chunks, two passes (of the backward)
GATE_SHAPES = [((2, 256, 14, 13, 32), 'bf16'), ((2, 64, 13, 17, 32), 'fp32'), ((3, 64, 3, 3, 8), 'bf16'), ((1, 64, 112, 111, 16), 'fp32'),
               ((1, 64, 112, 111, 16), 'bf16'), ((128, 72, 10, 10, 9), 'bf16'), ((64, 40, 10, 10, 5), 'fp32'), ((64, 40, 10, 10, 40), 'fp32')]


@pytest.mark.parametrize('shape,dtype', GATE_SHAPES, ids=str)
@pytest.mark.parametrize('two', [False, True], ids=['', 'two'])
def test_gradients_at_closed_gates_do_not_count(dev, shape, dtype, two):
    """Infinite and NaN gradients where ReLU is closed: zeros, as if nothing had arrived there."""
    from creamfl_amd import ops
    n, c, h, w, groups = shape
    gen = torch.Generator(device=dev).manual_seed(n + c)
    picks = sorted({0, n // 2, n - 1})
    x, r = fmap((n, c, h, w), dtype, dev, gen), fmap((n, c, h, w), dtype, dev, gen)
    ga, be = 1 + 0.3 * torch.randn(c, device=dev, generator=gen), 0.3 * torch.randn(c, device=dev, generator=gen)
    dy, dy2 = torch.zeros_like(x), torch.zeros_like(x)
    dy[picks] = fmap((len(picks), c, h, w), dtype, dev, gen)
    if two:
        dy2[picks] = fmap((len(picks), c, h, w), dtype, dev, gen)
    z = torch.nn.functional.group_norm(x.float(), groups, ga, be) + r.float()
    shut = z < -0.5                                            # (far beyond any rounding of z)
    g = dy.double() + dy2.double()
    g[shut] = 0
    want = sample_oracle(x, ga, be, groups, picks, 'relu', r, g, dtype)
    k = torch.randint(0, 4, shut.shape, device=dev, generator=gen)
    for i, bad in enumerate((float('inf'), float('nan'), -float('inf'))):
        dy[shut & (k == i)] = bad
    if two:
        dy2[shut & (k == 0)] = -float('inf')
    leaves = [t.requires_grad_(True) for t in (x, ga, be, r)]
    if two:
        y, y2 = ops.gn_act(x, ga, be, groups, act='relu', residual=r, two=True)
        grads = torch.autograd.grad([y, y2], leaves, [dy, dy2])
    else:
        grads = torch.autograd.grad(ops.gn_act(x, ga, be, groups, act='relu', residual=r), leaves, dy)
    for name, t in zip(('dx', 'dgamma', 'dbeta', 'dres'), grads):
        within(t if t.dim() == 1 else t[picks], want[name], name)


# Maps that run in two passes (a thread of 98 to 512 rows), in one pass and in chunks: the same statistics wherever a far value stands.
@pytest.mark.parametrize('shape,dtype', [((128, 64, 256, 256, 32), 'bf16'), ((128, 64, 256, 256, 8), 'bf16'), ((128, 64, 128, 128, 32), 'fp32'), ((256, 64, 256, 256, 8), 'fp32'),
                                         ((40, 64, 32, 32, 8), 'fp32'), ((1, 64, 256, 256, 8), 'fp32'), ((128, 72, 10, 10, 9), 'bf16'), ((64, 40, 52, 52, 40), 'fp32')], ids=str)
@pytest.mark.parametrize('rest', ['flat', 'noise', 'high'])
def test_statistics_keep_their_digits_beside_a_far_first_value(dev, shape, dtype, rest):
    """A first pixel at 30000 (1000.3 beside a flat rest): the variance is nearly all that pixel's, and xh of it sqrt(M) -- every digit of the sum of
    squares shows.  `high`: a mean of 300 deviations without a far value."""
    from creamfl_amd import ops
    n, c, h, w, groups = shape
    gen = torch.Generator(device=dev).manual_seed(h + groups)
    x = fmap((n, c, h, w), dtype, dev, gen)
    if rest == 'flat':
        x.copy_(torch.linspace(-1, 1, c, device=dev)[None, :, None, None].expand_as(x))
    if rest == 'high':
        x.add_(300)
    else:
        x[:, :, 0, 0] = 30000.0 if rest == 'noise' else 1000.3
    ga, be = 1 + 0.3 * torch.randn(c, device=dev, generator=gen), 0.3 * torch.randn(c, device=dev, generator=gen)
    y = ops.gn_act(x, ga, be, groups)
    picks = sorted({0, n // 2, n - 1})
    within(y[picks], sample_oracle(x, ga, be, groups, picks, 'none', None, None, dtype)['y'], 'y')


def test_constant_gradients_sum_without_drift(dev):
    """Equal gradients at every position (what mean pooling sends): a chain of equal terms rounds the same way at every step.  Two passes, 576 rows a
    thread; a constant for each of 32 channels."""
    from creamfl_amd import ops
    n, c, h, w, groups = 256, 32, 384, 384, 4
    gen = torch.Generator(device=dev).manual_seed(9)
    x = fmap((n, c, h, w), 'fp32', dev, gen).requires_grad_(True)
    ga, be = (1 + 0.3 * torch.randn(c, device=dev, generator=gen)).requires_grad_(True), torch.zeros(c, device=dev, requires_grad=True)
    picks = [0, n - 1]
    dy = torch.zeros_like(x, requires_grad=False)
    dy[picks] = (0.5 + torch.rand(c, device=dev, generator=gen))[None, :, None, None]
    dx, dga, dbe = torch.autograd.grad(ops.gn_act(x, ga, be, groups), [x, ga, be], dy)
    want = sample_oracle(x.detach(), ga.detach(), be.detach(), groups, picks, 'none', None, dy, 'fp32')
    within(dbe, want['dbeta'], 'dbeta')
    within(dga, want['dgamma'], 'dgamma')
    within(dx[picks], want['dx'], 'dx')


# (n, c, h, w, groups), type, the forward's and the backward's way as cfl_gn_plan names them: kind ('chunks', 'one', 'few', 'two'), threads, whether
# groups are whole records of 8 channels.  The server's trunk at a batch of 256 takes ('two', 1024) for its stem and first stage, 'one' with 14
# records a thread behind them; tests/test_tower_ops_limits.py checks on the CPU that every way is in this list.
PATHS = [
    ((256, 64, 113, 111, 32), 'bf16', ('two', 1024, False), ('two', 1024)),
    ((256, 64, 57, 55, 32), 'bf16', ('two', 1024, False), ('two', 1024)),
    ((256, 128, 57, 55, 8), 'bf16', ('two', 1024, True), ('two', 1024)),
    ((128, 72, 31, 29, 24), 'bf16', ('two', 512, False), ('two', 512)),
    ((128, 72, 31, 29, 9), 'bf16', ('two', 512, True), ('two', 512)),
    ((128, 72, 9, 11, 24), 'bf16', ('two', 256, False), ('two', 256)),
    ((128, 72, 9, 11, 9), 'bf16', ('two', 256, True), ('two', 256)),
    ((256, 64, 57, 55, 32), 'fp32', ('two', 1024, False), ('two', 1024)),
    ((256, 64, 57, 55, 8), 'fp32', ('two', 1024, True), ('two', 1024)),
    ((64, 40, 52, 53, 40), 'fp32', ('two', 512, False), ('two', 512)),
    ((64, 40, 52, 53, 5), 'fp32', ('two', 512, True), ('two', 512)),
    ((64, 40, 9, 11, 40), 'fp32', ('two', 256, False), ('two', 256)),
    ((64, 40, 9, 11, 5), 'fp32', ('two', 256, True), ('two', 256)),
    ((128, 512, 29, 27, 32), 'bf16', ('one', 512, True), ('one', 512)),
    ((256, 256, 14, 14, 32), 'bf16', ('one', 128, True), ('one', 128)),
    ((256, 128, 29, 27, 32), 'bf16', ('one', 256, False), ('one', 256)),
    ((128, 128, 29, 27, 32), 'fp32', ('one', 256, False), ('one', 256)),
    ((128, 256, 14, 14, 32), 'fp32', ('one', 128, True), ('one', 128)),
    ((128, 512, 7, 7, 32), 'bf16', ('few', 128, True), ('few', 128)),
    ((128, 64, 16, 16, 32), 'fp32', ('few', 256, False), ('few', 256)),
    ((128, 512, 7, 7, 32), 'fp32', ('few', 128, True), ('few', 128)),
    ((66, 64, 16, 16, 32), 'bf16', ('few', 256, False), ('few', 256)),
    ((1, 64, 113, 111, 32), 'bf16', ('chunks',), ('chunks',)),
    ((2, 64, 113, 111, 8), 'fp32', ('chunks',), ('chunks',)),
]


def way(shape, dtype, bwd):
    from creamfl_amd import _lib
    n, c, h, w, groups = shape
    p = _lib.load().cfl_gn_plan(n, h * w, c, groups, int(dtype == 'bf16'), int(bwd))
    assert p >= 0, p
    kind = ('chunks', 'few' if p & 4 else 'one', 'two')[p & 3]
    return (kind,) if kind == 'chunks' else (kind, p >> 4) if bwd else (kind, p >> 4, not p & 8)


@pytest.mark.parametrize('shape,dtype,fwd,bwd', PATHS, ids=str)
@pytest.mark.parametrize('act,res,two', [('none', False, False), ('relu', False, False), ('relu', True, True), ('silu', True, False)])
def test_every_way_matches_oracle(dev, shape, dtype, fwd, bwd, act, res, two):
    """Values and gradients of the first, the last and a middle sample, in the forms that the trunks call: with and without a residual, with one
    gradient and with two."""
    from creamfl_amd import ops
    assert way(shape, dtype, False) == fwd and way(shape, dtype, True) == bwd, (way(shape, dtype, False), way(shape, dtype, True))
    n, c, h, w, groups = shape
    gen = torch.Generator(device=dev).manual_seed(n * 31 + c + h)
    picks = sorted({0, n // 2, n - 1})
    x, r = fmap((n, c, h, w), dtype, dev, gen, 1.5, 0.5), fmap((n, c, h, w), dtype, dev, gen) if res else None
    ga, be = 1 + 0.3 * torch.randn(c, device=dev, generator=gen), 0.3 * torch.randn(c, device=dev, generator=gen)
    dy, dy2 = torch.zeros_like(x), torch.zeros_like(x) if two else None
    dy[picks] = fmap((len(picks), c, h, w), dtype, dev, gen)
    if two:
        dy2[picks] = fmap((len(picks), c, h, w), dtype, dev, gen)
    want = sample_oracle(x, ga, be, groups, picks, act, r, dy.double() + dy2.double() if two else dy, dtype)
    leaves = [t.requires_grad_(True) for t in ((x, ga, be, r) if res else (x, ga, be))]
    y = ops.gn_act(x, ga, be, groups, act=act, residual=r, two=two)
    grads = torch.autograd.grad(list(y) if two else [y], leaves, [dy, dy2] if two else [dy])
    y = y[0] if two else y
    within(y[picks], want['y'], 'y')
    for name, t in zip(('dx', 'dgamma', 'dbeta', 'dres'), grads):
        within(t if t.dim() == 1 else t[picks], want[name], name)
    rest = torch.ones(n, dtype=torch.bool, device=dev)
    rest[picks] = False
    assert bool(torch.isfinite(y[rest]).all()) and not bool((grads[0][rest] != 0).any())
    with torch.no_grad():                                  # the forward alone, on another stream: the same bits
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            again = ops.gn_act(x, ga, be, groups, act=act, residual=r)
        torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(again, y)


@pytest.mark.parametrize('shape', [(1, 8, 1000, 1000, 1), (1, 8, 300, 300, 1), (1, 64, 512, 512, 8), (130, 8, 100, 100, 1), (40, 64, 32, 32, 8)], ids=str)
def test_constant_gradients_sum_without_drift_in_chunks_and_in_one_pass(dev, shape):
    """dbeta of a constant gradient, 24 constants a channel; the bound is the oracle's for a sum (64 halves of a last place).  Eight channels have 256
    row phases to a chunk."""
    from creamfl_amd import ops
    n, c, h, w, groups = shape
    for seed in range(24):
        gen = torch.Generator(device=dev).manual_seed(seed)
        x = fmap((n, c, h, w), 'fp32', dev, gen).requires_grad_(True)
        ga, be = torch.ones(c, device=dev, requires_grad=True), torch.zeros(c, device=dev, requires_grad=True)
        k = 0.5 + torch.rand(c, device=dev, generator=gen)
        dy = k[None, :, None, None].expand(n, c, h, w).contiguous(memory_format=torch.channels_last)
        dbe = torch.autograd.grad(ops.gn_act(x, ga, be, groups), [x, ga, be], dy)[2]
        want = k.double().cpu() * (n * h * w)
        within(dbe, (want, 64 * 2.0 ** -24 * want), 'dbeta, seed %d' % seed)
