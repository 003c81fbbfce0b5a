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
