"""GPU: group norm, counter-based dropout and relative-position attention where the framework calls them -- the trunks, the text tower, the
server's training step (src/networks/models/pcme.py:43-57, src/algorithms/retrieval_trainer.py:192-214) -- against the same modules on the
library path in 32 bits on the CPU."""
import copy
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8             # one rounding to bf16: half a step, relative


@pytest.fixture(scope='module')
def dev():
    if not torch.cuda.is_available():
        pytest.skip('needs a GPU')
    return torch.device('cuda:0')


def off(a, b):
    a, b = a.detach().double().cpu().flatten(), b.detach().double().cpu().flatten()
    return float((a - b).norm() / (b.norm() + 1e-30))


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


def relative_bert(dropout=0.0):
    from creamfl_amd.networks.backbones import BertModel
    torch.manual_seed(3)
    m = BertModel('bert-mini-relative')
    with torch.no_grad():
        m.encoder.relative_attention_bias.weight.normal_()     # (a bias that matters)
    for mod in m.modules():
        if isinstance(mod, torch.nn.Dropout):
            mod.p = dropout
    return m


# A layer rounds to bf16: four weights and their inputs' products (query-key-value, out, two of the feed-forward), P, o, two normed sums, the
# activation: 13; four layers and the embeddings' two: 54.  Were each half a step off in the same direction, an output would be 54 half steps off
# relative to what flows through; the root mean square of a rounding is 1 / sqrt(3) of it: 31.  The gradients pass every layer twice.
BERT_OUT, BERT_GRAD = 31 * HALF, 62 * HALF


@pytest.mark.parametrize('L', [24, 90])
def test_relative_text_tower_padded_packed_and_cls(dev, L):
    """bf16 on the GPU in its three forms against 32 bits on the CPU: states of the real tokens, gradients of every parameter, the shared bias table
    among them (it collects all layers')."""
    from creamfl_amd.networks.backbones import BertModel
    ref = relative_bert()
    m = copy.deepcopy(ref).to(dev).train()
    B = 6
    g = torch.Generator().manual_seed(L)
    lens = torch.tensor([L, 3, 1, L - 5, L // 2, 17])
    mask = torch.arange(L)[None] < lens[:, None]
    ids = torch.randint(1, 1000, (B, L), generator=g) * mask
    wc, wf = torch.randn(B, 256, generator=g), torch.randn(B, L, 256, generator=g) * mask[..., None]

    def run(model, where, cls, pack=None):
        model.zero_grad(set_to_none=True)
        with torch.autocast('cuda', dtype=torch.bfloat16, enabled=where != 'cpu'):
            h = model(ids.to(where), attention_mask=mask.to(where), cls_only=cls, pack=pack)['last_hidden_state']
        h = h.float()
        ((h[:, 0] * wc.to(where)).sum() if cls else (h * wf.to(where)).sum()).backward()
        h = h[:, 0] if cls else h * mask[..., None].to(where)
        return h, {n: p.grad.float().cpu().clone() for n, p in model.named_parameters() if p.grad is not None}
    plan = BertModel.pack_plan(lens.tolist(), L, dev, m.pack_longest)
    assert plan is not None
    for cls in (False, True):
        want, gw = run(ref.train(), 'cpu', cls)
        for pack in (None, plan):
            (got, gg), names = launched(lambda: run(m, dev, cls, pack))
            assert 'relpos_fwd' in names and ('relpos_bwd32' if L <= 32 else 'relpos_dkv') in names, names
            assert off(got, want) <= BERT_OUT, (cls, pack is not None, off(got, want))
            assert set(gg) == set(gw)
            for n in gw:
                if not n.endswith('key.bias'):                  # (zero: a row's softmax does not see it)
                    assert off(gg[n], gw[n]) <= BERT_GRAD, (cls, pack is not None, n, off(gg[n], gw[n]))


def smallest_map(model, x):
    """Elements of the smallest normalised map in a pass of x."""
    seen = []
    hooks = [m.register_forward_hook(lambda m, i, o: seen.append((o[0] if isinstance(o, tuple) else o).numel()))
             for m in model.modules() if isinstance(m, torch.nn.GroupNorm)]
    with torch.no_grad():
        model(x)
    for h in hooks:
        h.remove()
    return min(seen)


def gate_bound(linear, step, smallest):
    """The bound of a ResNet-18's gradients: `linear`, and the ReLUs whose inputs are so near zero that rounding decides them.  An input with
    relative noise e (root mean square; the inputs are normalised) has the other sign with probability e / pi: the mean of |noise|, e sqrt(2 / pi),
    times the density at zero, 1 / sqrt(2 pi).  Half the gradients pass, so that flipped gates are 2 e / pi of the gradient's square.  Behind l
    layers of three roundings of `step` / sqrt(3) each, e = step sqrt(l); 17 layers add up their squares.  That is what is expected.  Where e is so
    small that a map has less than one such gate on the mean (23040 inputs, e = 2e-5: 0.15), one is still a gate of the N / 2 that pass: 2 / N of
    the square.  More than three beyond the mean in one map have a chance below 0.15^4 / 4! = 2e-5, so three in the smallest map are allowed for."""
    return (linear ** 2 + 2 / 3.141592653589793 * step * sum(l ** 0.5 for l in range(1, 18)) + 3 * 2 / smallest) ** 0.5


@pytest.mark.parametrize('half', [False, True], ids=['fp32', 'bf16'])
def test_group_normed_trunk(dev, half):
    """A ResNet-18 whose normalisation is per sample, channels_last: feature map and gradients against the CPU.  In 32 bits the convolutions'
    sums of up to 4608 products decide (20 of them, each at most 2^-24 sqrt(4608) off on the root mean square, twice in a gradient); in bf16
    every convolution rounds weight and output and every normalisation its output: 60 roundings, twice in a gradient, 1 / sqrt(3) of half a
    step each."""
    from creamfl_amd.networks import backbones
    torch.manual_seed(5)
    ref = backbones.resnet_trunk('resnet18', 'group')
    m = copy.deepcopy(ref).to(dev).to(memory_format=torch.channels_last).train()
    g = torch.Generator().manual_seed(2)
    x = torch.randn(5, 3, 96, 96, generator=g)
    w = torch.randn(5, 512, 3, 3, generator=g)

    def run(model, t):
        model.zero_grad(set_to_none=True)
        with torch.autocast('cuda', dtype=torch.bfloat16, enabled=half and t.is_cuda):
            y = model(t)
        (y.float() * w.to(t.device)).sum().backward()
        return y.float(), {n: p.grad.float().cpu().clone() for n, p in model.named_parameters()}
    want, gw = run(ref.train(), x)
    (got, gg), names = launched(lambda: run(m, x.to(dev).contiguous(memory_format=torch.channels_last)))
    assert 'gn_res' in names, names
    small = smallest_map(ref, x)
    bound = 60 * HALF / 3 ** 0.5 if half else 20 * 2.0 ** -24 * 4608 ** 0.5
    assert off(got, want) <= bound, off(got, want)
    for n in gw:
        assert off(gg[n], gw[n]) <= gate_bound(2 * bound, HALF if half else 2.0 ** -24 * 4608 ** 0.5, small), (n, off(gg[n], gw[n]))


def server(dev, half, dropout=None):
    from creamfl_amd.algorithms.retrieval_trainer import TrainerEngine
    from creamfl_amd.utils.config import default_config
    torch.manual_seed(0)
    cfg = default_config(embed_dim=64, cnn_type='resnet18', not_bert=False)
    cfg.model.bert_name, cfg.model.image_norm = 'bert-mini-relative', 'group'
    eng = TrainerEngine(device=dev)
    msgs = []
    eng.set_logger(SimpleNamespace(log=msgs.append, update_tracker=lambda *a, **k: None))
    eng.create(cfg, {'<pad>': 0}, None, False)
    eng.model_to_device()
    if half:
        eng.to_half()
    if dropout is not None:
        for mod in eng.model.modules():
            if isinstance(mod, torch.nn.Dropout):
                mod.p = dropout
    return eng, msgs


def test_server_step_calls_all_three(dev):
    """One training step of the server in bf16 with dropout on: every trainable parameter has a finite gradient, a step is taken, and the kernels ran."""
    from creamfl_amd.utils.synthetic import coco_batch
    eng, _ = server(dev, True)
    b = coco_batch(12, 'cpu', seed=5, bert=True, img=96)
    eng.model.train()
    before = {n: p.detach().float().clone() for n, p in eng.model.named_parameters()}
    (loss, _), names = launched(lambda: eng.train_step(b[0].to(dev), b[1].to(dev), None, b[3]))
    assert torch.isfinite(loss)
    assert {'gn_res', 'relpos_fwd', 'dropout'} <= names and names & {'relpos_bwd32', 'relpos_dkv'}, names
    for n, p in eng.model.named_parameters():
        if p.requires_grad:
            assert torch.isfinite(p).all(), n
    moved = [n for n, p in eng.model.named_parameters() if not torch.equal(p.detach().float(), before[n])]
    assert 'txt_enc.encoder.relative_attention_bias.weight' in moved and any('bn1.weight' in n for n in moved)


def test_server_step_in_a_graph(dev):
    """The captured step (towers on two streams, dropout by the device's tick) replays, and its weights stay finite; with dropout off it trains as the
    eager loop does.  The captured step pads the captions, the eager one packs them, so their gradients differ by the text tower's roundings,
    relatively by at most e = BERT_GRAD.  A step of this optimizer goes by a gradient's sign where it begins, and rounding decides that sign with
    probability e / pi (as in gate_bound); a turned step is off by twice its length: 4 e / pi of the square."""
    from creamfl_amd.utils.synthetic import coco_batch
    batches = [coco_batch(16, 'cpu', seed=70 + i, bert=True, img=64, min_len=18, max_len=24, index0=16 * i) for i in range(8)]

    def run(graph, dropout):
        eng, msgs = server(dev, True, dropout)
        first = torch.cat([p.detach().float().flatten() for p in eng.model.parameters()])
        eng.server_graph = graph
        with torch.backends.cudnn.flags(enabled=True, benchmark=False):
            eng.train(batches)
        torch.cuda.synchronize()
        if graph:
            gs = eng.graph_stats.get('train')
            assert gs is not None and gs['failed'] is None, (gs, msgs)
            assert gs['replays'] >= 4
        flat = torch.cat([p.detach().float().flatten() for p in eng.model.parameters()])
        assert bool(torch.isfinite(flat).all())
        return flat - first
    run(True, None)
    e, g = run(False, 0.0), run(True, 0.0)
    assert off(g, e) <= (4 * BERT_GRAD / 3.141592653589793) ** 0.5, off(g, e)


def test_client_step(dev):
    """A client's encoder with per-sample normalisation, 32 bits, channels_last, one image in its batch: features and gradients against the CPU."""
    from creamfl_amd.networks.resnet_client import resnet18_client
    torch.manual_seed(1)
    ref = resnet18_client(num_class=10, is_train=True, scale=128, embed_dim=512, norm='group')
    m = copy.deepcopy(ref).to(dev).to(memory_format=torch.channels_last).train()
    for B in (1, 4):
        x = torch.randn(B, 3, 32, 32, generator=torch.Generator().manual_seed(B))

        def run(model, t):
            model.zero_grad(set_to_none=True)
            out = model(t)
            outs = [o.float() for o in (out if isinstance(out, (tuple, list)) else (out,)) if torch.is_tensor(o)]
            sum((o * torch.linspace(-1, 1, o.numel(), device=o.device).view_as(o)).sum() for o in outs).backward()
            return outs, {n: p.grad.float().cpu().clone() for n, p in model.named_parameters() if p.grad is not None}
        want, gw = run(ref.train(), x)
        (got, gg), names = launched(lambda: run(m, x.to(dev).contiguous(memory_format=torch.channels_last)))
        assert 'gn_res' in names
        bound = 20 * 2.0 ** -24 * 4608 ** 0.5                  # (as for the trunk in 32 bits)
        for a, b in zip(got, want):
            assert off(a, b) <= bound, off(a, b)
        for n in gw:
            assert off(gg[n], gw[n]) <= gate_bound(2 * bound, 2.0 ** -24 * 4608 ** 0.5, smallest_map(ref, x)), (n, off(gg[n], gw[n]))
