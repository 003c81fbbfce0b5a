"""GPU: every call that the towers and the server's step make of group norm, counter-based dropout and relative-position attention, taken where it is
made -- the tensors the framework passes, the values and gradients that come back -- and held to the operators' own bounds (oracle/tower_ops.py).
Network-wide comparisons have to allow for the roundings of all layers; a call has only its own."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from oracle import tower_ops as ref

pytestmark = pytest.mark.gpu
U16 = 2.0 ** -8


@pytest.fixture(scope='module')
def dev():
    if not torch.cuda.is_available():
        pytest.skip('needs a GPU')
    return torch.device('cuda:0')


def within(got, value, bound, name):
    off = (got.detach().double().cpu() - value).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), '%s: %d of %d outside, worst %.3g of its bound at %s' % (
        name, int(bad.sum()), bad.numel(), float((off / bound).nan_to_num(nan=np.inf).max()), tuple(bad.nonzero()[0].tolist()))


class _Tap(torch.autograd.Function):
    """The tensor itself; its gradient -- what the operator behind it returns -- is kept."""
    @staticmethod
    def forward(ctx, t, call, name):
        ctx.to = (call, name)
        return t.view_as(t)

    @staticmethod
    def backward(ctx, g):
        call, name = ctx.to
        call[name] = g.detach().clone()
        return g, None, None


class Calls(list):
    """The operators' entry points replaced by ones that note each call and pass it on."""

    def __init__(self, monkeypatch):
        super().__init__()
        from creamfl_amd import ops
        for op in ('gn_act', 'dropout', 'relpos_attention', 'relpos_attention_varlen', 'relpos_attention_cls'):
            monkeypatch.setattr(ops, op, self._noted(op, getattr(ops, op)))

    def _noted(self, op, real):
        import inspect
        sig = inspect.signature(real)

        def fn(*args, **kw):
            b = sig.bind(*args, **kw)
            b.apply_defaults()
            call = dict(op=op, **{k: v.detach().clone() if torch.is_tensor(v) else v for k, v in b.arguments.items()})
            for k, v in b.arguments.items():
                if torch.is_tensor(v) and v.requires_grad:
                    b.arguments[k] = _Tap.apply(v, call, 'd_' + k)
            out = real(*b.args, **b.kwargs)
            outs = out if isinstance(out, tuple) else (out,)
            call['out'] = outs[0].detach().clone()
            call['d_out'] = []
            for o in outs:
                if o.requires_grad:
                    o.register_hook(lambda g: call['d_out'].append(g.detach().clone()) if g is not None else None)     # (None: an unused one of two)
            self.append(call)
            return out
        return fn

    def of(self, op):
        return [c for c in self if c['op'] == op]


def check_gn(c, name):
    dy = sum(g.double() for g in c['d_out']) if c['d_out'] else None
    x = c['x']
    w = ref.group_norm_act(x, c['weight'], c['bias'], c['groups'], c['eps'], c['act'], c['residual'], dy, bf16=x.dtype == torch.bfloat16)
    within(c['out'], *w['y'], name + ' y')
    n = 0
    for grad, key in (('d_x', 'dx'), ('d_residual', 'dres'), ('d_weight', 'dgamma'), ('d_bias', 'dbeta')):
        if grad in c:
            value, bound = w[key]
            if c[grad].dtype == torch.bfloat16 and key in ('dgamma', 'dbeta'):
                bound = bound + U16 * (value.abs() + bound)            # (a bf16 parameter's gradient is rounded once more)
            within(c[grad], value, bound, '%s %s' % (name, key))
            n += 1
    return n


def check_dropout(c, name):
    x, y, p = c['x'], c['out'], round(65536 * c['p']) / 65536
    half = torch.finfo(x.dtype).eps / 2
    keep = (y != 0) | (x == 0)
    f = 1 / (1 - p)
    want = torch.where(keep, x.double() * f, torch.zeros_like(x, dtype=torch.float64)).cpu()
    within(y, want, want.abs() * (half + 2.0 ** -23) + 1e-30, name + ' y')
    share, n = float(keep.double().mean()), keep.numel()
    assert abs(share - (1 - p)) <= 6 * (p * (1 - p) / n) ** 0.5 + 1 / n, (name, share)
    if 'd_x' in c:
        (dy,) = c['d_out']
        want = torch.where(keep, dy.double() * f, torch.zeros_like(dy, dtype=torch.float64)).cpu()
        within(c['d_x'], want, want.abs() * (half + 2.0 ** -23) + 1e-30, name + ' dx')


def check_attention(c, name):
    """Text by text, whatever the form."""
    heads, table, buckets = c['heads'], c['table'], c['buckets']
    H = heads * 64
    scale = 0.125 if c['scale'] is None else c['scale']
    form = c['op']
    trained = bool(c['d_out'])
    if form == 'relpos_attention_varlen':
        cu = c['cu_seqlens'].tolist()
        texts = [(slice(a, a + min(b - a, c['max_len'])), None) for a, b in zip(cu, cu[1:])]
    elif form == 'relpos_attention_cls' and c['cu_seqlens'] is not None:
        cu = c['cu_seqlens'].tolist()
        texts = [(slice(a, a + min(b - a, c['max_len'])), None) for a, b in zip(cu, cu[1:])]
    else:
        m = c['key_mask']
        B = (c['kv'] if form == 'relpos_attention_cls' else c['qkv']).shape[0]
        texts = [(b, None if m is None else m.reshape(B, -1)[b].bool().cpu()) for b in range(B)]
    dt, et = torch.zeros(table.shape, dtype=torch.float64), torch.zeros(table.shape, dtype=torch.float64)
    for b, (at, keep) in enumerate(texts):
        if form == 'relpos_attention_cls':
            q, src, lead = c['q'][b:b + 1], c['kv'][at], 0
            o, do = c['out'][b:b + 1], c['d_out'][0][b:b + 1] if trained else None
        else:
            src, lead = c['qkv'][at], H
            q, o, do = src[:, :H], c['out'][at], c['d_out'][0][at] if trained else None
        L = src.shape[0]
        q, k, v = (t.to(torch.bfloat16).reshape(-1, heads, 64) for t in (q, src[:, lead:lead + H], src[:, lead + H:]))
        w = ref.relpos_attention_text(q, k, v, table, buckets, keep, scale, None if do is None else do.reshape(-1, heads, 64))
        tag = '%s text %d ' % (name, b)
        within(o.reshape(-1, heads, 64), *w['o'], tag + 'o')
        if not trained:
            continue
        if form == 'relpos_attention_cls':
            dq, dk, dv = c['d_q'][b:b + 1], c['d_kv'][at][:, :H], c['d_kv'][at][:, H:]
        else:
            dq, dk, dv = c['d_qkv'][at].split(H, 1)
        for t, key in ((dq, 'dq'), (dk, 'dk'), (dv, 'dv')):
            within(t.reshape(-1, heads, 64), *w[key], tag + key)
        dt, et = dt + w['dtable'][0], et + w['dtable'][1]
    if trained:
        half = torch.finfo(c['d_table'].dtype).eps / 2
        within(c['d_table'], dt, et + half * (dt.abs() + et) + 1e-30, name + ' dtable')


@pytest.mark.parametrize('name,half', [('resnet18', False), ('resnet18', True), ('resnet50', False), ('resnet50', True)])
def test_group_norm_of_a_trunk_call_by_call(dev, monkeypatch, name, half):
    """Stem, blocks with their two gradients and residuals, projections: as many calls as there are normalisations, each within the operator's bounds."""
    from creamfl_amd import ops
    from creamfl_amd.networks import backbones
    torch.manual_seed(5)
    m = backbones.resnet_trunk(name, 'group').to(dev).to(memory_format=torch.channels_last).train()
    with torch.no_grad():
        for mod in m.modules():
            if isinstance(mod, torch.nn.GroupNorm):
                mod.weight.add_(0.3 * torch.randn_like(mod.weight))
                mod.bias.add_(0.3 * torch.randn_like(mod.bias))
    calls = Calls(monkeypatch)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(3, 3, 72, 88, generator=g).to(dev).contiguous(memory_format=torch.channels_last)
    with ops.join_scope():
        with torch.autocast('cuda', dtype=torch.bfloat16, enabled=half):
            y = m(x)
        (y.float() * torch.randn(y.shape, generator=g).to(dev)).sum().backward()
    torch.cuda.synchronize()
    norms = sum(isinstance(mod, torch.nn.GroupNorm) for mod in m.modules())
    assert len(calls) == norms == {'resnet18': 20, 'resnet50': 53}[name]
    for i, c in enumerate(calls):
        assert c['x'].dtype == (torch.bfloat16 if half else torch.float32)
        assert check_gn(c, 'call %d %s' % (i, tuple(c['x'].shape))) == (4 if c['residual'] is not None else 3)
    blocks = [c for c in calls if c['two']]
    assert len(blocks) == {'resnet18': 8, 'resnet50': 16}[name] and all(len(c['d_out']) == 2 for c in blocks[:-1])


@pytest.mark.parametrize('L', [24, 90])
@pytest.mark.parametrize('packed', [False, True], ids=['padded', 'packed'])
@pytest.mark.parametrize('cls', [False, True], ids=['all', 'cls'])
def test_attention_of_a_text_tower_call_by_call(dev, monkeypatch, L, packed, cls):
    """Four layers, the last one for [CLS] alone where that is asked for: the mask or the offsets that the tower passes are the batch's, and every
    layer's values and gradients are within the operator's bounds."""
    from creamfl_amd.networks.backbones import BertModel
    torch.manual_seed(3)
    m = BertModel('bert-mini-relative').to(dev).train()
    with torch.no_grad():
        m.encoder.relative_attention_bias.weight.normal_()
        for layer in m.encoder.layer:                          # (attention that picks: fresh weights give nearly equal scores)
            layer.attention.self.query.weight.mul_(8)
            layer.attention.self.key.weight.mul_(8)
    calls = Calls(monkeypatch)
    g = torch.Generator().manual_seed(L)
    lens = torch.tensor([L, 3, 1, L - 5, L // 2, 17])
    mask = torch.arange(L)[None] < lens[:, None]
    ids = torch.randint(1, 1000, (6, L), generator=g) * mask
    plan = BertModel.pack_plan(lens.tolist(), L, dev, m.pack_longest) if packed else None
    with torch.autocast('cuda', dtype=torch.bfloat16):
        h = m(ids.to(dev), attention_mask=mask.to(dev), cls_only=cls, pack=plan)['last_hidden_state']
    (h.float() * torch.randn(h.shape, generator=g).to(dev) * (1 if cls else mask[..., None].to(dev))).sum().backward()
    torch.cuda.synchronize()
    forms = [c['op'] for c in calls if c['op'] != 'dropout']
    long_form = 'relpos_attention_varlen' if packed else 'relpos_attention'
    assert forms == [long_form] * (3 if cls else 4) + ['relpos_attention_cls'] * int(cls)
    for i, c in enumerate(c for c in calls if c['op'] != 'dropout'):
        assert torch.equal(c['table'], m.encoder.relative_attention_bias.weight.detach()) and torch.equal(c['buckets'], m.encoder.relative_buckets)
        if packed:
            assert c['cu_seqlens'].tolist() == [0] + lens.cumsum(0).tolist() and c['max_len'] >= int(lens.max())
        else:
            assert torch.equal(c['key_mask'].cpu().reshape(6, L).bool(), mask)
        check_attention(c, 'layer %d' % i)
    (d,) = calls.of('dropout')
    check_dropout(d, 'embeddings')


def server(dev, half, cnn='resnet18'):
    from creamfl_amd.algorithms.retrieval_trainer import TrainerEngine
    from creamfl_amd.utils.config import default_config
    torch.manual_seed(0)
    cfg = default_config(embed_dim=64, cnn_type=cnn, not_bert=False)
    cfg.model.bert_name, cfg.model.image_norm = 'bert-mini-relative', 'group'
    eng = TrainerEngine(device=dev)
    eng.set_logger(SimpleNamespace(log=lambda *a: None, update_tracker=lambda *a, **k: None))
    eng.create(cfg, {'<pad>': 0}, None, False)
    eng.model_to_device()
    if half:
        eng.to_half()
    return eng


@pytest.mark.parametrize('cnn', ['resnet18', 'resnet50'])
def test_server_step_call_by_call(dev, monkeypatch, cnn):
    """One training step of the server in bf16, dropout on, its towers on two streams: all calls of the three operators, the gradients that
    the step's own backward gives them."""
    from creamfl_amd.utils.synthetic import coco_batch
    eng = server(dev, True, cnn)
    b = coco_batch(12, 'cpu', seed=5, bert=True, img=96)
    eng.model.train()
    calls = Calls(monkeypatch)
    loss, _ = eng.train_step(b[0].to(dev), b[1].to(dev), None, b[3])
    torch.cuda.synchronize()
    assert torch.isfinite(loss)
    gn, att, drop = calls.of('gn_act'), [c for c in calls if c['op'].startswith('relpos')], calls.of('dropout')
    assert len(gn) == {'resnet18': 20, 'resnet50': 53}[cnn] and len(att) == 4 and len(drop) == 1
    assert att[-1]['op'] == 'relpos_attention_cls' and all(c['d_out'] for c in gn + att + drop)
    for i, c in enumerate(gn):
        check_gn(c, 'gn %d' % i)
    for i, c in enumerate(att):
        check_attention(c, 'layer %d' % i)
    check_dropout(drop[0], 'embeddings')


def test_captured_step_call_by_call(dev, monkeypatch):
    """Forward and backward of the server's step -- two towers on two streams, group norm, relative positions, the criterion -- captured once and
    replayed on two batches in turn, with the program's own work between: what every captured call of the operators reads and gives in a replay is
    within its bounds.  (The step as a whole does not repeat itself to the bit, captured or not: the library's convolutions of small maps sum in a
    changing order.)"""
    from creamfl_amd import ops, streams
    from creamfl_amd.graphs import GraphedStep
    from creamfl_amd.utils.synthetic import coco_batch
    eng = server(dev, True)
    for mod in eng.model.modules():
        if isinstance(mod, torch.nn.Dropout):
            mod.p = 0.0
    eng.model.train()
    with torch.no_grad():
        eng.model.txt_enc.encoder.relative_attention_bias.weight.normal_()
    params = [p for p in eng.model.parameters() if p.requires_grad]
    calls = Calls(monkeypatch)
    batches = []
    for i in range(2):
        b = coco_batch(16, 'cpu', seed=70 + i, bert=True, img=64, min_len=24, max_len=24, index0=16 * i)
        cut = torch.tensor([24, 20, 24, 9] * 4).roll(i)        # (padding that the mask has to drop)
        caps = b[1] * (torch.arange(b[1].shape[1])[None] < cut[:, None])
        batches.append([b[0].to(dev).contiguous(memory_format=torch.channels_last), caps.to(dev), cut.to(dev)])

    def fn(images, captions, lens):
        for p in params:
            p.grad = None
        with ops.join_scope():
            loss, _ = eng.forward_loss(images, captions, None, lens, gather=False)
            eng.backward(loss)
        streams.join_into_current(dev)
        for p in params:
            p.grad = None
        return loss.detach()
    with torch.backends.cudnn.flags(enabled=True, benchmark=False):
        gs = GraphedStep(fn, warmup=2, guard_params=params)
        for k in (0, 1):
            gs(*batches[k], device=dev)
        assert gs.graph is None
        calls.clear()                                          # (from here on: the tensors of the captured step)
        seen = []
        for k in (0, 1, 1, 0):
            loss = gs(*batches[k], device=dev)
            torch.cuda.synchronize()
            torch.randn(1 << 20, device=dev).sort()            # (work of the program's own between replays)
            gn, att = calls.of('gn_act'), [c for c in calls if c['op'].startswith('relpos')]
            assert gs.failed is None and bool(torch.isfinite(loss)) and len(gn) == 20 and len(att) == 4
            for i, c in enumerate(gn):
                assert check_gn(c, 'replay on batch %d: gn %d' % (k, i)) >= 3
            lens = batches[k][2].cpu()
            for i, c in enumerate(att):
                assert torch.equal(c['key_mask'].cpu().reshape(16, -1).bool(), torch.arange(24)[None] < lens[:, None])
                check_attention(c, 'replay on batch %d: layer %d' % (k, i))
            seen.append((k, att[0]['d_qkv'].clone(), gn[0]['out'].clone()))
    assert gs.replays == 4
    for k, dqkv, y in seen[1:]:
        assert k == seen[0][0] or not (torch.equal(y, seen[0][2]) or torch.equal(dqkv, seen[0][1]))      # (another batch, other values)
