"""The encoder towers' operators on the CPU: the oracle against differentiation and differences, the bucket map, refusals."""
import numpy as np
import pytest
import torch

from oracle import tower_ops as ref


@pytest.mark.parametrize('act', ['none', 'relu', 'silu'])
@pytest.mark.parametrize('residual', [False, True])
def test_oracle_group_norm_is_the_derivative(act, residual):
    g = torch.Generator().manual_seed(3)
    x, r, dy = (torch.randn(2, 12, 3, 5, generator=g, dtype=torch.float64) for _ in range(3))
    ga, be = 1 + 0.3 * torch.randn(12, generator=g, dtype=torch.float64), torch.randn(12, generator=g, dtype=torch.float64)
    got = ref.group_norm_act(x, ga, be, 4, act=act, residual=r if residual else None, dy=dy)
    leaves = [t.requires_grad_(True) for t in (x, ga, be, r)]
    z = torch.nn.functional.group_norm(x, 4, ga, be, 1e-5)
    z = z + r if residual else z
    y = {'none': lambda t: t, 'relu': torch.relu, 'silu': torch.nn.functional.silu}[act](z)
    want = torch.autograd.grad(y, leaves if residual else leaves[:3], dy)
    for name, t in zip(('dx', 'dgamma', 'dbeta', 'dres'), want):
        np.testing.assert_allclose(got[name][0].numpy(), t.numpy(), rtol=1e-9, atol=1e-11)
    np.testing.assert_allclose(got['y'][0].numpy(), y.detach().numpy(), rtol=1e-9, atol=1e-11)


def test_oracle_attention_is_the_derivative_and_the_difference():
    g = torch.Generator().manual_seed(4)
    lq, lk, heads = 5, 9, 2
    q = torch.randn(lq, heads, 64, generator=g, dtype=torch.float64)
    k, v = (torch.randn(lk, heads, 64, generator=g, dtype=torch.float64) for _ in range(2))
    do = torch.randn(lq, heads, 64, generator=g, dtype=torch.float64)
    table = torch.randn(6, heads, generator=g, dtype=torch.float64)
    buckets = torch.tensor([5, 0, 1, 2, 2, 3, 4], dtype=torch.int32)
    keep = torch.tensor([1, 1, 0, 1, 1, 1, 0, 1, 1], dtype=torch.bool)
    got = ref.relpos_attention_text(q, k, v, table, buckets, keep, 0.2, do)

    def value(q, k, v, table):
        which = buckets.long()[(torch.arange(lk)[None] - torch.arange(lq)[:, None]).clamp(-3, 3) + 3]
        s = torch.einsum('ihd,jhd->hij', q, k) * 0.2 + table[which].permute(2, 0, 1)
        return torch.einsum('hij,jhd->ihd', torch.softmax(s.masked_fill(~keep, -1e300), 2), v)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, table)]
    for name, t in zip(('dq', 'dk', 'dv', 'dtable'), torch.autograd.grad(value(*leaves), leaves, do)):
        np.testing.assert_allclose(got[name][0].numpy(), t.numpy(), rtol=1e-9, atol=1e-12)
    for i in (0, 2, 5):                                    # dtable against central differences (error of order h^2)
        h = 1e-4
        up, dn = table.clone(), table.clone()
        up[i, 1] += h
        dn[i, 1] -= h
        num = ((value(q, k, v, up) - value(q, k, v, dn)) * do).sum() / (2 * h)
        assert abs(float(num - got['dtable'][0][i, 1])) < 1e-6


def test_oracle_keep_flags_are_the_rate():
    k = ref.keep_flags(7, 0.25, 200001)
    assert k.shape == (200001,) and abs(float(k.double().mean()) - 0.75) < 5 * (0.25 * 0.75 / 200001) ** 0.5
    assert bool(ref.keep_flags(7, 0.0, 99).all()) and not bool(ref.keep_flags(7, 1.0, 99).any())


@pytest.mark.parametrize('nb,far', [(4, 2), (8, 16), (32, 128), (32, 512), (64, 100), (6, 40)])
def test_bucket_map(nb, far):
    from creamfl_amd import ops
    m = ops.relpos_buckets(nb, far).tolist()
    assert len(m) == 2 * far + 1 and m[far] == 0
    n = nb // 2
    assert [m[far + d] for d in range(1, n // 2)] == [n + d for d in range(1, n // 2)]             # single distances first
    for side in (m[:far + 1][::-1], [0] + [v - n for v in m[far + 1:]]):
        assert all(a <= b for a, b in zip(side, side[1:])) and side[-1] == n - 1                   # growing, up to the last one
        assert all(0 <= b < n for b in side)
    e = n // 2
    for a in range(e, far + 1):                            # the logarithm's formula, away from its borders
        exact = e + np.log(a / e) / np.log(far / e) * (n - e)
        if abs(exact - round(exact)) > 1e-6:
            assert m[far - a] == min(n - 1, int(exact))


@pytest.mark.parametrize('nb,far', [(3, 10), (2, 10), (32, 8), (32, 513), (0, 4)])
def test_bucket_map_refusals(nb, far):
    from creamfl_amd import _lib, ops
    with pytest.raises(_lib.CreamflHipError):
        ops.relpos_buckets(nb, far)


def test_ops_refuse_cpu_tensors():
    from creamfl_amd import _lib, ops
    x = torch.randn(2, 8, 3, 3).contiguous(memory_format=torch.channels_last)
    b = ops.relpos_buckets(4, 2)
    for call in (lambda: ops.gn_act(x, torch.ones(8), torch.zeros(8), 2), lambda: ops.dropout(x, 0.1),
                 lambda: ops.relpos_attention(torch.randn(1, 4, 192), torch.zeros(4, 1), b, 1),
                 lambda: ops.relpos_attention_varlen(torch.randn(4, 192), torch.tensor([0, 4], dtype=torch.int32), 4, torch.zeros(4, 1), b, 1),
                 lambda: ops.relpos_attention_cls(torch.randn(1, 64), torch.randn(1, 4, 128), torch.zeros(4, 1), b, 1)):
        with pytest.raises(_lib.CreamflHipError):
            call()
    assert not ops.gn_act_supported(x, 8, 2)


def test_entries_refuse_bad_arguments():
    """The C entries' own checks: each call ends in an error code before anything could be launched (there is no GPU here, and the
    pointers are no device memory)."""
    from creamfl_amd import _lib
    lib = _lib.load()
    P = 4096
    EINVAL, EALIGN, ELIMIT = -1, -2, -3

    def drop(x=P, dt=1, n=8, p=0.1, y=P):
        return lib.cfl_dropout(x, dt, n, p, 1, None, y, None, None)
    assert drop(x=None) == EINVAL and drop(y=None) == EINVAL and drop(dt=3) == EINVAL and drop(n=0) == EINVAL
    assert drop(p=-0.1) == EINVAL and drop(p=1.5) == EINVAL and drop(p=float('nan')) == EINVAL
    assert drop(x=P + 1) == EALIGN and drop(dt=0, y=P + 2) == EALIGN and drop(n=1 << 50) == ELIMIT

    def gn(x=P, gamma=P, dt=1, n=2, hw=9, c=16, g=4, eps=1e-5, act=1, y=P, mean=P, rstd=P, ws=P):
        return lib.cfl_gn_fwd(x, None, gamma, P, dt, n, hw, c, g, eps, act, y, mean, rstd, ws, None)
    for kw in (dict(x=None), dict(gamma=None), dict(dt=2), dict(n=0), dict(hw=0), dict(g=3), dict(g=0), dict(eps=-1.0), dict(act=3), dict(y=None),
               dict(rstd=None), dict(ws=None)):
        assert gn(**kw) == EINVAL, kw
    assert gn(x=P + 8) == EALIGN and gn(c=12, g=4) == ELIMIT and gn(c=2056, g=1) == ELIMIT and gn(n=70000) == ELIMIT
    assert lib.cfl_gn_bwd(None, None, P, None, P, P, P, P, 1, 2, 9, 16, 4, 1, 0, P, None, P, P, P, None) == EINVAL
    assert lib.cfl_gn_bwd(P, None, P, None, P, P, P, P, 1, 2, 9, 16, 4, 1, 1, P, None, P, P, P, None) == EINVAL      # dres wanted, none given
    assert lib.cfl_gn_ws_bytes(2, 9, 16, 3) == 0 and lib.cfl_gn_ws_bytes(2, 9, 16, 4) > 0

    def fwd(q=P, ldq=192, mask=None, cu=None, b=2, lq=4, lk=4, t=0, heads=1, hd=64, table=P, nb=4, bucket=P, r=2, o=P, ldo=64):
        return lib.cfl_relpos_fwd(q, ldq, P, P, 192, mask, cu, b, lq, lk, t, heads, hd, 0.125, table, 1, nb, bucket, r, o, ldo, None, None, None)
    for kw in (dict(q=None), dict(b=0), dict(lq=0), dict(lk=0), dict(heads=0), dict(table=None), dict(nb=0), dict(bucket=None), dict(r=-1),
               dict(o=None), dict(cu=P, t=0), dict(cu=P, t=8, mask=P)):
        assert fwd(**kw) == EINVAL, kw
    assert fwd(ldq=100) == EALIGN and fwd(q=P + 2) == EALIGN and fwd(ldo=66) == EALIGN and fwd(o=P + 8) == EALIGN
    assert fwd(hd=32) == ELIMIT and fwd(r=513) == ELIMIT and fwd(b=1 << 30) == ELIMIT and fwd(ldq=1 << 24) == ELIMIT
    assert fwd(heads=4) == EINVAL                          # (rows shorter than the heads)
    assert lib.cfl_relpos_bwd(P, 192, P, P, 192, None, None, 2, 4, 4, 0, 1, 64, 0.125, P, 1, 4, P, 2, P, P, 64, P, None, P, 192, P, P, 192, P, P,
                              None) == EINVAL
    assert lib.cfl_relpos_bwd_ws_bytes(0, 4, 4, 0, 1, 4, 2) == 0 and lib.cfl_relpos_bwd_ws_bytes(2, 0, 4, 8, 1, 4, 2) > 0
    assert lib.cfl_relpos_fwd_ws_bytes(1, 1, 4096, 0, 1) > 0 and lib.cfl_relpos_fwd_ws_bytes(64, 64, 64, 0, 12) == 0
    assert fwd(b=1, lq=1, lk=4096) == EINVAL               # (a split forward without its workspace)


# ------------------------------------------------------------------------------------------------ the towers that call them
def test_group_normed_trunk_on_the_library_path():
    from creamfl_amd.networks import backbones
    from creamfl_amd.networks.resnet_client import resnet18_client
    torch.manual_seed(0)
    m = backbones.resnet_trunk('resnet18', 'group')
    assert not any(isinstance(x, torch.nn.BatchNorm2d) for x in m.modules())
    y = m(torch.randn(2, 3, 64, 64))
    assert y.shape == (2, 512, 2, 2) and torch.isfinite(y).all()
    one = m(torch.randn(1, 3, 64, 64))
    assert one.shape == (1, 512, 2, 2)                     # (statistics per sample: a batch of one is a batch)
    y.sum().backward()
    assert all(p.grad is not None for p in m.parameters())
    assert backbones.resnet_trunk('resnet50', 'group').layer1[0].conv3.bn_follows is False
    assert backbones.resnet_trunk('resnet50').layer1[0].conv3.bn_follows is True
    c = resnet18_client(num_class=10, is_train=True, scale=128, embed_dim=512, norm='group')
    assert not any(isinstance(x, torch.nn.BatchNorm2d) for x in c.modules())
    with pytest.raises(ValueError):
        backbones.resnet_trunk('resnet18', 'layer')


def test_relative_bert_on_the_library_path():
    from creamfl_amd.networks.backbones import BertConfig, BertModel
    torch.manual_seed(1)
    m = BertModel('bert-mini-relative').eval()
    assert not any('position_embeddings' in n for n, _ in m.named_parameters())
    ids = torch.randint(1, 1000, (3, 40))
    mask = torch.arange(40)[None] < torch.tensor([40, 9, 23])[:, None]
    out = m(ids, attention_mask=mask)['last_hidden_state']
    cls = m(ids, attention_mask=mask, cls_only=True)['last_hidden_state']
    np.testing.assert_allclose(cls[:, 0].detach().numpy(), out[:, 0].detach().numpy(), rtol=1e-4, atol=1e-5)
    shorter = m(ids[1:2, :9])['last_hidden_state']         # padding changes nothing for the real tokens
    np.testing.assert_allclose(shorter[0].detach().numpy(), out[1, :9].detach().numpy(), rtol=1e-4, atol=1e-5)
    out.square().sum().backward()
    assert float(m.encoder.relative_attention_bias.weight.grad.abs().max()) > 0
    assert m(torch.randint(1, 1000, (1, 700)))['last_hidden_state'].shape == (1, 700, 256)         # longer than any position table
    assert BertModel('bert-mini').pack_longest == 32 and m.pack_longest > 700
    with pytest.raises(ValueError):
        BertConfig(position_embedding_type='rotary')


def test_flags_reach_the_models():
    import argparse
    from creamfl_amd import flags
    from creamfl_amd.networks.models import get_model
    from creamfl_amd.utils.config import default_config
    ns = flags.add_build_flags(argparse.ArgumentParser()).parse_args(['--image_norm', 'group', '--bert_name', 'bert-mini-relative'])
    assert flags.get(ns, 'image_norm') == 'group' and flags.get(argparse.Namespace(), 'image_norm') == 'batch'
    cfg = default_config(embed_dim=64, cnn_type='resnet18')
    cfg.model.image_norm, cfg.model.bert_name = ns.image_norm, ns.bert_name
    m = get_model({'<pad>': 0}, cfg.model, False)
    assert not any(isinstance(x, torch.nn.BatchNorm2d) for x in m.img_enc.modules())
    assert m.txt_enc.config.position_embedding_type == 'relative_bucket'
