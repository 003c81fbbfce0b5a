"""What is measured of the operators for the encoder towers: group normalisation with an activation on channels_last feature maps,
dropout from a counter-based generator, and self-attention with a learned relative position bias by buckets.

A case names one operator ("op"), its sizes and its direction ("train": forward and backward, else forward alone).  `run` computes the
plain form -- elementary torch operations in 32 bits, rounded once -- or, where `own` is true, calls creamfl_amd.ops."""
import math
import random

import numpy as np
import torch

own = False

HEAD_DIM = 64                        # every BERT / ViT configuration of this repository
NUM_BUCKETS, MAX_DISTANCE = 32, 128  # generic: 32 buckets, logarithmic up to a distance of 128 tokens
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one image through the last stage of a bottleneck trunk: block output with its residual, evaluation (latency)
        dict(name='gn_eval_one_image', op='gn', n=1, c=2048, h=7, w=7, groups=32, dtype='bf16', act='relu', residual=True, train=False),
        # the last stage of a client's encoder on two images, fp32 like the clients' training, ReLU (latency)
        dict(name='gn_train_two_images', op='gn', n=2, c=512, h=7, w=7, groups=32, dtype='fp32', act='relu', residual=True, train=True),
        # a client's batch of 128 at the second stage, fp32
        dict(name='gn_train_client', op='gn', n=128, c=128, h=28, w=28, groups=32, dtype='fp32', act='silu', residual=False, train=True),
        # the server's batch of 256 at the first bottleneck stage's block output, bf16: the largest
        dict(name='gn_train_server', op='gn', n=256, c=256, h=56, w=56, groups=32, dtype='bf16', act='silu', residual=True, train=True),
        # the embeddings of one caption through dropout (latency)
        dict(name='dropout_one_caption', op='dropout', rows=24, cols=256, dtype='bf16', p=0.1, train=True),
        # the embeddings of a batch of 256 texts of 512 tokens, base width
        dict(name='dropout_batch', op='dropout', rows=131072, cols=768, dtype='bf16', p=0.1, train=True),
        # one caption of 17 tokens through the mini tower, retrieval at serving time (latency)
        dict(name='attn_one_caption', op='attn', b=1, l=17, heads=4, form='padded', lens_seed=0, train=False),
        # a batch of 256 captions of 8 to 32 tokens, packed, base width: the text tower's training step
        dict(name='attn_captions', op='attn', b=256, l=32, heads=12, form='packed', lens_seed=1, train=True),
        # 24 texts of odd length with padding, three heads
        dict(name='attn_odd', op='attn', b=24, l=197, heads=3, form='padded', lens_seed=2, train=True),
        # 32 paragraphs of up to the position table's 512 tokens, base width
        dict(name='attn_paragraphs', op='attn', b=32, l=512, heads=12, form='padded', lens_seed=3, train=True),
        # two long documents
        dict(name='attn_documents', op='attn', b=2, l=4096, heads=12, form='packed', lens_seed=0, train=True),
        # the last layer's single query per text ([CLS]) over 512 tokens, evaluation
        dict(name='attn_cls', op='attn', b=128, l=512, heads=12, form='cls', lens_seed=4, train=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(('gn', 'gn', 'dropout', 'attn', 'attn', 'cls'))
    train = rng.random() < 0.7
    if kind == 'gn':
        while True:
            cpg, groups = rng.choice((1, 2, 3, 4, 5, 8, 12, 16, 32, 64)), rng.choice((1, 4, 8, 16, 24, 32, 40))
            n, h, w = _log_int(rng, 1, 256), _log_int(rng, 1, 112), _log_int(rng, 1, 112)
            c = cpg * groups
            # (groups of a handful of values make the gradient a difference of nearly equal numbers, and 32 bits say nothing)
            if c % 8 == 0 and c <= 2048 and cpg * h * w >= 48 and n * c * h * w <= 64_000_000:
                break
        # ReLU's derivative jumps at its border: over millions of values some lie within 32 bits' rounding of it, so the
        # trained ReLU is drawn on small maps
        acts = ['none', 'silu'] + (['relu'] if not train or n * c * h * w <= 60_000 else [])
        return dict(op='gn', n=n, c=c, h=h, w=w, groups=groups, dtype=rng.choice(('bf16', 'fp32')), act=rng.choice(acts),
                    residual=rng.random() < 0.5, train=train)
    if kind == 'dropout':
        cols = rng.choice((1, 3, 64, 100, 256, 301, 768, 1000, 1024, 2047, 4096))
        return dict(op='dropout', rows=_log_int(rng, 1, 50_000_000 // cols), cols=cols, dtype=rng.choice(('bf16', 'fp16', 'fp32')),
                    p=rng.choice((0.0, 0.05, 0.1, 0.25, 0.5, 0.9)), train=train)
    heads = rng.choice((1, 3, 4, 8, 12))
    l = _log_int(rng, 1, 4096)
    b = _log_int(rng, 1, max(1, min(512, int(4e8 / (heads * l * l)) if kind == 'attn' else int(1.2e8 / (heads * l * HEAD_DIM)))))
    return dict(op='attn', b=b, l=l, heads=heads, form='cls' if kind == 'cls' else rng.choice(('padded', 'packed')),
                lens_seed=rng.choice((0, rng.randint(1, 10 ** 6))), train=train)


def _lens(case):
    """The texts' lengths: all `l` for lens_seed 0, else between a quarter and all of it; one text in sixteen is empty."""
    b, l = case['b'], case['l']
    if not case['lens_seed']:
        return [l] * b
    r = random.Random(case['lens_seed'])
    lens = [r.randint(max(1, l // 4), l) for _ in range(b)]
    for i in range(15, b, 16):
        lens[i] = 0
    lens[0] = l
    return lens


def work(case):
    if case['op'] == 'gn':
        e = case['n'] * case['c'] * case['h'] * case['w']
        size = DTYPES[case['dtype']].itemsize
        r = int(case['residual'])
        moved = e * size * (2 + r + ((2 + r) if case['train'] else 0)) + 4 * case['c'] * (4 if case['train'] else 2)
        return {'bytes': moved, 'flops': e * (24 if case['train'] else 8)}
    if case['op'] == 'dropout':
        e = case['rows'] * case['cols']
        return {'bytes': e * DTYPES[case['dtype']].itemsize * (4 if case['train'] else 2), 'flops': e * (2 if case['train'] else 1)}
    lens, h, l = _lens(case), case['heads'], case['l']
    width = h * HEAD_DIM
    table = 2 * NUM_BUCKETS * h
    if case['form'] == 'cls':
        rows = sum(lens) if case['train'] else sum(lens)
        pairs = sum(lens)
        moved = 2 * width * (2 * len(lens) + 2 * rows) + table
        if case['train']:
            moved += 2 * width * (2 * len(lens) + 2 * len(lens) * l) + table
    else:
        tokens = sum(lens) if case['form'] == 'packed' else len(lens) * l
        pairs = sum(n * n for n in lens) if case['form'] == 'packed' else sum(n * l for n in lens)
        moved = 2 * width * 4 * tokens + table
        if case['train']:
            moved += 2 * width * 4 * tokens + table
    return {'bytes': moved, 'flops': pairs * h * HEAD_DIM * (14 if case['train'] else 4)}


# ------------------------------------------------------------------------------------------------ inputs
def _bucket_map():
    """int32 [2 R + 1]: the bucket of the clipped distance d = key - query, at place d + R.  Half of the buckets are for keys behind the
    query; of a half, the first half are single distances and the others grow geometrically up to MAX_DISTANCE.  Borders by whole
    numbers: |d| belongs to bucket k or above where (|d| / e)^(n - e) >= (MAX_DISTANCE / e)^(k - e)."""
    n = NUM_BUCKETS // 2
    e = n // 2

    def one(d):
        a, off = abs(d), n if d > 0 else 0
        if a < e:
            return off + a
        k = e
        while k + 1 < n and a ** (n - e) * e ** (k + 1 - e) >= MAX_DISTANCE ** (k + 1 - e) * e ** (n - e):
            k += 1
        return off + k
    return torch.tensor([one(d) for d in range(-MAX_DISTANCE, MAX_DISTANCE + 1)], dtype=torch.int32)


def prepare(case, seed):
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(int(seed))
    if case['op'] == 'gn':
        dt = DTYPES[case['dtype']]
        n, c, h, w = case['n'], case['c'], case['h'], case['w']

        def fmap(scale, shift=0.0):
            t = torch.empty((n, c, h, w), dtype=dt, device=dev, memory_format=torch.channels_last)
            return t.normal_(shift, scale, generator=g)
        s = dict(case=case, x=fmap(1.5, 0.3), gamma=1 + 0.2 * torch.randn(c, generator=g, device=dev),
                 beta=0.2 * torch.randn(c, generator=g, device=dev), res=fmap(1.0) if case['residual'] else None)
        s['dy'] = fmap(1.0) if case['train'] else None
        return s
    if case['op'] == 'dropout':
        dt = DTYPES[case['dtype']]
        shape = (case['rows'], case['cols'])
        s = dict(case=case, x=torch.empty(shape, dtype=dt, device=dev).normal_(generator=g), seed=(int(seed) * 2654435761 + 12345) & 0xffffffff)
        s['dy'] = torch.empty(shape, dtype=dt, device=dev).normal_(generator=g) if case['train'] else None
        return s
    b, l, h = case['b'], case['l'], case['heads']
    lens = _lens(case)
    width = h * HEAD_DIM

    def act(*shape):
        return torch.empty(shape, dtype=torch.bfloat16, device=dev).normal_(generator=g)
    s = dict(case=case, buckets=_bucket_map().to(dev), table=torch.empty((NUM_BUCKETS, h), dtype=torch.bfloat16, device=dev).normal_(generator=g))
    lengths = torch.tensor(lens)
    if case['form'] == 'packed':
        t = sum(lens)
        s['qkv'] = act(t, 3 * width)
        s['do'] = act(t, width)
        s['cu'] = torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]).to(torch.int32).to(dev)
    else:
        s['mask'] = (torch.arange(l)[None, :] < lengths[:, None]).to(dev)
        if case['form'] == 'cls':
            s['q'], s['kv'], s['do'] = act(b, width), act(b, l, 2 * width), act(b, width)
        else:
            s['qkv'], s['do'] = act(b, l, 3 * width), act(b, l, width)
    return s


# ------------------------------------------------------------------------------------------------ group norm
def _gn_plain(s):
    c = s['case']
    n, ch, h, w, gr = c['n'], c['c'], c['h'], c['w'], c['groups']
    x = s['x'].permute(0, 2, 3, 1).reshape(n, h * w, gr, ch // gr).float()
    gamma, beta = s['gamma'].view(gr, ch // gr), s['beta'].view(gr, ch // gr)
    m = h * w * (ch // gr)
    mu = x.sum((1, 3), keepdim=True) / m
    xc = x - mu
    r = 1.0 / torch.sqrt((xc * xc).sum((1, 3), keepdim=True) / m + 1e-5)
    xh = xc * r
    z = xh * gamma + beta
    if s['res'] is not None:
        z = z + s['res'].permute(0, 2, 3, 1).reshape(z.shape).float()

    def out(t):
        return t.to(s['x'].dtype).reshape(n, h, w, ch).permute(0, 3, 1, 2)
    if c['act'] == 'relu':
        y = torch.where(z > 0, z, torch.zeros_like(z))
    elif c['act'] == 'silu':
        sg = 1.0 / (1.0 + torch.exp(-z))
        y = z * sg
    else:
        y = z
    if not c['train']:
        return [out(y)]
    dz = s['dy'].permute(0, 2, 3, 1).reshape(z.shape).float()
    if c['act'] == 'relu':
        dz = torch.where(z > 0, dz, torch.zeros_like(dz))
    elif c['act'] == 'silu':
        dz = dz * (sg * (1.0 + z * (1.0 - sg)))
    dbeta = dz.sum(1).double().sum(0).float().reshape(ch)
    dgamma = (dz * xh).sum(1).double().sum(0).float().reshape(ch)
    gg = dz * gamma
    s1 = gg.sum((1, 3), keepdim=True) / m
    s2 = (gg * xh).sum((1, 3), keepdim=True) / m
    dx = r * (gg - s1 - xh * s2)
    got = [out(y), out(dx), dgamma, dbeta]
    return got + [out(dz)] if s['res'] is not None else got


def _gn_own(s):
    from creamfl_amd import ops, runtime
    c = s['case']
    if not c['train']:
        with torch.no_grad():
            return [ops.gn_act(s['x'], s['gamma'], s['beta'], c['groups'], act=c['act'], residual=s['res'])]
    leaves = [s[k].detach().requires_grad_(True) for k in ('x', 'gamma', 'beta', 'res') if s[k] is not None]
    y = ops.gn_act(leaves[0], leaves[1], leaves[2], c['groups'], act=c['act'], residual=leaves[3] if s['res'] is not None else None)
    with runtime.backward_here():                              # (the framework's steps run their backward on the calling thread)
        return [y.detach(), *torch.autograd.grad(y, leaves, s['dy'])]


def _gn_exact(s):
    """A few images at a time, from the definition, gradients by differentiation."""
    c = s['case']
    n, ch, h, w = c['n'], c['c'], c['h'], c['w']
    gamma, beta = (s[k].double().requires_grad_(c['train']) for k in ('gamma', 'beta'))
    per = max(1, 8_000_000 // (ch * h * w))
    parts, dgamma, dbeta = [], torch.zeros_like(gamma), torch.zeros_like(beta)
    for i in range(0, n, per):
        x = s['x'][i:i + per].double().contiguous().requires_grad_(c['train'])
        var, mean = torch.var_mean(x.view(x.shape[0], c['groups'], -1), 2, correction=0, keepdim=True)
        z = ((x.view(x.shape[0], c['groups'], -1) - mean) * torch.rsqrt(var + 1e-5)).view(x.shape)
        z = z * gamma[None, :, None, None] + beta[None, :, None, None]
        leaves = [x, gamma, beta]
        if s['res'] is not None:
            leaves.append(s['res'][i:i + per].double().contiguous().requires_grad_(c['train']))
            z = z + leaves[3]
        y = z.clamp(min=0) if c['act'] == 'relu' else torch.nn.functional.silu(z) if c['act'] == 'silu' else z
        part = [y.detach()]
        if c['train']:
            got = torch.autograd.grad(y, leaves, s['dy'][i:i + per].double().contiguous())
            dgamma += got[1]
            dbeta += got[2]
            part += [got[0], *got[3:]]
        parts.append(part)
    whole = [torch.cat(v) for v in zip(*parts)]
    return whole if not c['train'] else [whole[0], whole[1], dgamma, dbeta, *whole[2:]]


# ------------------------------------------------------------------------------------------------ dropout
def _keep(seed, n, p, device):
    """Element e is kept where 16 random bits are at least 65536 p: the low or high half (e even / odd) of a 32-bit mix of the seed and
    the pair's number e / 2."""
    def mul(a, m):
        return (a * m) & 0xffffffff
    i = torch.arange((n + 1) // 2, device=device)
    h = mul(i & 0xffffffff, 0x9E3779B1) ^ ((seed + (i >> 32) * 0x632BE5AB) & 0xffffffff)
    h = mul(h ^ (h >> 16), 0x85EBCA6B)
    h = mul(h ^ (h >> 13), 0xC2B2AE35)
    h = h ^ (h >> 16)
    bits = torch.stack([h & 0xffff, h >> 16], 1).reshape(-1)[:n]
    return bits >= int(round(65536 * p))


def _dropout_plain(s):
    c = s['case']
    p = int(round(65536 * c['p'])) / 65536
    keep = _keep(s['seed'], s['x'].numel(), c['p'], s['x'].device).view(s['x'].shape)

    def drop(t):
        t32 = t.float()
        return torch.where(keep, t32 * (1.0 / (1.0 - p)), torch.zeros_like(t32)).to(t.dtype)
    return [drop(s['x']), drop(s['dy'])] if c['train'] else [drop(s['x'])]


def _dropout_own(s):
    from creamfl_amd import ops, runtime
    c = s['case']
    if not c['train']:
        with torch.no_grad():
            return [ops.dropout(s['x'], c['p'], seed=s['seed'])]
    x = s['x'].detach().requires_grad_(True)
    y = ops.dropout(x, c['p'], seed=s['seed'])
    with runtime.backward_here():
        return [y.detach(), *torch.autograd.grad(y, [x], s['dy'])]


def _dropout_exact(s):
    c = s['case']
    n = s['x'].numel()
    with np.errstate(over='ignore'):
        i = np.arange((n + 1) // 2, dtype=np.uint32)          # (fewer than 2^33 elements in every case)
        h = i * np.uint32(0x9E3779B1) ^ np.uint32(s['seed'])
        h ^= h >> np.uint32(16)
        h *= np.uint32(0x85EBCA6B)
        h ^= h >> np.uint32(13)
        h *= np.uint32(0xC2B2AE35)
        h ^= h >> np.uint32(16)
    thr = int(round(65536 * c['p']))
    keep = torch.from_numpy(np.ascontiguousarray(h).view(np.uint16)[:n] >= thr).to(s['x'].device).view(s['x'].shape)
    factor = 65536.0 / (65536 - thr)
    return [t.double() * keep * factor for t in ([s['x'], s['dy']] if c['train'] else [s['x']])]


# ------------------------------------------------------------------------------------------------ attention
def _attn_plain(s):
    c = s['case']
    b, l, h = c['b'], c['l'], c['heads']
    width, scale = h * HEAD_DIM, 1.0 / math.sqrt(HEAD_DIM)
    packed, cls = c['form'] == 'packed', c['form'] == 'cls'
    dev = s['table'].device

    def heads_of(t):                                           # [B, n, H] -> [B, heads, n, 64] in 32 bits
        return t.view(b, -1, h, HEAD_DIM).transpose(1, 2).float().contiguous()
    if packed:
        cu = s['cu'].long()
        place = torch.arange(l, device=dev)[None, :]
        keep = place < (cu[1:] - cu[:-1])[:, None]             # [B, L]
        flat = (cu[:-1, None] + place)[keep]                   # rows of the packed tensors, in order

        def padded(t):
            p = torch.zeros((b, l, t.shape[-1]), dtype=t.dtype, device=dev)
            p[keep] = t[flat]
            return p
        qkv, do = padded(s['qkv']), padded(s['do'])
        q, k, v = qkv[..., :width], qkv[..., width:2 * width], qkv[..., 2 * width:]
    elif cls:
        keep, do, q = s['mask'], s['do'], s['q']
        k, v = s['kv'][..., :width], s['kv'][..., width:]
    else:
        keep, do = s['mask'], s['do']
        q, k, v = s['qkv'][..., :width], s['qkv'][..., width:2 * width], s['qkv'][..., 2 * width:]
    q, k, v, do = heads_of(q.contiguous()), heads_of(k.contiguous()), heads_of(v.contiguous()), heads_of(do.contiguous())
    lq = q.shape[2]
    dist = torch.arange(l, device=dev)[None, :] - torch.arange(lq, device=dev)[:, None]
    which = s['buckets'].long()[dist.clamp(-MAX_DISTANCE, MAX_DISTANCE) + MAX_DISTANCE]        # [Lq, L]
    bias = s['table'].float()[which].permute(2, 0, 1)
    sc = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale + bias
    sc = sc.masked_fill(~keep[:, None, None, :], -math.inf)
    top = sc.amax(3, keepdim=True).clamp(min=-3e38)
    p = torch.exp(sc - top)
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p, v)

    def rows(t):                                               # back to token rows, rounded once
        t = t.transpose(1, 2).reshape(b, -1, width)
        t = t[keep] if packed else t[:, 0] if cls and t.shape[1] == 1 else t
        return t.to(torch.bfloat16)
    if not c['train']:
        return [rows(o)]
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (dp - (p * dp).sum(3, keepdim=True))
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    # sums along the diagonals: rows in reverse order, each padded to 2 L and cut one value short, stand one place further right
    t = ds.double().sum(0).flip(1) if lq * l <= 1 << 20 else ds.sum(0).flip(1)
    t = torch.cat([t, torch.zeros((h, lq, lq), dtype=t.dtype, device=dev)], 2).reshape(h, -1)[:, :lq * (l + lq - 1)]
    diag = t.reshape(h, lq, l + lq - 1).double().sum(1)       # place d + Lq - 1
    d = torch.arange(l + lq - 1, device=dev) - (lq - 1)
    hot = s['buckets'].long()[d.clamp(-MAX_DISTANCE, MAX_DISTANCE) + MAX_DISTANCE][:, None] == torch.arange(NUM_BUCKETS, device=dev)
    dtable = torch.matmul(diag, hot.double()).t().to(torch.bfloat16)
    if cls:
        dkv = torch.cat([dk.transpose(1, 2).reshape(b, l, width), dv.transpose(1, 2).reshape(b, l, width)], 2).to(torch.bfloat16)
        return [rows(o), rows(dq), dkv, dtable]
    return [rows(o), torch.cat([rows(dq), rows(dk), rows(dv)], -1), dtable]


def _attn_own(s):
    from creamfl_amd import ops, runtime
    c = s['case']
    names = ('q', 'kv', 'table') if c['form'] == 'cls' else ('qkv', 'table')
    leaves = [s[k].detach().requires_grad_(c['train']) for k in names]
    if c['form'] == 'cls':
        o = ops.relpos_attention_cls(leaves[0], leaves[1], leaves[2], s['buckets'], c['heads'], key_mask=s['mask'])
    elif c['form'] == 'packed':
        o = ops.relpos_attention_varlen(leaves[0], s['cu'], c['l'], leaves[1], s['buckets'], c['heads'])
    else:
        o = ops.relpos_attention(leaves[0], leaves[1], s['buckets'], c['heads'], key_mask=s['mask'])
    if not c['train']:
        return [o]
    with runtime.backward_here():
        return [o.detach(), *torch.autograd.grad(o, leaves, s['do'])]


def _attn_exact(s):
    """Text by text, from the definition, gradients by differentiation."""
    c = s['case']
    h, width = c['heads'], c['heads'] * HEAD_DIM
    cls, packed = c['form'] == 'cls', c['form'] == 'packed'
    table = s['table'].double().requires_grad_(c['train'])
    where = s['buckets'].long()
    outs, grads, dtable = [], [], torch.zeros_like(table)
    at = 0
    for i, n in enumerate(_lens(c)):
        src = (s['qkv'][at:at + n] if packed else s['kv'][i] if cls else s['qkv'][i]).double().requires_grad_(c['train'])
        qs = s['q'][i:i + 1].double().requires_grad_(c['train']) if cls else src
        do = (s['do'][at:at + n] if packed else s['do'][i:i + 1] if cls else s['do'][i]).double()
        at += n
        lead = 0 if cls else width
        q = qs[:, :width].reshape(-1, h, HEAD_DIM).permute(1, 0, 2)
        k = src[:n, lead:lead + width].reshape(-1, h, HEAD_DIM).permute(1, 2, 0)
        v = src[:n, lead + width:].reshape(-1, h, HEAD_DIM).permute(1, 0, 2)
        off = torch.arange(n, device=table.device)[None] - torch.arange(q.shape[1], device=table.device)[:, None]
        a = torch.softmax(q @ k / 8.0 + table.t()[:, where[off.clamp(-MAX_DISTANCE, MAX_DISTANCE) + MAX_DISTANCE]], 2)
        o = (a @ v).permute(1, 0, 2).reshape(-1, width)        # (no keys: an empty sum, zero)
        outs.append(o.detach())
        if c['train']:
            got = torch.autograd.grad(o, [qs, src, table] if cls else [src, table], do)
            grads.append(got[:-1])
            dtable += got[-1]
        del a, o
    join = torch.cat if packed or cls else torch.stack
    res = [join(outs)]
    if c['train']:
        res.append(join([x[0] for x in grads]))
        if cls:
            res.append(torch.stack([x[1] for x in grads]))
        res.append(dtable)
    return res


# ------------------------------------------------------------------------------------------------ entry points
def run(state):
    op = state['case']['op']
    if own:
        return _gn_own(state) if op == 'gn' else _dropout_own(state) if op == 'dropout' else _attn_own(state)
    return _gn_plain(state) if op == 'gn' else _dropout_plain(state) if op == 'dropout' else _attn_plain(state)


def exact(case, seed):
    s = prepare(case, seed)
    return _gn_exact(s) if case['op'] == 'gn' else _dropout_exact(s) if case['op'] == 'dropout' else _attn_exact(s)
