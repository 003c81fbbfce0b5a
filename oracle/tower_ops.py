"""CPU restatement, in 64 bits, of the encoder towers' operators: group normalisation with an activation, the keep flags of the
counter-based dropout, self-attention with a bucketed relative position bias.  Next to every result stands a bound on what a kernel that
rounds where it says it does may be off by (u16 = 2^-8: half a step of bf16 relative to the value; u32 = 2^-24)."""
import numpy as np
import torch

U16, U32 = 2.0 ** -8, 2.0 ** -24


def group_norm_act(x, gamma, beta, groups, eps=1e-5, act='none', residual=None, dy=None, bf16=False):
    """x, residual, dy: [N, C, H, W]; returns {name: (value, bound)} for y and, with dy, dx, dres, dgamma, dbeta.
    Bounds: the kernel's sums have at most 2^16 terms a thread and level and few levels, so a sum of n terms is off by less than 64 u32 of
    the sum of magnitudes; xh, z and the activation take a few more roundings of values of size |xh| + 1, |z| + 1."""
    x, gamma, beta = (t.detach().cpu().double() for t in (x, gamma, beta))
    n, c, h, w = x.shape
    m = c // groups * h * w
    xg = x.reshape(n, groups, m)
    mu = xg.mean(2, keepdim=True)
    var = ((xg - mu) ** 2).mean(2, keepdim=True)
    r = (var + eps) ** -0.5
    xh = ((xg - mu) * r).reshape(x.shape)
    # (the subtraction x - mu cancels: what the mean's own roundings leave counts relative to |x|, not to |x - mu|)
    exh = 64 * U32 * ((xg.abs() + xg.abs().mean(2, keepdim=True)) * r + 1).reshape(x.shape)
    ga, be = gamma[None, :, None, None], beta[None, :, None, None]
    z = xh * ga + be
    ez = exh * ga.abs() + 8 * U32 * (z.abs() + be.abs())
    if residual is not None:
        residual = residual.detach().cpu().double()
        z = z + residual
        ez = ez + 8 * U32 * residual.abs()
    if act == 'relu':
        y, dact, ddact = z.clamp(min=0), (z > 0).double(), 0.0
    elif act == 'silu':
        s = torch.sigmoid(z)
        y, dact, ddact = z * s, s * (1 + z * (1 - s)), 0.5
    else:
        y, dact, ddact = z, torch.ones_like(z), 0.0
    out_u = U16 if bf16 else U32
    res = {'y': (y, 1.1 * ez + 16 * U32 * y.abs() + out_u * y.abs() + 1e-30)}
    if dy is None:
        return res
    dy = dy.detach().cpu().double()
    dz = dy * dact
    edz = dy.abs() * (ddact * ez + 32 * U32)
    if act == 'relu':                                      # within the rounding of z the derivative is either of the two
        edz = torch.where(z.abs() <= ez, dy.abs(), edz)
    res['dres'] = (dz, edz + out_u * dz.abs() + 1e-30)
    res['dbeta'] = (dz.sum((0, 2, 3)), (edz + 64 * U32 * dz.abs()).sum((0, 2, 3)) + 1e-30)
    res['dgamma'] = ((dz * xh).sum((0, 2, 3)), (edz * xh.abs() + dz.abs() * exh + 64 * U32 * (dz * xh).abs()).sum((0, 2, 3)) + 1e-30)
    g, eg = dz * ga, edz * ga.abs() + 4 * U32 * (dz * ga).abs()

    def grp(t):
        return t.reshape(n, groups, m).mean(2, keepdim=True).expand(n, groups, m).reshape(x.shape)
    s1, s2 = grp(g), grp(g * xh)
    es1, es2 = grp(eg + 64 * U32 * g.abs()), grp(eg * xh.abs() + g.abs() * exh + 64 * U32 * (g * xh).abs())
    rr = r.expand(n, groups, m).reshape(x.shape)
    dx = rr * (g - s1 - xh * s2)
    edx = rr * (eg + es1 + es2 * xh.abs() + exh * s2.abs() + 64 * U32 * (g.abs() + s1.abs() + (xh * s2).abs()))
    res['dx'] = (dx, edx + out_u * dx.abs() + 1e-30)
    return res


def keep_flags(seed, p, n):
    """The flags of n elements (fewer than 2^33) for a 32-bit seed."""
    with np.errstate(over='ignore'):
        i = np.arange((n + 1) // 2, dtype=np.uint32)
        h = i * np.uint32(0x9E3779B1) ^ np.uint32(seed & 0xFFFFFFFF)
        h ^= h >> np.uint32(16)
        h *= np.uint32(0x85EBCA6B)
        h ^= h >> np.uint32(13)
        h *= np.uint32(0xC2B2AE35)
        h ^= h >> np.uint32(16)
    bits = np.stack([h & np.uint32(0xFFFF), h >> np.uint32(16)], 1).reshape(-1)[:n]
    return torch.from_numpy(bits.astype(np.int64) >= int(round(65536 * p)))


def relpos_attention_text(q, k, v, table, buckets, keep=None, scale=0.125, do=None, terms=1):
    """One text: q [Lq, heads, 64], k, v [Lk, heads, 64], table [nb, heads], buckets [2 R + 1], keep [Lk] flags.  Returns {name: (value,
    bound)} for o and, with do [Lq, heads, 64], dq, dk, dv and (in the bound without the output's own rounding) dtable.
    Bounds count: p (in `terms` bf16 terms where it meets v) and ds rounded to bf16 before they meet v, k, q, do; o rounded before D = do . o is formed (but for dtable); outputs rounded."""
    q, k, v, table = (t.detach().cpu().double() for t in (q, k, v, table))
    buckets = buckets.detach().cpu().long()
    lq, heads, hd = q.shape
    lk, R, nb = k.shape[0], buckets.numel() // 2, table.shape[0]
    keep = torch.ones(lk, dtype=torch.bool) if keep is None else keep.detach().cpu().bool()
    k, v = (torch.where(keep[:, None, None], t, torch.zeros_like(t)) for t in (k, v))
    which = buckets[(torch.arange(lk)[None] - torch.arange(lq)[:, None]).clamp(-R, R) + R].clamp(0, nb - 1)      # [Lq, Lk]
    qh, kh, vh = (t.permute(1, 0, 2) for t in (q, k, v))                                        # [heads, L, 64]
    drop = (table <= -1e30)[which].permute(2, 0, 1)         # a bias that low drops the key as the mask does
    table = torch.where(table <= -1e30, torch.zeros_like(table), table)
    s = scale * qh @ kh.transpose(1, 2) + table[which].permute(2, 0, 1)
    s = torch.where(keep[None, None] & ~drop, s, torch.full_like(s, -np.inf))
    p = torch.softmax(s, 2)
    p = torch.where(torch.isnan(p), torch.zeros_like(p), p) # a row without a key
    s = torch.where(torch.isinf(s), torch.zeros_like(s), s)
    # a score's 32-bit error moves p by its size: products of 64 terms, the bias, the log-sum
    es = 80 * U32 * (abs(scale) * qh.abs() @ kh.abs().transpose(1, 2) + table.abs().max() + s.abs() + 8)
    ep = p * (4 * es + 1e-6)
    o = p @ vh
    eo = (U16 ** terms * p + ep) @ vh.abs()

    def rows(t, extra=0.0):
        return t.permute(1, 0, 2)
    res = {'o': (rows(o), rows(1.02 * eo + U16 * o.abs() + 1e-30))}
    if do is None:
        return res
    g = do.detach().cpu().double().permute(1, 0, 2)
    dp = g @ vh.transpose(1, 2)
    edp = 80 * U32 * g.abs() @ vh.abs().transpose(1, 2)
    D = (p * dp).sum(2, keepdim=True)
    eD = (g.abs() * (1.02 * eo + U16 * o.abs())).sum(2, keepdim=True) + 80 * U32 * (g * o).abs().sum(2, keepdim=True)
    ds = p * (dp - D)
    eds = ep * (dp - D).abs() + p * (edp + eD)             # of ds in 32 bits
    er = eds + U16 * (ds.abs() + eds)                      # ... and rounded to bf16
    dq, dk, dv = scale * ds @ kh, scale * ds.transpose(1, 2) @ qh, p.transpose(1, 2) @ g
    edq, edk, edv = abs(scale) * er @ kh.abs(), abs(scale) * er.transpose(1, 2) @ qh.abs(), (U16 * p + ep).transpose(1, 2) @ g.abs()
    for name, t, e in (('dq', dq, edq), ('dk', dk, edk), ('dv', dv, edv)):
        res[name] = (rows(t), rows(1.02 * e + U16 * t.abs() + 1e-30))
    dt, et = torch.zeros(nb, heads, dtype=torch.float64), torch.zeros(nb, heads, dtype=torch.float64)
    dt.index_add_(0, which.reshape(-1), ds.permute(1, 2, 0).reshape(-1, heads))
    # the table's gradient adds up a whole row's error of D, so its D is held in 32 bits: sums of p dp over the row, and of ds with the rounded D
    eD = (p * edp + ep * dp.abs() + 80 * U32 * p * (dp.abs() + D.abs() + eD)).sum(2, keepdim=True)
    eds = ep * (dp - D).abs() + p * (edp + eD)
    et.index_add_(0, which.reshape(-1), (eds + 64 * U32 * ds.abs()).permute(1, 2, 0).reshape(-1, heads))
    res['dtable'] = (dt, et)
    return res
