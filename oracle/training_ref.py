"""Restatement in 64 bits of the training operators (otter_amd.training, otter_amd.inbatch.inbatch_loss) and, for each output,
a bound of how far a float32 computation with the documented roundings may be from it.

Bounds.  e = 2^-24 is float32's half step, u the output type's (bfloat16 2^-8, float32 e).  A sum of n products in float32, in
any order, is off by at most (n + 1) e sum |terms| to first order; an exponential 2^x of an x off by d is off by the relative
d ln 2 plus two half steps.  bfloat16 attention rounds the probabilities (dropped and kept) and dS to bfloat16 in front of the
matrix unit: u of each.  Every bound below is a sum of such terms over what the formula says, with SLACK for what is of second
order (products of errors) and a few half steps of the last operations."""
import math

import numpy as np
import torch

M32 = 0xFFFFFFFF
E32 = 2.0 ** -24
SLACK = 1.05


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------------------- draws
def philox(c0, c1, c2, c3, seed, rounds=7):
    """Philox4x32 of broadcast counters (numpy), [..., 4] uint64 words below 2^32."""
    c = [np.asarray(x, dtype=np.uint64) for x in np.broadcast_arrays(c0, c1, c2, c3)]
    k = [seed & M32, (seed >> 32) & M32]
    m32, s32 = np.uint64(M32), np.uint64(32)
    for _ in range(rounds):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> s32) ^ c[1] ^ np.uint64(k[0]), p1 & m32, (p0 >> s32) ^ c[3] ^ np.uint64(k[1]), p0 & m32]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return np.stack(c, -1)


def threshold(p):
    """Draws below it are dropped; p as the float32 the C interface takes."""
    return int(float(np.float32(p)) * 65536.0 + 0.5)


def _factor(draws, p):
    t = threshold(p)
    return torch.from_numpy(np.where(draws >= t, 65536.0 / (65536 - t), 0.0))


def row_factor(rows, cols, p, seed, call):
    """[rows, cols] float64: 0 where dropped, 1 / (1 - p) elsewhere."""
    if threshold(p) == 0:
        return torch.ones((rows, cols), dtype=torch.float64)
    col = np.arange(cols)
    w = philox((np.arange((cols + 7) // 8))[None, :], np.arange(rows)[:, None], M32, call, seed)      # [rows, groups, 4]
    word = w[:, col >> 3, (col & 7) >> 1]
    return _factor((word >> (16 * (col & 1)).astype(np.uint64)) & np.uint64(0xFFFF), p)


def score_factor(b, heads, n, p, seed, call):
    """[heads, n, n] float64 of sequence b."""
    if threshold(p) == 0:
        return torch.ones((heads, n, n), dtype=torch.float64)
    i, j = np.arange(n), np.arange(n)
    w = philox(np.arange((n + 3) // 4)[None, None, :], np.arange((n + 1) // 2)[None, :, None],
               (b * heads + np.arange(heads))[:, None, None], call, seed)
    word = w[:, (i >> 1)[:, None], (j >> 2)[None, :], (j & 3)[None, :]]
    return _factor((word >> (16 * (i & 1)).astype(np.uint64)[None, :, None]) & np.uint64(0xFFFF), p)


# --------------------------------------------------------------------------------------------------------- layer norm
def layer_norm(x, weight, bias, eps, residual, p, seed, call, dy, dtype, wdtype):
    """{name: (value, bound)} of y, mean, rstd, dx, dresidual, dweight, dbias; float64 [rows, cols] inputs."""
    R, C = x.shape
    f = row_factor(R, C, p, seed, call)
    res = torch.zeros_like(x) if residual is None else residual
    z = f * x + res
    mean = z.mean(1, keepdim=True)
    var = ((z - mean) ** 2).mean(1, keepdim=True)
    rstd = (var + eps) ** -0.5
    xh = (z - mean) * rstd
    a = dy * weight
    m1, m2 = a.mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
    dz = rstd * (a - m1 - xh * m2)
    out = {"y": xh * weight + bias, "mean": mean[:, 0], "rstd": rstd[:, 0], "dx": dz * f, "dresidual": dz,
           "dweight": (dy * xh).sum(0), "dbias": dy.sum(0)}
    # a row's sums: at most 64 additions in a row (32 elements a lane, the lanes, the waves), then a division
    N = 64
    ez = 3 * E32 * (f * x).abs() + E32 * z.abs()                                     # the factor, the product, the sum
    emean = ez.mean(1, keepdim=True) + (N + 2) * E32 * z.abs().mean(1, keepdim=True)
    edev = ez + emean + E32 * (z - mean).abs()
    # var: 2 |dev| edev averaged, its own sum; rstd: half the relative error of var + eps, root and division
    evar = 2 * ((z - mean).abs() * edev).mean(1, keepdim=True) + (edev ** 2).mean(1, keepdim=True) + (N + 4) * E32 * var
    rrstd = 0.5 * evar / (var + eps) + 4 * E32
    rrstd = torch.where(rrstd < 0.25, rrstd * (1 + 2 * rrstd), torch.full_like(rrstd, math.inf))
    exh = rstd * edev + xh.abs() * (rrstd + 2 * E32)
    u, uw = half_step(dtype), half_step(wdtype)
    y = out["y"]
    ey = exh * weight.abs() + 2 * E32 * ((xh * weight).abs() + bias.abs()) + E32 * y.abs()
    em1 = (N + 3) * E32 * a.abs().mean(1, keepdim=True)
    em2 = (a.abs() * exh).mean(1, keepdim=True) + (N + 4) * E32 * (a * xh).abs().mean(1, keepdim=True)
    inner = a.abs() + m1.abs() + (xh * m2).abs()
    edz = rstd * (em1 + exh * m2.abs() + xh.abs() * em2 + 4 * E32 * inner) + rrstd * dz.abs() + 2 * E32 * dz.abs()
    ew = (dy.abs() * exh).sum(0) + (R + 64) * E32 * (dy * xh).abs().sum(0)
    bounds = {"y": ey + u * y.abs(), "mean": emean[:, 0], "rstd": (rstd * rrstd)[:, 0],
              "dresidual": edz + u * dz.abs(), "dx": f * edz + 3 * E32 * out["dx"].abs() + u * out["dx"].abs(),
              "dweight": ew + uw * out["dweight"].abs(), "dbias": (R + 64) * E32 * dy.abs().sum(0) + uw * out["dbias"].abs()}
    return {k: (v, SLACK * bounds[k] + 1e-37) for k, v in out.items()}


# ---------------------------------------------------------------------------------------------------------- attention
def attention_sequence(q, k, v, key, p, seed, call, b, dout, scale, dtype):
    """One sequence, float64 [heads, n, 64]; key: bool [n].  {name: (value, bound)} of out, lse, dq, dk, dv."""
    H, n, D = q.shape
    even = not bool(key.any())
    u = half_step(dtype)
    ur = u if dtype == torch.bfloat16 else 0.0                      # rounding in front of the second products
    if not even:                                                    # keys left out reach nothing
        k = torch.where(key[None, :, None], k, torch.zeros_like(k))
        v = torch.where(key[None, :, None], v, torch.zeros_like(v))
        S = torch.matmul(q, k.transpose(1, 2)) * scale
        aS = torch.matmul(q.abs(), k.abs().transpose(1, 2)) * abs(scale)
        S = S.masked_fill(~key[None, None, :], -math.inf)
    else:
        S = torch.zeros((H, n, n), dtype=torch.float64)
        aS = torch.zeros_like(S)
    live = key if not even else torch.ones_like(key)
    f = score_factor(b, H, n, p, seed, call)
    lse = torch.logsumexp(S, 2)
    P = torch.exp(S - lse[:, :, None])
    W = P * f
    O = torch.matmul(W, v)
    fin = torch.where(live[None, None, :], S, torch.zeros_like(S)).abs()
    top = torch.maximum(fin.amax(2, keepdim=True), lse.abs()[:, :, None])
    eS = (D + 4) * E32 * aS                                                          # product, scale
    spread = (P * eS).sum(2, keepdim=True)
    # exponents are formed from the scaled score and the maximum or lse: three roundings of values up to `top`
    rP = eS + spread + (6 * top + n + 24) * E32
    elseb = spread[:, :, 0] + (4 * top[:, :, 0] + n + 24) * E32
    eO = torch.matmul(W * (rP + ur + 4 * E32), v.abs()) + (n + 4) * E32 * torch.matmul(W, v.abs())
    bO = eO + u * O.abs()
    res = {"out": (O, bO), "lse": (lse, elseb)}
    if dout is not None:
        dPd = torch.matmul(dout, v.transpose(1, 2))
        adP = torch.matmul(dout.abs(), v.abs().transpose(1, 2))
        delta = (dout * O).sum(2, keepdim=True)
        ed = (dout.abs() * bO).sum(2, keepdim=True) + (D + 2) * E32 * (dout * O).abs().sum(2, keepdim=True)
        zero = torch.zeros_like(P)
        dS = zero if even else torch.where(key[None, None, :], P * (f * dPd - delta), zero)
        mag = P * (f * dPd.abs() + delta.abs())
        edS = P * (f * (D + 4) * E32 * adP + ed) + mag * (rP + 4 * E32)
        edS = zero if even else torch.where(key[None, None, :], edS + ur * dS.abs(), zero)
        dq, dk = torch.matmul(dS, k) * scale, torch.matmul(dS.transpose(1, 2), q) * scale
        dv = torch.matmul(W.transpose(1, 2), dout)
        s = abs(scale)
        edq = s * (torch.matmul(edS, k.abs()) + (n + 4) * E32 * torch.matmul(dS.abs(), k.abs()))
        edk = s * (torch.matmul(edS.transpose(1, 2), q.abs()) + (n + 4) * E32 * torch.matmul(dS.abs().transpose(1, 2), q.abs()))
        edv = torch.matmul((W * (rP + ur + 4 * E32)).transpose(1, 2), dout.abs()) + (n + 4) * E32 * torch.matmul(W.transpose(1, 2), dout.abs())
        res.update(dq=(dq, edq + u * dq.abs()), dk=(dk, edk + u * dk.abs()), dv=(dv, edv + u * dv.abs()))
    return {name: (x, SLACK * e + 1e-37) for name, (x, e) in res.items()}


def attention(q, k, v, mask, cu, p, seed, call, dout, scale, dtype):
    """Whole tensors, laid out as the operator's: dense [B, L, H, 64] with mask [B, L] or None, packed [T, H, 64] with cu."""
    packed = cu is not None
    B = len(cu) - 1 if packed else q.shape[0]
    names = ("out", "dq", "dk", "dv") if dout is not None else ("out",)
    full = {n: [torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)] for n in names}
    H = q.shape[-2]
    shape = (H, q.shape[0]) if packed else (B, H, q.shape[1])
    full["lse"] = [torch.zeros(shape, dtype=torch.float64), torch.zeros(shape, dtype=torch.float64)]
    for b in range(B):
        at = slice(cu[b], cu[b + 1]) if packed else b
        n = cu[b + 1] - cu[b] if packed else q.shape[1]
        if n == 0:
            continue
        key = torch.ones(n, dtype=torch.bool) if mask is None else mask[b] != 0
        one = attention_sequence(*(t[at].transpose(0, 1).contiguous() for t in (q, k, v)), key, p, seed, call, b,
                                 None if dout is None else dout[at].transpose(0, 1).contiguous(), scale, dtype)
        for name, pair in one.items():
            for t, x in zip(full[name], pair):
                if name == "lse":
                    if packed:
                        t[:, at] = x
                    else:
                        t[b] = x
                else:
                    t[at] = x.transpose(0, 1)
    return {n: tuple(p) for n, p in full.items()}


# -------------------------------------------------------------------------------------------------------------- loss
def inbatch_loss(q, c, neg, dloss=1.0):
    """{name: (value, bound)} of loss, product, lse, dq, dc, dneg; float64 [B, d]."""
    B, d = q.shape
    S, aS = q @ c.t(), q.abs() @ c.abs().t()
    if neg is not None:
        S = torch.cat((S, (q * neg).sum(1, keepdim=True)), 1)
        aS = torch.cat((aS, (q * neg).abs().sum(1, keepdim=True)), 1)
    n = S.shape[1]
    lse = torch.logsumexp(S, 1)
    diag_out = S.clone()
    diag_out[:, :B].fill_diagonal_(-math.inf)
    rows = torch.nn.functional.softplus(torch.logsumexp(diag_out, 1) - torch.diagonal(S)) if n > 1 else torch.zeros(B, dtype=torch.float64)
    P = torch.exp(S - lse[:, None])
    eS = (d + 8) * E32 * aS
    spread = (P * eS).sum(1)
    top = torch.maximum(S.abs().amax(1), lse.abs())
    elseb = spread + (6 * top + n + 24) * E32
    erow = elseb + torch.diagonal(eS) + 2 * E32 * (lse.abs() + torch.diagonal(S).abs())
    g = dloss / B
    one = torch.zeros_like(P)
    one[:, :B] = torch.eye(B, dtype=torch.float64)
    # the diagonal is minus the sum of the other probabilities: no number near 1 is subtracted from 1, nor lse from the target's
    # score; each term's relative error is that of a difference of two scores (and of lse where the target is not the largest)
    off = torch.ones_like(P)
    off[:, :B] -= torch.eye(B, dtype=torch.float64)
    rest = (P * off).sum(1)
    rel = eS + elseb[:, None] + (6 * top[:, None] + 8) * E32
    diag = torch.diagonal(eS)
    erest = (P * off * rel).sum(1) + rest * (diag + (n + 24 + 6 * top) * E32)
    largest = torch.diagonal(S) >= S.masked_fill(off == 0, -math.inf).amax(1)
    erest = torch.where(largest, erest, erest + 4 * E32)
    erow = torch.where(largest, erest / (1 - rest).clamp(min=0.5) + 4 * E32 * rows, erow)
    G = P * off * g
    G[:, :B] -= torch.diag(rest) * g
    eG = abs(g) * P * off * (rel + 4 * E32)
    eG[:, :B] += torch.diag(erest + 4 * E32 * rest) * abs(g)
    out = {"loss": (rows.mean(), erow.mean() + 2 * E32 * rows.mean().abs()), "product": (S, eS), "lse": (lse, elseb),
           "rest": (rest, erest)}
    A, eA = G[:, :B], eG[:, :B]
    dq, edq = A @ c, eA @ c.abs() + (B + 4) * E32 * (A.abs() @ c.abs())
    out["dc"] = (A.t() @ q, eA.t() @ q.abs() + (B + 4) * E32 * (A.abs().t() @ q.abs()))
    if neg is not None:
        gn, en = G[:, B:], eG[:, B:]
        dq, edq = dq + gn * neg, edq + (en + 4 * E32 * gn.abs()) * neg.abs()
        out["dneg"] = (gn * q, (en + 4 * E32 * gn.abs()) * q.abs())
    out["dq"] = (dq, edq + 2 * E32 * dq.abs())
    return {name: (x, SLACK * e + 1e-37) for name, (x, e) in out.items()}
