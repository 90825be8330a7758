"""What the training operators of the bi-encoder are timed on: attention, layer norm of a sum, dropout and the in-batch
loss, each with its backward pass, as cases with inputs, a plain form in elementary torch operations and the exact values.

`own` False: `run` is the plain form (float32, rounded once at the end).  `own` True: `run` calls the framework.

Random numbers: Philox4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw 2011), the key is a 64-bit seed, one call makes eight
draws of 16 bits; a value is dropped where its draw is below T = round(65536 p) and scaled by 65536 / (65536 - T) elsewhere.
  rows       counter (col >> 3, row, 0xFFFFFFFF, call), draw of col:   word (col & 7) >> 1, low half for even col
  attention  counter (j >> 2, i >> 1, b * heads + h, call), draw of query i, key j: word j & 3, low half for even i
"""
import math

import torch

own = False

_M = 0xFFFFFFFF
_HEAD = 64
_CALL = 5


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # fine-tuning on table-text blocks: the layer's attention at the usual batch, blocks padded to 512 tokens
        {"name": "attention-blocks", "op": "attention", "dtype": "bf16", "layout": "dense", "B": 16, "L": 512, "heads": 12,
         "p": 0.1, "train": True, "ragged": True},
        # the question side of the same step: short sequences, where a call's own cost counts
        {"name": "attention-questions", "op": "attention", "dtype": "bf16", "layout": "dense", "B": 16, "L": 70, "heads": 12,
         "p": 0.1, "train": True, "ragged": True},
        # the float32 path, held against the reference's numbers
        {"name": "attention-float32", "op": "attention", "dtype": "f32", "layout": "dense", "B": 8, "L": 512, "heads": 12,
         "p": 0.1, "train": True, "ragged": True},
        # a large batch without its padding: sequences back to back
        {"name": "attention-packed", "op": "attention", "dtype": "bf16", "layout": "packed", "B": 128, "L": 512, "heads": 12,
         "p": 0.1, "train": True, "ragged": True},
        # long documents, evaluation only: no dropout, no gradient, an odd length
        {"name": "attention-long-forward", "op": "attention", "dtype": "bf16", "layout": "dense", "B": 2, "L": 4001,
         "heads": 12, "p": 0.0, "train": False, "ragged": False},
        # the residual layer norm of the question side
        {"name": "norm-questions", "op": "norm", "dtype": "bf16", "rows": 1120, "cols": 768, "p": 0.1, "residual": True},
        # the residual layer norm of 128 blocks of 512 tokens
        {"name": "norm-blocks", "op": "norm", "dtype": "bf16", "rows": 65536, "cols": 768, "p": 0.1, "residual": True},
        # a plain layer norm in float32 over rows whose length is no multiple of anything
        {"name": "norm-odd-float32", "op": "norm", "dtype": "f32", "rows": 4097, "cols": 771, "p": 0.0, "residual": False},
        # dropout behind the embedding's layer norm, question side
        {"name": "dropout-questions", "op": "dropout", "dtype": "bf16", "rows": 1120, "cols": 768, "p": 0.1},
        # the same for 128 blocks of 512 tokens in float32
        {"name": "dropout-blocks-float32", "op": "dropout", "dtype": "f32", "rows": 65536, "cols": 768, "p": 0.1},
        # the loss of one GPU's batch, three vectors of 768 a block, a hard negative each
        {"name": "loss-batch", "op": "loss", "B": 64, "d": 2304, "neg": True},
        # the loss over a batch gathered from many GPUs
        {"name": "loss-gathered", "op": "loss", "B": 4096, "d": 768, "neg": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "norm", "dropout", "loss"])
    if op == "attention":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        train = rng.random() < 0.75
        heads = rng.choice([4, 8, 12, 16])
        L = _log_int(rng, 1, 4096)
        cap = (128 if dtype == "bf16" else 8) * 12 * 512 * 512 // 2      # half the listed batches' scores
        B = min(_log_int(rng, 1, 128), max(1, cap // (heads * L * L)))
        return {"op": op, "dtype": dtype, "layout": rng.choice(["dense", "packed"]), "B": B, "L": L, "heads": heads,
                "p": rng.choice([0.0, 0.1, 0.1, round(rng.uniform(0.01, 0.5), 3)]), "train": train,
                "ragged": rng.random() < 0.7}
    if op == "loss":
        return {"op": op, "B": _log_int(rng, 1, 4096), "d": rng.choice([256, 512, 768, _log_int(rng, 1, 768)]),
                "neg": rng.random() < 0.6}
    rows = _log_int(rng, 1, 65536)
    cols = rng.choice([256, 512, 768, 768, 1024, _log_int(rng, 1, 4096)])
    rows = max(1, min(rows, 65536 * 768 // cols))
    case = {"op": op, "dtype": rng.choice(["bf16", "f32"]), "rows": rows, "cols": cols,
            "p": rng.choice([0.0, 0.1, 0.1, round(rng.uniform(0.01, 0.5), 3)])}
    if op == "norm":
        case["residual"] = rng.random() < 0.6
    elif case["p"] == 0.0:
        case["p"] = 0.1
    return case


def _lengths(case):
    """Tokens of each sequence: spread evenly from an eighth of L to L, the longest is L."""
    B, L = case["B"], case["L"]
    if not case["ragged"]:
        return [L] * B
    lo = max(1, L // 8)
    return [L - ((L - lo) * i) // max(1, B - 1) for i in range(B)]


def _threshold(p):
    return int(round(65536.0 * p))


# ----------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)

    s = {"case": case, "seed": torch.randint(0, 2 ** 62, (1,), generator=g, device=dev, dtype=torch.int64)}
    op = case["op"]
    if op == "loss":
        B, d = case["B"], case["d"]
        # blocks, questions near their block, hard negatives a little further away: scores of a few units
        s["c"] = randn(B, d, scale=d ** -0.25)
        s["q"] = (s["c"] * (2.0 / math.sqrt(d)) + randn(B, d, scale=d ** -0.25)).contiguous()
        s["neg"] = (s["c"] * (1.0 / math.sqrt(d)) + randn(B, d, scale=d ** -0.25)).contiguous() if case["neg"] else None
        s["dloss"] = torch.ones((), device=dev)
        return s
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    if op == "attention":
        B, L, H = case["B"], case["L"], case["heads"]
        lens = _lengths(case)
        order = torch.randperm(B, generator=g, device=dev).tolist()
        lens = [lens[i] for i in order]
        if case["layout"] == "dense":
            shape = (B, L)
            # the collate's mask: int64, ones over a sequence's tokens
            s["mask"] = (torch.arange(L, device=dev)[None, :] < torch.tensor(lens, device=dev)[:, None]).to(torch.int64)
            s["cu"] = None
        else:
            cu = [0]
            for n in lens:
                cu.append(cu[-1] + n)
            shape = (cu[-1],)
            s["mask"] = None
            s["cu"] = torch.tensor(cu, dtype=torch.int32, device=dev)
        # q, k and v are views of one projection's output
        qkv = randn(*shape, 3, H, _HEAD, dtype=dt)
        s["q"], s["k"], s["v"] = qkv.unbind(-3)
        if case["train"]:
            s["dout"] = randn(*shape, H, _HEAD, dtype=dt)
        return s
    R, C = case["rows"], case["cols"]
    s["x"] = randn(R, C, dtype=dt)
    s["dy"] = randn(R, C, dtype=dt)
    if op == "norm":
        s["residual"] = randn(R, C, dtype=dt) if case["residual"] else None
        s["weight"] = 1.0 + randn(C, scale=0.1)
        s["bias"] = randn(C, scale=0.1)
    return s


# ------------------------------------------------------------------------------------------------------- plain forms
def _philox(c0, c1, c2, c3, seed):
    """Four 32-bit words (int64 tensors) of the counters; an int64 product wraps, its 64 bits are the right ones."""
    k0, k1 = seed & _M, (seed >> 32) & _M
    for _ in range(7):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & _M) ^ c1 ^ k0, p1 & _M, ((p0 >> 32) & _M) ^ c3 ^ k1, p0 & _M
        k0, k1 = (k0 + 0x9E3779B9) & _M, (k1 + 0xBB67AE85) & _M
    return torch.stack(torch.broadcast_tensors(c0, c1, c2, c3), -1)


def _row_factor(R, C, p, seed):
    """float32 [R, C]: 0 where dropped, 1 / (1 - p) elsewhere."""
    dev, T = seed.device, _threshold(p)
    groups = torch.arange((C + 7) // 8, device=dev)[None, :]
    rows = torch.arange(R, device=dev)[:, None]
    const = torch.tensor([_M, _CALL], device=dev)
    w = _philox(groups, rows, const[0], const[1], seed)                     # [R, groups, 4]
    d = torch.stack((w & 0xFFFF, w >> 16), -1).reshape(R, -1)[:, :C]
    return (d >= T).to(torch.float32) * (65536.0 / (65536 - T))


def _score_factor(B, H, L, p, seed):
    """float32 [B, H, L, L]."""
    dev, T = seed.device, _threshold(p)
    Li, Lj = (L + 1) // 2, (L + 3) // 4
    c0 = torch.arange(Lj, device=dev)[None, None, None, :]
    c1 = torch.arange(Li, device=dev)[None, None, :, None]
    c2 = torch.arange(B * H, device=dev).reshape(B, H, 1, 1)
    w = _philox(c0, c1, c2, torch.full((), _CALL, device=dev), seed)        # [B, H, Li, Lj, 4]
    d = torch.stack((w & 0xFFFF, w >> 16), 3).reshape(B, H, 2 * Li, 4 * Lj)[:, :, :L, :L]
    return (d >= T).to(torch.float32) * (65536.0 / (65536 - T))


def _plain_attention(s):
    case = s["case"]
    B, L, H = case["B"], case["L"], case["heads"]
    dev = s["q"].device
    if s["cu"] is None:
        key = s["mask"] != 0

        def spread(t):                                                      # [B, L, H, 64] -> float32 [B, H, L, 64]
            return t.float().transpose(1, 2).contiguous()

        def gather(t):
            return t.transpose(1, 2).contiguous()
    else:
        T = s["q"].shape[0]
        pos = torch.arange(T, device=dev)
        seq = torch.searchsorted(s["cu"][1:].to(torch.int64), pos, right=True)
        slot = seq * L + pos - s["cu"].to(torch.int64)[seq]
        key = torch.arange(L, device=dev)[None, :] < (s["cu"][1:] - s["cu"][:-1])[:, None]

        def spread(t):
            dense = torch.zeros((B * L, H, _HEAD), device=dev)
            dense[slot] = t.float()
            return dense.reshape(B, L, H, _HEAD).transpose(1, 2).contiguous()

        def gather(t):
            return t.transpose(1, 2).reshape(B * L, H, _HEAD)[slot]

    dt = s["q"].dtype
    scale = 1.0 / math.sqrt(_HEAD)
    q, k, v = spread(s["q"]), spread(s["k"]), spread(s["v"])
    sc = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    sc = torch.where(key[:, None, None, :], sc, torch.full((), -1e30, device=dev))
    e = torch.exp(sc - sc.amax(-1, keepdim=True))
    prob = e / e.sum(-1, keepdim=True)
    fac = _score_factor(B, H, L, case["p"], s["seed"]) if _threshold(case["p"]) else None
    pd = prob if fac is None else prob * fac
    out = torch.matmul(pd, v)
    res = {"out": gather(out).to(dt)}
    if not case["train"]:
        return res
    do = spread(s["dout"])
    dv = torch.matmul(pd.transpose(2, 3).contiguous(), do)
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    if fac is not None:
        dp = dp * fac
    ds = prob * (dp - (prob * dp).sum(-1, keepdim=True))
    ds = torch.where(key[:, None, None, :], ds, torch.zeros((), device=dev))
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    res.update(dq=gather(dq).to(dt), dk=gather(dk).to(dt), dv=gather(dv).to(dt))
    return res


def _plain_norm(s):
    case, x = s["case"], s["x"]
    R, C = x.shape
    fac = _row_factor(R, C, case["p"], s["seed"]) if _threshold(case["p"]) else None
    z = x.float() if fac is None else x.float() * fac
    if s["residual"] is not None:
        z = z + s["residual"].float()
    mean = z.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((z - mean) ** 2).mean(-1, keepdim=True) + 1e-5)
    xh = (z - mean) * rstd
    y = xh * s["weight"] + s["bias"]
    dy = s["dy"].float()
    a = dy * s["weight"]
    dz = rstd * (a - a.mean(-1, keepdim=True) - xh * (a * xh).mean(-1, keepdim=True))
    dx = dz if fac is None else dz * fac
    res = {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dweight": (dy * xh).sum(0), "dbias": dy.sum(0)}
    if s["residual"] is not None:
        res["dresidual"] = dz.to(x.dtype)
    return res


def _plain_dropout(s):
    x = s["x"]
    fac = _row_factor(x.shape[0], x.shape[1], s["case"]["p"], s["seed"])
    return {"y": (x.float() * fac).to(x.dtype), "dx": (s["dy"].float() * fac).to(x.dtype)}


def _plain_loss(s):
    q, c, neg = s["q"], s["c"], s["neg"]
    B = q.shape[0]
    prod = torch.matmul(q, c.t().contiguous())
    if neg is not None:
        prod = torch.cat((prod, (q * neg).sum(-1, keepdim=True)), 1)
    top = prod.amax(1, keepdim=True)
    e = torch.exp(prod - top)
    z = e.sum(1, keepdim=True)
    target = torch.arange(B, device=q.device)
    loss = (top[:, 0] + torch.log(z[:, 0]) - prod[target, target]).mean()
    G = e / z
    G[target, target] -= 1.0
    G = G * (s["dloss"] / B)
    dq = torch.matmul(G[:, :B].contiguous(), c)
    res = {"loss": loss, "dc": torch.matmul(G[:, :B].t().contiguous(), q)}
    if neg is not None:
        dq = dq + G[:, B:] * neg
        res["dneg"] = G[:, B:] * q
    res["dq"] = dq
    return res


# ---------------------------------------------------------------------------------------------------- the framework
def _own_attention(s):
    from otter_amd import training
    case = s["case"]
    kw = {"mask": s["mask"], "dropout_p": case["p"], "seed": s["seed"] if case["p"] else None, "call": _CALL}
    if s["cu"] is not None:
        kw.update(cu_seqlens=s["cu"], max_seqlen=case["L"])
    out, lse = training.attention_forward(s["q"], s["k"], s["v"], **kw)
    if not case["train"]:
        return {"out": out}
    dq, dk, dv = training.attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **kw)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _own_norm(s):
    from otter_amd import training
    p = s["case"]["p"]
    kw = {"residual": s["residual"], "dropout_p": p, "seed": s["seed"] if p else None, "call": _CALL}
    y, mean, rstd = training.layer_norm_forward(s["x"], s["weight"], s["bias"], eps=1e-5, **kw)
    dx, dres, dw, db = training.layer_norm_backward(s["dy"], s["x"], s["weight"], mean, rstd, **kw)
    res = {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    if s["residual"] is not None:
        res["dresidual"] = dres
    return res


def _own_dropout(s):
    from otter_amd import training
    p = s["case"]["p"]
    return {"y": training.dropout_forward(s["x"], p, s["seed"], call=_CALL),
            "dx": training.dropout_backward(s["dy"], p, s["seed"], call=_CALL)}


def _own_loss(s):
    from otter_amd import inbatch
    loss, product, lse = inbatch.inbatch_loss_forward(s["q"], s["c"], s["neg"])
    dq, dc, dneg = inbatch.inbatch_loss_backward(s["dloss"], s["q"], s["c"], s["neg"], product, lse)
    res = {"loss": loss, "dc": dc}
    if s["neg"] is not None:
        res["dneg"] = dneg
    res["dq"] = dq
    return res


def run(state):
    op = state["case"]["op"]
    forms = ((_own_attention, _own_norm, _own_dropout, _own_loss) if own else
             (_plain_attention, _plain_norm, _plain_dropout, _plain_loss))
    return forms[("attention", "norm", "dropout", "loss").index(op)](state)


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "loss":
        B, d = case["B"], case["d"]
        n = 3 if case["neg"] else 2
        return {"bytes": 2 * n * B * d * 4 + 4, "flops": 6 * B * B * d + (6 * B * d if case["neg"] else 0)}
    size = 2 if case["dtype"] == "bf16" else 4
    if op == "attention":
        L, H, lens = case["L"], case["heads"], _lengths(case)
        if case["layout"] == "dense":                          # every query of the batch attends to its sequence's keys
            rows, pairs = case["B"] * L, sum(L * n for n in lens)
        else:
            rows, pairs = sum(lens), sum(n * n for n in lens)
        tensors = 8 if case["train"] else 4                    # q, k, v, out; with gradients dout, dq, dk, dv
        extra = case["B"] * L * 8 if case["layout"] == "dense" else 4 * (case["B"] + 1)
        # two products forward; backward four more, the scores need not be computed twice
        return {"bytes": tensors * rows * H * _HEAD * size + extra, "flops": (12 if case["train"] else 4) * pairs * H * _HEAD}
    n = case["rows"] * case["cols"]
    if op == "dropout":
        return {"bytes": 4 * n * size, "flops": 2 * n}
    tensors = 6 if case["residual"] else 4                     # x, dy, y, dx; with a residual its values and gradient
    return {"bytes": tensors * n * size + 4 * case["cols"] * 4, "flops": 20 * n}


# ------------------------------------------------------------------------------------- exact values, from the definition
def _words(a, b, c, d, seed):
    """The generator again, its 32 x 32 bit products put together from 16-bit halves."""
    def mul(x, m):
        xl, xh, ml, mh = x & 0xFFFF, x >> 16, m & 0xFFFF, m >> 16
        mid = xh * ml + ((xl * ml) >> 16)
        mid2 = xl * mh + (mid & 0xFFFF)
        return xh * mh + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | ((xl * ml) & 0xFFFF)

    lo, hi = int(seed) & _M, (int(seed) >> 32) & _M
    for r in range(7):
        h0, l0 = mul(a, 0xD2511F53)
        h1, l1 = mul(c, 0xCD9E8D57)
        a, b, c, d = h1 ^ b ^ ((lo + r * 0x9E3779B9) & _M), l1, h0 ^ d ^ ((hi + r * 0xBB67AE85) & _M), l0
    return a, b, c, d


def _pick(words, which, odd):
    w = torch.where(which == 0, words[0], torch.where(which == 1, words[1], torch.where(which == 2, words[2], words[3])))
    return torch.where(odd, w >> 16, w & 0xFFFF)


def _kept_rows(r0, r1, C, p, seed, dev):
    row = torch.arange(r0, r1, device=dev)[:, None].expand(r1 - r0, C)
    col = torch.arange(C, device=dev)[None, :].expand(r1 - r0, C)
    w = _words(col >> 3, row, torch.full_like(row, _M), torch.full_like(row, _CALL), seed)
    T = _threshold(p)
    return torch.where(_pick(w, (col & 7) >> 1, (col & 1) == 1) < T, 0.0, 65536.0 / (65536 - T)).double()


def _exact_attention(s, case):
    H, dev = case["heads"], s["q"].device
    dense = case["layout"] == "dense"
    seed = s["seed"].item()
    T = _threshold(case["p"])
    res = {"out": torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)}
    if case["train"]:
        for n in ("dq", "dk", "dv"):
            res[n] = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    starts = None if dense else s["cu"].tolist()
    for b in range(case["B"]):
        where = b if dense else slice(starts[b], starts[b + 1])
        n = case["L"] if dense else starts[b + 1] - starts[b]
        keys = (s["mask"][b] != 0) if dense else torch.ones(n, dtype=torch.bool, device=dev)
        i = torch.arange(n, device=dev)[:, None].expand(n, n)
        j = torch.arange(n, device=dev)[None, :].expand(n, n)
        for h in range(H):
            q, k, v = (s[name][where][:, h].double() for name in ("q", "k", "v"))
            a = torch.mm(q, k.t()) / 8.0
            a = a.masked_fill(~keys[None, :], -math.inf) if bool(keys.any()) else torch.zeros_like(a)
            prob = torch.softmax(a, 1)
            f = torch.ones((), dtype=torch.float64, device=dev)
            if T:
                w = _words(j >> 2, i >> 1, torch.full_like(i, b * H + h), torch.full_like(i, _CALL), seed)
                f = torch.where(_pick(w, j & 3, (i & 1) == 1) < T, 0.0, 65536.0 / (65536 - T)).double()
            o = torch.mm(prob * f, v)
            res["out"][where][:, h] = o
            if case["train"]:
                do = s["dout"][where][:, h].double()
                delta = (do * o).sum(1, keepdim=True)
                da = prob * (f * torch.mm(do, v.t()) - delta) * keys[None, :]
                res["dq"][where][:, h] = torch.mm(da, k) / 8.0
                res["dk"][where][:, h] = torch.mm(da.t(), q) / 8.0
                res["dv"][where][:, h] = torch.mm((prob * f).t(), do)
    return res


def _exact_norm(s, case):
    R, C = s["x"].shape
    dev, seed = s["x"].device, s["seed"].item()
    w, b = s["weight"].double(), s["bias"].double()
    parts = {"y": [], "dx": [], "dresidual": []}
    dw, db = torch.zeros(C, dtype=torch.float64, device=dev), torch.zeros(C, dtype=torch.float64, device=dev)
    for r0 in range(0, R, 8192):
        r1 = min(R, r0 + 8192)
        x, dy = s["x"][r0:r1].double(), s["dy"][r0:r1].double()
        f = _kept_rows(r0, r1, C, case["p"], seed, dev) if _threshold(case["p"]) else torch.ones_like(x)
        z = f * x + (s["residual"][r0:r1].double() if case["residual"] else 0.0)
        var, mean = torch.var_mean(z, 1, correction=0, keepdim=True)
        sd = torch.sqrt(var + 1e-5)
        n = (z - mean) / sd
        parts["y"].append(n * w + b)
        u = dy * w
        dz = (u - (u.sum(1, keepdim=True) + n * (u * n).sum(1, keepdim=True)) / C) / sd
        parts["dx"].append(dz * f)
        parts["dresidual"].append(dz)
        dw += (dy * n).sum(0)
        db += dy.sum(0)
    res = {"y": torch.cat(parts["y"]), "dx": torch.cat(parts["dx"]), "dweight": dw, "dbias": db}
    if case["residual"]:
        res["dresidual"] = torch.cat(parts["dresidual"])
    return res


def _exact_dropout(s, case):
    R, C = s["x"].shape
    dev, seed = s["x"].device, s["seed"].item()
    y, dx = [], []
    for r0 in range(0, R, 8192):
        r1 = min(R, r0 + 8192)
        f = _kept_rows(r0, r1, C, case["p"], seed, dev)
        y.append(s["x"][r0:r1].double() * f)
        dx.append(s["dy"][r0:r1].double() * f)
    return {"y": torch.cat(y), "dx": torch.cat(dx)}


def _exact_loss(s, case):
    q, c = s["q"].double(), s["c"].double()
    neg = s["neg"].double() if case["neg"] else None
    B = q.shape[0]
    a = torch.mm(q, c.t())
    if neg is not None:
        a = torch.cat((a, torch.sum(q * neg, 1)[:, None]), 1)
    logp = torch.log_softmax(a, 1)
    share = torch.exp(logp)
    one = torch.zeros_like(share)
    one[:, :B] = torch.eye(B, dtype=torch.float64, device=q.device)
    G = (share - one) * s["dloss"].double() / B
    res = {"loss": -torch.diagonal(logp).mean(), "dc": torch.mm(G[:, :B].t(), q)}
    dq = torch.mm(G[:, :B], c)
    if neg is not None:
        dq = dq + G[:, B:] * neg
        res["dneg"] = G[:, B:] * q
    res["dq"] = dq
    return res


def exact(case, seed):
    s = prepare(case, seed)
    forms = {"attention": _exact_attention, "norm": _exact_norm, "dropout": _exact_dropout, "loss": _exact_loss}
    return forms[case["op"]](s, case)
