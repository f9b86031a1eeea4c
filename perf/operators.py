"""The operators of a transformer block's training step that stand next to the matrix products:
layer normalisation, dropout from a counter-based generator, the two fused behind a residual
connection, and attention with a learned relative position bias.

Matrices are column-major, as everywhere in this repository: a (rows, cols) tensor with strides
(1, ld); attention operands are (head size, time, heads, batch) tensors with strides
(1, ld, head stride, batch stride).
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16}
_EPS = 1e-5


# ---- the cases -----------------------------------------------------------------------------

def listed():
    return [
        # one column block of a small model while it generates: the call's own latency
        {"name": "norm forward small", "op": "norm_forward", "dtype": "f16", "rows": 1024, "cols": 128},
        # a narrow fp32 model with many columns: 64 sequences of 256 tokens
        {"name": "norm backward narrow", "op": "norm_backward", "dtype": "f32", "rows": 384, "cols": 16384},
        # a wide Half model at the extent of the benchmark's products
        {"name": "norm backward wide", "op": "norm_backward", "dtype": "f16", "rows": 8192, "cols": 8192},
        # the block of a pre-norm transformer at the MLP benchmark's width, forward and backward
        {"name": "residual train", "op": "residual_train", "dtype": "f16", "rows": 1024, "cols": 16384, "p": 0.1},
        # no extent a multiple of anything: unaligned columns
        {"name": "residual forward odd", "op": "residual_forward", "dtype": "f32", "rows": 1001, "cols": 5003, "p": 0.2},
        # dropout behind an embedding of a Half model, with the residual added in the same pass
        {"name": "dropout forward", "op": "dropout_forward", "dtype": "f16", "rows": 4096, "cols": 16384, "p": 0.1, "residual": True},
        {"name": "dropout backward odd", "op": "dropout_backward", "dtype": "f32", "rows": 1023, "cols": 4097, "p": 0.5, "residual": False},
        # the attention benchmark's shape (256 heads of 256 x 64, causal), forward alone and a training step
        {"name": "attention forward", "op": "attention_forward", "dtype": "f32", "tq": 256, "tk": 256, "hs": 64, "heads": 8, "kv_heads": 8,
         "batch": 32, "causal": True, "buckets": 32, "reach": 128, "padded": False, "packed": False},
        {"name": "attention train fp32", "op": "attention_train", "dtype": "f32", "tq": 256, "tk": 256, "hs": 64, "heads": 8, "kv_heads": 8,
         "batch": 32, "causal": True, "buckets": 32, "reach": 128, "padded": False, "packed": False},
        # an encoder's padded batch of ragged sequences out of one packed projection
        {"name": "attention train padded", "op": "attention_train", "dtype": "f16", "tq": 500, "tk": 500, "hs": 64, "heads": 8, "kv_heads": 8,
         "batch": 16, "causal": False, "buckets": 32, "reach": 128, "padded": True, "packed": True},
        # one long sequence: the largest case
        {"name": "attention train long", "op": "attention_train", "dtype": "f16", "tq": 4096, "tk": 4096, "hs": 128, "heads": 16, "kv_heads": 16,
         "batch": 1, "causal": True, "buckets": 32, "reach": 128, "padded": False, "packed": False},
        # one new token of each of 32 sequences against their caches, four query heads to a cached one
        {"name": "attention token", "op": "attention_forward", "dtype": "f16", "tq": 1, "tk": 8192, "hs": 128, "heads": 16, "kv_heads": 4,
         "batch": 32, "causal": True, "buckets": 32, "reach": 128, "padded": True, "packed": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_forward", "norm_backward", "residual_forward", "residual_train", "dropout_forward", "dropout_backward",
                     "attention_forward", "attention_train", "attention_token", "attention_train"])
    dtype = rng.choice(["f16", "f32"])
    if not op.startswith("attention"):
        rows = _log_int(rng, 1, 16384)
        if rng.random() < 0.5:
            rows = max(8, rows // 8 * 8)
        c = {"op": op, "dtype": dtype, "rows": rows, "cols": _log_int(rng, 1, min(65536, max(2, (1 << 25) // rows)))}
        if not op.startswith("norm"):
            c["p"] = rng.choice([0.0, 0.1, 0.25, 0.5, 0.9])
        if op.startswith("dropout"):
            c["residual"] = op == "dropout_forward" and rng.random() < 0.5
        return c
    hs = rng.choice([16, 32, 64, 64, 80, 96, 128, 128, 57, 40])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 4])
    causal = rng.random() < 0.5
    if op == "attention_token":
        tq, tk = rng.choice([1, 1, 2, 5]), _log_int(rng, 1, 16384)
        batch = _log_int(rng, 1, max(1, min(64, (1 << 22) // (tk * kv))))
        packed, op = False, "attention_forward"
    else:
        tk = _log_int(rng, 1, 2048)
        tq = tk if rng.random() < 0.7 else _log_int(rng, 1, 2048)
        batch = _log_int(rng, 1, max(1, min(64, (1 << 25) // (tq * tk * heads))))
        packed = tq == tk and rng.random() < 0.5
    buckets, reach = rng.choice([(32, 128), (32, 128), (16, 20), (8, 64), (65, 32)])
    return {"op": op, "dtype": dtype, "tq": tq, "tk": tk, "hs": hs, "heads": heads, "kv_heads": kv, "batch": batch, "causal": causal,
            "buckets": buckets, "reach": reach, "padded": rng.random() < 0.5, "packed": packed}


# ---- inputs --------------------------------------------------------------------------------

def _randn(gen, shape, dtype, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale + shift).to(dtype)


def _matrix(gen, rows, cols, dtype, scale=1.0):
    return _randn(gen, (cols, rows), dtype, scale).t()


def _empty_matrix(rows, cols, dtype):
    return torch.empty((cols, rows), device="cuda", dtype=dtype).t()


def _empty_heads(hs, t, heads, batch, dtype):
    return torch.empty((batch, heads, t, hs), device="cuda", dtype=dtype).permute(3, 2, 1, 0)


def _bucket(d, buckets, reach, bidirectional):
    """Bucket of the relative distance d = key - query, in whole numbers: the near half of the
    buckets one to a distance, the far ones logarithmic up to `reach`."""
    base = 0
    if bidirectional:
        buckets //= 2
        base, d = (buckets if d > 0 else 0), abs(d)
    else:
        d = max(-d, 0)
    near = max(buckets // 2, 1)
    if d < near:
        return base + min(d, buckets - 1)
    steps, e = buckets - near, 0
    # largest e with (reach / near)^(e / steps) <= d / near
    while e + 1 < steps and reach ** (e + 1) * near ** steps <= d ** steps * near ** (e + 1):
        e += 1
    return base + near + e if steps > 0 else base + buckets - 1


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt, op = _DTYPES[case["dtype"]], case["op"]
    s = {"case": case, "dtype": dt}
    if op.startswith("attention"):
        tq, tk, hs, heads, kv, batch = (case[n] for n in ("tq", "tk", "hs", "heads", "kv_heads", "batch"))
        if case["packed"]:  # one projection's output: q, k and v of all heads side by side in a token's column
            qkv = _randn(gen, (batch, tq, heads + 2 * kv, hs), dt)
            parts = [qkv[:, :, :heads], qkv[:, :, heads:heads + kv], qkv[:, :, heads + kv:]]
            s["q"], s["k"], s["v"] = [x.permute(3, 1, 2, 0) for x in parts]
        else:
            s["q"] = _randn(gen, (batch, heads, tq, hs), dt).permute(3, 2, 1, 0)
            s["k"] = _randn(gen, (batch, kv, tk, hs), dt).permute(3, 2, 1, 0)
            s["v"] = _randn(gen, (batch, kv, tk, hs), dt).permute(3, 2, 1, 0)
        s["scale"] = 1.0 / math.sqrt(hs)
        s["table"] = _matrix(gen, case["buckets"], heads, dt)
        both = not case["causal"]
        s["map"] = torch.tensor([_bucket(d, case["buckets"], case["reach"], both) for d in range(-case["reach"], case["reach"] + 1)],
                                dtype=torch.int32, device="cuda")
        s["q_lengths"] = s["k_lengths"] = None
        s["q_offset"] = tk - tq if tk > tq else 0
        s["q_offsets"] = None
        if case["padded"]:
            cut = torch.randint(tk // 4, tk + 1, (batch,), generator=gen, device="cuda", dtype=torch.int32)
            s["k_lengths"] = cut
            if tq == tk:
                s["q_lengths"] = cut
            else:
                s["q_offsets"] = cut - tq
        s["o"] = _empty_heads(hs, tq, heads, batch, dt)
        s["lse"] = torch.empty((batch, heads, tq), device="cuda")
        if op == "attention_train":
            s["d_o"] = _randn(gen, (batch, heads, tq, hs), dt).permute(3, 2, 1, 0)
            s["dq"] = _empty_heads(hs, tq, heads, batch, dt)
            s["dk"], s["dv"] = (_empty_heads(hs, tk, kv, batch, dt) for _ in "kv")
            s["dtable"] = _empty_matrix(case["buckets"], heads, dt)
        return s
    rows, cols = case["rows"], case["cols"]
    if op.startswith("norm") or op.startswith("residual"):
        s["gain"], s["bias"] = _randn(gen, (rows,), dt, 0.2, 1.0), _randn(gen, (rows,), dt, 0.2)
        s["mean"], s["rstd"] = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    # activations have means and scales of their own, column by column
    x = _randn(gen, (cols, rows), dt)
    x = (x.float() * (0.5 + torch.rand((cols, 1), generator=gen, device="cuda")) + torch.randn((cols, 1), generator=gen, device="cuda")).to(dt)
    s["x"] = x.t()
    if "p" in case:
        s["p"] = case["p"]
        s["seed"], s["offset"] = 0x9E3779B97F4A7C15 ^ seed, 3 + seed % 1000
    if op.startswith("residual") or case.get("residual"):
        s["res"] = _matrix(gen, rows, cols, dt)
    if op == "norm_backward":
        f = x.float()
        s["mean"] = f.mean(1)
        s["rstd"] = (((f - s["mean"][:, None]) ** 2).mean(1) + _EPS).rsqrt()
    if op in ("norm_backward", "residual_train", "dropout_backward"):
        s["dy"] = _matrix(gen, rows, cols, dt)
        s["dx"] = _empty_matrix(rows, cols, dt)
    if op in ("norm_backward", "residual_train"):
        s["dgain"], s["dbias"] = torch.empty(rows, device="cuda", dtype=dt), torch.empty(rows, device="cuda", dtype=dt)
    if op == "residual_train":
        s["dh"] = _matrix(gen, rows, cols, dt)
        s["dres"] = _empty_matrix(rows, cols, dt)
    if op.startswith("residual"):
        s["h"] = _empty_matrix(rows, cols, dt)
    if op in ("norm_forward", "residual_forward", "residual_train", "dropout_forward"):
        s["y"] = _empty_matrix(rows, cols, dt)
    return s


# ---- one pass ------------------------------------------------------------------------------

def _keep(rows, cols, p, seed, offset, device):
    """Which elements of a rows x cols matrix dropout keeps, and their factor.  Element e = row +
    rows * column takes half-word e % 8 of Philox4x32-10 block e / 8 under the key `seed`, the
    upper two counter words being `offset`; it is kept when that is not below round(65536 p)."""
    n = rows * cols
    low = 0xFFFFFFFF
    block = torch.arange((n + 7) // 8, device=device, dtype=torch.int64)
    c0, c1 = block & low, block >> 32
    c2, c3 = torch.full_like(block, offset & low), torch.full_like(block, offset >> 32)
    k0, k1 = seed & low, seed >> 32

    def mul(m, x):  # 32 x 32 -> (high, low) without leaving 63 bits
        a, b = m * (x & 0xFFFF), m * (x >> 16)
        t = b + (a >> 16)
        return t >> 16, ((t & 0xFFFF) << 16) | (a & 0xFFFF)

    for _ in range(10):
        h0, l0 = mul(0xD2511F53, c0)
        h1, l1 = mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], 1)
    threshold = int(math.floor(p * 65536 + 0.5))
    keep = (words.reshape(-1)[:n] >= threshold).view(cols, rows).t()
    return keep, 65536.0 / (65536 - threshold)


def _norm(x, gain, bias):
    """Column normalisation of an fp32 matrix."""
    mean = x.mean(0)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(0) + _EPS)
    return (x - mean) * rstd * gain[:, None] + bias[:, None], mean, rstd


def _norm_grad(x, gain, mean, rstd, dy):
    xhat, g = (x - mean) * rstd, dy * gain[:, None]
    dx = rstd * (g - g.mean(0) - xhat * (g * xhat).mean(0))
    return dx, (dy * xhat).sum(1), dy.sum(1)


def _heads_first(x):
    """(hs, t, heads, batch) -> (batch, heads, t, hs) in fp32."""
    return x.permute(3, 2, 1, 0).float()


def _visible(s, device):
    """Which (batch, query, key) pairs take part, and the bucket of each pair's distance."""
    c = s["case"]
    tq, tk, batch = c["tq"], c["tk"], c["batch"]
    i, j = torch.arange(tq, device=device), torch.arange(tk, device=device)
    off = s["q_offsets"].long() if s["q_offsets"] is not None else torch.full((batch,), s["q_offset"], device=device)
    dist = j[None, None, :] - i[None, :, None] - off[:, None, None]
    seen = dist <= 0 if c["causal"] else torch.ones_like(dist, dtype=torch.bool)
    if s["k_lengths"] is not None:
        seen = seen & (j[None, :] < s["k_lengths"][:, None])[:, None, :]
    if s["q_lengths"] is not None:
        seen = seen & (i[None, :] < s["q_lengths"][:, None])[:, :, None]
    reach = c["reach"]
    return seen, s["map"].long()[dist.clamp(-reach, reach) + reach], off


def _attention(s):
    """Attention with the bias, in fp32; with a training case its gradients too."""
    c = s["case"]
    tq, tk, hs, heads, kv, batch = (c[n] for n in ("tq", "tk", "hs", "heads", "kv_heads", "batch"))
    q, k, v = (_heads_first(s[n]) for n in "qkv")
    if s["k_lengths"] is not None:  # what lies behind a sequence's end is never looked at
        real = torch.arange(tk, device=q.device)[None, :] < s["k_lengths"][:, None]
        k, v = (torch.where(real[:, None, :, None], x, 0.0) for x in (k, v))
    q = q.reshape(batch, kv, heads // kv * tq, hs)
    seen, bucket, off = _visible(s, q.device)
    bias = s["table"].float().t()[:, bucket].permute(1, 0, 2, 3)
    score = (q @ k.transpose(2, 3)).reshape(batch, heads, tq, tk) * s["scale"] + bias
    score = torch.where(seen[:, None], score, -math.inf)
    top = score.amax(3, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    p = torch.exp(score - top)
    total = p.sum(3, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    lse = (torch.log(total) + top).squeeze(3)
    grouped = p.reshape(batch, kv, heads // kv * tq, tk)
    o = grouped @ v
    out = {"o": _back(o.reshape(batch, heads, tq, hs), s["o"].dtype), "lse": lse}
    if c["op"] != "attention_train":
        return out
    do = _heads_first(s["d_o"])
    if s["q_lengths"] is not None:
        do = torch.where((torch.arange(tq, device=q.device)[None, :] < s["q_lengths"][:, None])[:, None, :, None], do, 0.0)
    do = do.reshape(batch, kv, heads // kv * tq, hs)
    dp = do @ v.transpose(2, 3)
    ds = grouped * (dp - (grouped * dp).sum(3, keepdim=True))
    dq = s["scale"] * (ds @ k)
    dk = s["scale"] * (ds.transpose(2, 3) @ q)
    dv = grouped.transpose(2, 3) @ do
    # sums along the diagonals: rows in reverse order, each shifted one further than the last
    skew = torch.zeros((batch, heads, tq, tk + tq), device=q.device)
    skew[..., :tk] = ds.reshape(batch, heads, tq, tk).flip(2)
    skew = skew.reshape(batch, heads, -1)[..., :tq * (tk + tq - 1)].reshape(batch, heads, tq, tk + tq - 1)
    diagonal = skew.sum(2, dtype=torch.float64)
    reach = c["reach"]
    dist = torch.arange(1 - tq, tk, device=q.device)[None, :] - off[:, None]
    to = s["map"].long()[dist.clamp(-reach, reach) + reach]
    dtable = torch.zeros((heads, c["buckets"]), device=q.device, dtype=torch.float64)
    dtable.index_add_(1, to.reshape(-1), diagonal.permute(1, 0, 2).reshape(heads, -1))
    dt = s["o"].dtype
    out |= {"dq": _back(dq.reshape(batch, heads, tq, hs), dt), "dk": _back(dk, dt), "dv": _back(dv, dt), "dtable": dtable.t().to(dt)}
    return out


def _back(x, dtype):
    return x.to(dtype).permute(3, 2, 1, 0)


def _plain(s):
    op, dt = s["case"]["op"], s["dtype"]
    if op.startswith("attention"):
        return _attention(s)
    x = s["x"].float()
    if op == "norm_forward":
        y, mean, rstd = _norm(x, s["gain"].float(), s["bias"].float())
        return {"y": y.to(dt), "mean": mean, "rstd": rstd}
    if op == "norm_backward":
        dx, dgain, dbias = _norm_grad(x, s["gain"].float(), s["mean"], s["rstd"], s["dy"].float())
        return {"dx": dx.to(dt), "dgain": dgain.to(dt), "dbias": dbias.to(dt)}
    rows, cols = x.shape
    keep, factor = _keep(rows, cols, s["p"], s["seed"], s["offset"], x.device)
    if op == "dropout_backward":
        return {"dx": torch.where(keep, s["dy"].float() * factor, 0.0).to(dt)}
    h = torch.where(keep, x * factor, 0.0)
    if "res" in s:
        h = h + s["res"].float()
    h = h.to(dt)
    if op == "dropout_forward":
        return {"y": h}
    y, mean, rstd = _norm(h.float(), s["gain"].float(), s["bias"].float())
    out = {"h": h, "y": y.to(dt), "mean": mean, "rstd": rstd}
    if op == "residual_train":
        dh, dgain, dbias = _norm_grad(h.float(), s["gain"].float(), mean, rstd, s["dy"].float())
        dh = dh + s["dh"].float()
        out |= {"dx": torch.where(keep, dh * factor, 0.0).to(dt), "dres": dh.to(dt), "dgain": dgain.to(dt), "dbias": dbias.to(dt)}
    return out


def _kernels(s):
    import ginn_b200 as gb

    c = s["case"]
    op = c["op"]
    if op.startswith("attention"):
        kw = dict(scale=s["scale"], causal=c["causal"], q_offset=s["q_offset"], q_offsets=s["q_offsets"],
                  q_lengths=s["q_lengths"], k_lengths=s["k_lengths"])
        gb.relative_attention_forward(s["q"], s["k"], s["v"], s["table"], s["map"], s["o"], s["lse"], **kw)
        out = {"o": s["o"], "lse": s["lse"]}
        if op == "attention_train":
            gb.relative_attention_backward(s["q"], s["k"], s["v"], s["table"], s["map"], s["o"], s["lse"], s["d_o"],
                                           dq=s["dq"], dk=s["dk"], dv=s["dv"], dtable=s["dtable"], accumulate=False, **kw)
            out |= {n: s[n] for n in ("dq", "dk", "dv", "dtable")}
        return out
    if op == "norm_forward":
        gb.layer_norm_forward(s["x"], s["gain"], s["bias"], s["y"], s["mean"], s["rstd"], eps=_EPS)
        return {n: s[n] for n in ("y", "mean", "rstd")}
    if op == "norm_backward":
        gb.layer_norm_backward(s["x"], s["gain"], s["mean"], s["rstd"], s["dy"], s["dx"], s["dgain"], s["dbias"], accumulate=False)
        return {n: s[n] for n in ("dx", "dgain", "dbias")}
    rng = dict(p=s["p"], seed=s["seed"], offset=s["offset"])
    if op == "dropout_forward":
        gb.dropout_forward(s["x"], s["y"], residual=s.get("res"), **rng)
        return {"y": s["y"]}
    if op == "dropout_backward":
        gb.dropout_backward(s["dy"], s["dx"], accumulate=False, **rng)
        return {"dx": s["dx"]}
    gb.residual_norm_forward(s["x"], s["res"], s["gain"], s["bias"], s["h"], s["y"], s["mean"], s["rstd"], eps=_EPS, **rng)
    out = {n: s[n] for n in ("h", "y", "mean", "rstd")}
    if op == "residual_train":
        gb.residual_norm_backward(s["h"], s["gain"], s["mean"], s["rstd"], s["dy"], s["dh"], s["dx"], s["dres"], s["dgain"], s["dbias"],
                                  accumulate=False, **rng)
        out |= {n: s[n] for n in ("dx", "dres", "dgain", "dbias")}
    return out


def run(state):
    return _kernels(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    e, op = (4 if case["dtype"] == "f32" else 2), case["op"]
    if not op.startswith("attention"):
        n = case["rows"] * case["cols"]
        # matrices read and written once; per element the normalisation's few operations
        matrices = {"norm_forward": 2, "norm_backward": 3, "dropout_forward": 3 if case.get("residual") else 2, "dropout_backward": 2,
                    "residual_forward": 4, "residual_train": 4 + 5}[op]
        if op == "residual_train":
            matrices -= 1  # h goes from the forward to the backward pass: written once, not an input
        vectors = {"norm_forward": 2, "norm_backward": 3, "residual_forward": 2, "residual_train": 4}.get(op, 0) * case["rows"] * e
        stats = 0 if op.startswith("dropout") else 8 * case["cols"]
        return {"bytes": matrices * n * e + vectors + stats,
                "flops": n * {"norm_forward": 8, "norm_backward": 14, "residual_forward": 10, "residual_train": 26}.get(op, 2)}
    tq, tk, hs, heads, kv, batch = (case[n] for n in ("tq", "tk", "hs", "heads", "kv_heads", "batch"))
    share = 5 / 8 if case["padded"] else 1.0  # lengths are uniform between a quarter and all
    pairs = tq * tk * share * (share if tq == tk else 1.0)
    if case["causal"] and tq == tk:
        pairs /= 2
    q, k = hs * tq * heads * batch, hs * tk * kv * batch * share
    train = op == "attention_train"
    return {"bytes": e * ((5 if train else 2) * q + (4 if train else 2) * k + case["buckets"] * heads * (2 if train else 1)) + 4 * tq * heads * batch,
            "flops": (7 if train else 2) * 2 * pairs * hs * heads * batch}


# ---- the definition in 64 bits -------------------------------------------------------------

def _exact_mask(rows, cols, p, seed, offset):
    """Philox4x32-10 with unsigned 64-bit words on the host."""
    n = rows * cols
    with np.errstate(over="ignore"):
        low = np.uint64(0xFFFFFFFF)
        ctr = np.zeros((4, (n + 7) // 8), np.uint64)
        ctr[0] = np.arange(ctr.shape[1], dtype=np.uint64)
        ctr[1] = ctr[0] >> np.uint64(32)
        ctr[0] &= low
        ctr[2], ctr[3] = np.uint64(offset) & low, np.uint64(offset) >> np.uint64(32)
        key = [seed % 2**32, seed // 2**32]
        for r in range(10):
            a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
            k0, k1 = (np.uint64((key[i] + r * w) % 2**32) for i, w in enumerate((0x9E3779B9, 0xBB67AE85)))
            ctr = np.stack([(b >> np.uint64(32)) ^ ctr[1] ^ k0, b & low, (a >> np.uint64(32)) ^ ctr[3] ^ k1, a & low])
    halves = ctr.T.astype("<u4", order="C").view("<u2").reshape(-1)[:n]
    cut = int(math.floor(p * 65536 + 0.5))
    return torch.from_numpy(halves >= cut).view(cols, rows).t().cuda().double() * (65536.0 / (65536 - cut))


def exact(case, seed):
    if case["op"].startswith("attention"):
        pairs = case["tq"] * case["tk"] * case["heads"] * case["batch"]
        return None if pairs > 1 << 29 else _exact_attention(case, prepare(case, seed))
    s, op = prepare(case, seed), case["op"]
    d = lambda n: s[n].double()  # noqa: E731
    mask = _exact_mask(case["rows"], case["cols"], s["p"], s["seed"], s["offset"]) if "p" in s else None
    if op == "dropout_backward":
        return {"dx": d("dy") * mask}
    x = d("x")
    if mask is not None:
        x = x * mask
        if "res" in s:
            x = x + d("res")
        if op == "dropout_forward":
            return {"y": x}
        h = x
        x = x.to(s["dtype"]).double()  # the normalisation's input is the stored sum
    var, mean = torch.var_mean(x, 0, unbiased=False)
    scale = (var + _EPS) ** -0.5
    if op == "norm_backward":
        mean, scale = d("mean"), d("rstd")
    z = (x - mean[None]) * scale[None]
    out = {"y": z * d("gain")[:, None] + d("bias")[:, None], "mean": mean, "rstd": scale}
    if op == "norm_forward":
        return out
    if op != "norm_backward":
        out = {"h": h, **out}
        if op == "residual_forward":
            return out
    dy = d("dy")
    dz = dy * d("gain")[:, None]
    n = x.shape[0]
    dx = (dz - dz.sum(0) / n - z * ((z * dz).sum(0) / n)) * scale
    weights = {"dgain": torch.einsum("rc,rc->r", z, dy), "dbias": dy.sum(1)}
    if op == "norm_backward":
        return {"dx": dx, **weights}
    total = dx + d("dh")
    return {**out, "dx": total * mask, "dres": total, **weights}


def _exact_attention(case, s):
    """One sequence after the other, each cut to its own length, through the definition and the
    chain rule."""
    tq, tk, hs, heads, kv, batch = (case[n] for n in ("tq", "tk", "hs", "heads", "kv_heads", "batch"))
    group, train = heads // kv, case["op"] == "attention_train"
    zeros = lambda *n: torch.zeros(n, device="cuda", dtype=torch.float64)  # noqa: E731
    o, lse = zeros(hs, tq, heads, batch), torch.full((batch, heads, tq), -math.inf, device="cuda", dtype=torch.float64)
    dq, dk, dv, dtable = zeros(hs, tq, heads, batch), zeros(hs, tk, kv, batch), zeros(hs, tk, kv, batch), zeros(case["buckets"], heads)
    table = s["table"].double()
    for b in range(batch):
        nk = int(s["k_lengths"][b]) if s["k_lengths"] is not None else tk
        nq = int(s["q_lengths"][b]) if s["q_lengths"] is not None else tq
        first = int(s["q_offsets"][b]) if s["q_offsets"] is not None else s["q_offset"]
        if nk == 0 or nq == 0:
            continue
        where = torch.arange(nk, device="cuda")[:, None] - (torch.arange(nq, device="cuda")[None] + first)  # (key, query)
        kind = s["map"].long()[torch.clamp(where, -case["reach"], case["reach"]) + case["reach"]]
        for n in range(kv):
            k, v = s["k"][:, :nk, n, b].double(), s["v"][:, :nk, n, b].double()
            for h in range(n * group, (n + 1) * group):
                q = s["q"][:, :nq, h, b].double()
                logits = s["scale"] * (k.t() @ q) + table[kind, h]
                if case["causal"]:
                    logits = logits.masked_fill(where > 0, -math.inf)
                norm = torch.logsumexp(logits, 0)
                w = torch.nan_to_num(torch.exp(logits - norm))
                lse[b, h, :nq], o[:, :nq, h, b] = norm, v @ w
                if train:
                    g = s["d_o"][:, :nq, h, b].double()
                    dw = v.t() @ g
                    dl = w * (dw - torch.einsum("kq,kq->q", w, dw))
                    dv[:, :nk, n, b] += g @ w.t()
                    dk[:, :nk, n, b] += s["scale"] * (q @ dl.t())
                    dq[:, :nq, h, b] = s["scale"] * (k @ dl)
                    dtable[:, h] += torch.bincount(kind.reshape(-1), weights=dl.reshape(-1), minlength=case["buckets"])
    out = {"o": o, "lse": lse}
    return {**out, "dq": dq, "dk": dk, "dv": dv, "dtable": dtable} if train else out
