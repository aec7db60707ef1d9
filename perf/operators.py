"""Cases of the token-block operators: root-mean-square norm with the residual's addition, rotary positions over several axes, and attention
with capped scores, distance bias, document and prefix masks.

An image or video encoder over patch tokens runs the three in this order: the norm adds a sub-layer's output to the residual stream and
normalises it, the rotation puts the row / column / time positions into queries and keys, attention mixes the tokens.  Sizes: patch grids of
this repository's image sizes (192 x 640 and 320 x 1024 in patches of 16: 480 and 1280 tokens; 3 frames of the latter: 3840), batch 12,
and generic widths.

own = False: elementary torch operations in 32 bits (64 for the angles of the rotation), rounded once at the end.
own = True:  the calls of sqd.nnops.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


# --------------------------------------------------------------------------------------------------------------------------- cases
def _norm(name, rows, width, dtype, train, wtype="f32"):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "wtype": wtype, "train": train}


def _rotary(name, batch, grid, heads, kv_heads, dim, dtype, train, first=0):
    """grid: "T x H x W" tokens of a video or "H x W" of an image; first: time (or row) of the first token."""
    return {"name": name, "op": "rotary", "batch": batch, "grid": grid, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "train": train, "first": first}


def _attn(name, batch, sq, sk, heads, kv_heads, dim, dtype, train, softcap=0.0, slopes=False, causal=False, prefix=0, docs=0, ragged=False):
    """docs: documents (clips) in a row, the last tenth of it padding; ragged: every row of the batch has its own number of keys."""
    return {"name": name, "op": "attention", "batch": batch, "sq": sq, "sk": sk, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "train": train, "softcap": softcap, "slopes": slopes, "causal": causal, "prefix": prefix, "docs": docs, "ragged": ragged}


def listed():
    return [
        # one new token for each of 12 streams: the smallest call of a stream that answers frame by frame
        _norm("norm_12_tokens", 12, 1024, "bf16", False),
        # a training step's norm over the patch tokens of a batch of 12 images of 192 x 640
        _norm("norm_train_image", 12 * 480, 768, "bf16", True),
        # odd rows and an odd width in full precision, the type this repository trains in
        _norm("norm_train_f32_odd", 4 * 1281, 1001, "f32", True),
        # eight clips of 16 frames of 20 x 64 patches through a wide encoder
        _norm("norm_video_wide", 8 * 16 * 1280, 2048, "f16", False, "f16"),
        # one new token a stream, far into a video
        _rotary("rotary_12_tokens", 12, "1x1x1", 16, 4, 64, "bf16", False, 100000),
        # row and column positions of a training batch
        _rotary("rotary_train_image", 12, "12x40", 12, 12, 64, "bf16", True),
        # time, row and column positions of two clips with grouped key heads
        _rotary("rotary_video", 2, "16x20x64", 16, 4, 128, "bf16", False),
        # one new token a stream against caches of up to 8191 keys of different lengths
        _attn("attn_token_cache", 16, 1, 8191, 32, 8, 128, "bf16", False, softcap=30.0, causal=True, ragged=True),
        # a training step over the patch tokens of 12 images, with the bias by distance along the sequence
        _attn("attn_train_image", 12, 480, 480, 12, 12, 64, "bf16", True, slopes=True),
        # full precision, odd lengths, image tokens that see each other in front of a causal tail
        _attn("attn_train_f32_odd", 2, 1281, 1281, 8, 4, 40, "f32", True, causal=True, prefix=481),
        # two rows of packed clips with capped scores, trained: 3 frames of 20 x 64 patches
        _attn("attn_train_video", 2, 3840, 3840, 16, 4, 128, "bf16", True, softcap=50.0, docs=3),
        # a long causal prompt behind a prefix of image tokens
        _attn("attn_long_prompt", 1, 8192, 8192, 16, 4, 128, "f16", False, causal=True, prefix=1280),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "attention", "attention"])
    dtype, train = rng.choice(["bf16", "bf16", "f16", "f32"]), rng.random() < 0.5
    if op == "norm":
        width = _log(rng, 64, 4096)
        width = width if rng.random() < 0.3 else max(8, width // 8 * 8)
        rows = min(_log(rng, 1, 160000), (40 if train else 160) * 1000 * 1000 // width)
        c = _norm("", rows, width, dtype, train, rng.choice(["f32", dtype]))
    elif op == "rotary":
        kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([16, 32, 40, 64, 96, 128])
        heads = kv * rng.choice([1, 2, 4])
        h, w, t = _log(rng, 1, 40), _log(rng, 1, 128), rng.choice([0, 1, _log(rng, 2, 16)])
        most = 40 * 1000 * 1000 // (dim * (heads + kv) * h * w * max(1, t))
        c = _rotary("", max(1, min(_log(rng, 1, 16), most)), "%dx%dx%d" % (t, h, w) if t else "%dx%d" % (h, w), heads, kv, dim, dtype, train,
                    rng.choice([0, _log(rng, 1, 1000000)]))
    else:
        kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([16, 32, 40, 64, 96, 128])
        heads = kv * rng.choice([1, 2, 3, 4])
        kind = rng.choice(["token", "self", "self"])
        cap, slopes = rng.choice([0.0, 0.0, 20.0, 50.0]), rng.random() < 0.3
        if kind == "token":
            sk = _log(rng, 1, 16000)
            sq = min(sk, rng.choice([1, 1, 1, 2, 5]))
            batch = max(1, min(_log(rng, 1, 32), 250 * 1000 * 1000 // (sk * heads * dim)))
            c = _attn("", batch, sq, sk, heads, kv, dim, dtype, False, cap, slopes, True, 0, 0, rng.random() < 0.7)
        else:
            s = _log(rng, 1, 4000)
            batch = max(1, min(_log(rng, 1, 16), (200 if dtype == "f32" else 400) * 1000 * 1000 // (s * s * heads)))
            mask = rng.choice(["none", "causal", "prefix", "docs", "docs"])
            c = _attn("", batch, s, s, heads, kv, dim, dtype, train, cap, slopes, mask in ("causal", "prefix"),
                      rng.randint(1, s) if mask == "prefix" else 0, rng.randint(1, 6) if mask == "docs" else 0)
    del c["name"]
    return c


def _grid(case):
    return [int(n) for n in case["grid"].split("x")]


def _sections(case):
    """rotation pairs of each axis: a quarter of the pairs for the time, the rest shared by rows and columns; without a time axis halves"""
    pairs = case["dim"] // 2
    if len(_grid(case)) == 2:
        return (pairs // 2, pairs - pairs // 2)
    t = pairs // 4
    return (t, (pairs - t) // 2, pairs - t - (pairs - t) // 2)


def _lengths(case):
    """keys of each row of the batch: all of them, or between one key and all"""
    B, Sk = case["batch"], case["sk"]
    return [max(1, Sk - (Sk * b) // (2 * B)) for b in range(B)] if case["ragged"] else [Sk] * B


def _documents(case):
    """document of each token: equal parts of the first nine tenths, -1 (padding) behind them"""
    n, real = case["docs"], max(1, case["sk"] * 9 // 10)
    return [j * n // real if j < real else -1 for j in range(case["sk"])]


def _visible(case):
    """pairs of query and key that the masks leave, over the batch, for one head"""
    Sq, total = case["sq"], 0
    if case["docs"]:
        ids = _documents(case)
        return case["batch"] * sum(ids.count(d) ** 2 for d in range(case["docs"]))
    for n in _lengths(case):
        total += sum(min(n, max(0, i + n - Sq + 1, case["prefix"])) for i in range(Sq)) if case["causal"] else Sq * n
    return total


def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        # forward: x, residual -> y, stream; a training step reads the gradients of both outputs and writes one gradient more
        return {"bytes": n * size * (7 if case["train"] else 4) + 2 * case["width"] * 4, "flops": n * (15 if case["train"] else 5)}
    if case["op"] == "rotary":
        tokens = case["batch"] * math.prod(_grid(case))
        n = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        times = 2 if case["train"] else 1
        return {"bytes": times * (2 * n * size) + tokens * 4 * len(_grid(case)), "flops": times * 3 * n}
    B, H, Hk, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    qo = B * case["sq"] * H * D * size
    kv = sum(_lengths(case)) * Hk * D * size
    pairs = _visible(case) * H
    # two products forward, five more backward (scores again, and the gradients of probabilities, values, queries and keys)
    return {"bytes": (4 * qo + 4 * kv) if case["train"] else 2 * qo + 2 * kv, "flops": 2.0 * pairs * D * (7 if case["train"] else 2)}


# ------------------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev, dt, train = torch.device("cuda"), DTYPES[case["dtype"]], case["train"]
    g = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape, dtype=dt, std=1.0):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).mul_(std).to(dtype)

    st = {"case": case}
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        # a residual stream grows with depth and has a few strong features; a sub-layer's output is smaller
        strong = 1.0 + 20.0 * (torch.rand(width, generator=g, device=dev) < 0.01).float()
        st["x"] = rand(rows, width)
        st["res"] = (rand(rows, width, dtype=torch.float32, std=3.0) * strong).to(dt)
        st["w"] = rand(width, dtype=torch.float32, std=0.2).add_(1.0).to(DTYPES[case["wtype"]])
        if train:
            st["gy"], st["gs"] = rand(rows, width), rand(rows, width, std=0.5)
            for k in ("x", "res", "w"):
                st[k].requires_grad_(True)
    elif case["op"] == "rotary":
        B, dims = case["batch"], _grid(case)
        S = math.prod(dims)
        st["q"], st["k"] = rand(B, S, case["heads"], case["dim"]), rand(B, S, case["kv_heads"], case["dim"])
        pos = torch.cartesian_prod(*[torch.arange(n, device=dev, dtype=torch.int32) for n in dims]).view(S, len(dims)).clone()
        pos[:, 0] += case["first"]
        st["pos"] = pos
        # every axis has its own ladder of frequencies (radians for each unit of position), in 64 bits: a table that a model keeps
        st["freq"] = torch.cat([10000.0 ** (-torch.arange(n, device=dev, dtype=torch.float64) / max(1, n)) for n in _sections(case)])
        if train:
            st["gq"], st["gk"] = rand(*st["q"].shape), rand(*st["k"].shape)
            st["q"].requires_grad_(True), st["k"].requires_grad_(True)
    else:
        B, Sq, Sk, H, Hk, D = (case[k] for k in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
        st["q"], st["k"], st["v"] = rand(B, Sq, H, D, std=2.0), rand(B, Sk, Hk, D), rand(B, Sk, Hk, D)
        st["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device=dev, dtype=torch.float32) / H) if case["slopes"] else None
        st["prefix"] = torch.full((B,), case["prefix"], device=dev, dtype=torch.int32) if case["prefix"] else None
        st["lengths"] = torch.tensor(_lengths(case), device=dev, dtype=torch.int32) if case["ragged"] else None
        st["docs"] = torch.tensor(_documents(case), device=dev, dtype=torch.int32).expand(B, Sk).contiguous() if case["docs"] else None
        if train:
            st["go"] = rand(B, Sq, H, D)
            for k in ("q", "k", "v"):
                st[k].requires_grad_(True)
    return st


# ---------------------------------------------------------------------------------------------------------------------- plain forms
def _plain_norm(st):
    case, x, res, w = st["case"], st["x"], st["res"], st["w"]
    # the stream is kept in the inputs' type: that rounding is part of the operator, and what is normalised is the stream
    s = (x.detach().float() + res.detach().float()).to(x.dtype)
    s32, w32 = s.float(), w.detach().float()
    r = torch.rsqrt((s32 * s32).mean(-1, keepdim=True) + EPS)
    xhat = s32 * r
    out = {"y": (xhat * w32).to(x.dtype), "stream": s}
    if case["train"]:
        gy, gs = st["gy"].float(), st["gs"].float()
        gh = gy * w32
        gx = (gs + r * (gh - xhat * (gh * xhat).mean(-1, keepdim=True))).to(x.dtype)
        out["gx"], out["gres"], out["gw"] = gx, gx, (gy * xhat).sum(0).to(w.dtype)
    return out


def _plain_angles(st):
    sections = _sections(st["case"])
    p = st["pos"].double()
    return torch.cat([p[:, a:a + 1].expand(-1, n) for a, n in enumerate(sections)], 1) * st["freq"]


def _plain_rotate(x, cos, sin):
    n, xf = cos.shape[-1], x.detach().float()
    a, b, rest = xf[..., :n], xf[..., n:2 * n], xf[..., 2 * n:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).to(x.dtype)


def _plain_rotary(st):
    ang = _plain_angles(st)
    cos, sin = ang.cos().float()[None, :, None], ang.sin().float()[None, :, None]
    out = {"q": _plain_rotate(st["q"], cos, sin), "k": _plain_rotate(st["k"], cos, sin)}
    if st["case"]["train"]:
        out["gq"], out["gk"] = _plain_rotate(st["gq"], cos, -sin), _plain_rotate(st["gk"], cos, -sin)
    return out


def _plain_attention(st):
    case = st["case"]
    B, Sq, Sk, H, Hk, D = (case[k] for k in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
    G, dev, dt, train = H // Hk, st["q"].device, st["q"].dtype, case["train"]
    q = st["q"].detach().float().view(B, Sq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Sq, D)
    k = st["k"].detach().float().permute(0, 2, 1, 3).contiguous()
    v = st["v"].detach().float().permute(0, 2, 1, 3).contiguous()
    kT = k.transpose(2, 3).contiguous()
    raw = torch.matmul(q, kT).view(B, Hk, G, Sq, Sk) / math.sqrt(D)
    s, cap = raw, case["softcap"]
    if cap:
        t = torch.tanh(raw / cap)
        s = cap * t
    j = torch.arange(Sk, device=dev)
    n = st["lengths"].long() if st["lengths"] is not None else torch.full((B,), Sk, device=dev)
    at = torch.arange(Sq, device=dev)[None] + n[:, None] - Sq                                        # position of each query [B, Sq]
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, Hk, G, 1, 1) * (at[:, :, None] - j).abs().float()[:, None, None]
    see = (j[None, None] < n[:, None, None]).expand(B, Sq, Sk)
    if case["causal"]:
        early = st["prefix"][:, None, None] if st["prefix"] is not None else 0
        see = see & ((j <= at[:, :, None]) | (j < early))
    if st["docs"] is not None:
        d = st["docs"]
        see = see & (d[:, :, None] == d[:, None]) & (d[:, :, None] >= 0)
    see = see[:, None, None]
    s = s.masked_fill(~see, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(p.view(B, Hk, G * Sq, Sk), v)

    def back(x, S, heads):
        return x.view(B, Hk, heads, S, D).permute(0, 3, 1, 2, 4).reshape(B, S, Hk * heads, D).to(dt)

    out = {"o": back(o, Sq, G)}
    if train:
        go = st["go"].float().view(B, Sq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Sq, D)
        gv = torch.matmul(p.view(B, Hk, G * Sq, Sk).transpose(2, 3).contiguous(), go)
        gp = torch.matmul(go, v.transpose(2, 3).contiguous()).view(B, Hk, G, Sq, Sk)
        gs = p * (gp - (gp * p).sum(-1, keepdim=True))
        if cap:
            gs = gs * (1.0 - t * t)
        gs = gs.view(B, Hk, G * Sq, Sk) / math.sqrt(D)
        out["gq"] = back(torch.matmul(gs, k), Sq, G)
        out["gk"], out["gv"] = back(torch.matmul(gs.transpose(2, 3).contiguous(), q), Sk, 1), back(gv, Sk, 1)
    return out


# ----------------------------------------------------------------------------------------------------------- the framework's kernels
def _nnops():
    src = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sfmnext-impl_amd")
    if src not in sys.path:
        sys.path.insert(0, src)
    from sqd import nnops
    return nnops


def _own_norm(st):
    y, s = _nnops().rms_norm_residual(st["x"], st["w"], st["res"], eps=EPS)
    out = {"y": y.detach(), "stream": s.detach()}
    if st["case"]["train"]:
        out["gx"], out["gres"], out["gw"] = torch.autograd.grad((y, s), (st["x"], st["res"], st["w"]), (st["gy"], st["gs"]))
    return out


def _own_rotary(st):
    q, k = _nnops().rotary_axes(st["q"], st["k"], st["pos"], st["freq"], _sections(st["case"]))
    out = {"q": q.detach(), "k": k.detach()}
    if st["case"]["train"]:
        out["gq"], out["gk"] = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"]))
    return out


def _own_attention(st):
    case = st["case"]
    o = _nnops().attention(st["q"], st["k"], st["v"], softcap=case["softcap"], slopes=st["slopes"], causal=case["causal"], prefix=st["prefix"],
                           q_docs=st["docs"], k_docs=st["docs"], k_len=st["lengths"])
    out = {"o": o.detach()}
    if case["train"]:
        out["gq"], out["gk"], out["gv"] = torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["go"])
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return (_own_norm if op == "norm" else _own_rotary if op == "rotary" else _own_attention)(state)
    return (_plain_norm if op == "norm" else _plain_rotary if op == "rotary" else _plain_attention)(state)


# ------------------------------------------------------------------------------------------------- the operators' definitions, 64 bits
def _exact_norm(st, case):
    """stream = round(x + residual); y_c = w_c stream_c / sqrt(mean stream^2 + eps), and the vector-Jacobian products, a slab of rows at a time"""
    x, res, w = st["x"].detach(), st["res"].detach(), st["w"].detach().double()
    ys, ss, gxs, gw = [], [], [], torch.zeros_like(w)
    for i in range(0, x.shape[0], 16384):
        s = (x[i:i + 16384].double() + res[i:i + 16384].double()).to(x.dtype)
        sd = s.double()
        rms = (sd.pow(2).mean(1) + EPS).sqrt()[:, None]
        ys.append(sd / rms * w)
        ss.append(sd)
        if case["train"]:
            gy = st["gy"][i:i + 16384].double()
            proj = (gy * w * sd).sum(1, keepdim=True) / (case["width"] * rms.pow(3))
            gxs.append(st["gs"][i:i + 16384].double() + gy * w / rms - sd * proj)
            gw += (gy * sd / rms).sum(0)
    out = {"y": torch.cat(ys), "stream": torch.cat(ss)}
    if case["train"]:
        out["gx"] = out["gres"] = torch.cat(gxs)
        out["gw"] = gw
    return out


def _exact_rotary(st, case):
    """the pair (x_p, x_{p+P}) as a complex number, times e^{i angle}"""
    sections = _sections(case)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    ang = st["pos"].double()[:, axis] * st["freq"]
    turn = torch.polar(torch.ones_like(ang), ang)[None, :, None]
    P = len(axis)

    def rotate(x, by):
        x = x.detach().double()
        z = torch.complex(x[..., :P], x[..., P:2 * P]) * by
        return torch.cat([z.real, z.imag, x[..., 2 * P:]], -1)

    out = {"q": rotate(st["q"], turn), "k": rotate(st["k"], turn)}
    if case["train"]:
        out["gq"], out["gk"] = rotate(st["gq"], turn.conj()), rotate(st["gk"], turn.conj())
    return out


def _exact_attention(st, case):
    """one query head of one row of the batch at a time"""
    B, Sq, Sk, H, Hk, D = (case[k] for k in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
    if B * H * Sq * Sk > 1.6e9:
        return None
    G, dev, cap, scale, train = H // Hk, st["q"].device, case["softcap"], 1.0 / math.sqrt(D), case["train"]
    names = ("gq", "gk", "gv") if train else ()
    out = {"o": torch.zeros(B, Sq, H, D, device=dev, dtype=torch.float64)}
    for name in names:
        out[name] = torch.zeros(B, Sq if name == "gq" else Sk, H if name == "gq" else Hk, D, device=dev, dtype=torch.float64)
    col, ids = torch.arange(Sk, device=dev)[None], st["docs"]
    for b, n in enumerate(_lengths(case)):
        row = (torch.arange(Sq, device=dev) + (n - Sq))[:, None]
        hidden = col >= n
        if case["causal"]:
            hidden = hidden | ((col > row) & (col >= case["prefix"]))
        if ids is not None:
            hidden = hidden | (ids[b][:, None] != ids[b][None]) | (ids[b] < 0)[:, None]
        hidden = hidden.expand(Sq, Sk)
        for h in range(H):
            q, k, v = st["q"].detach()[b, :, h].double(), st["k"].detach()[b, :, h // G].double(), st["v"].detach()[b, :, h // G].double()
            z = q @ k.T * scale
            slope_of_cap = None
            if cap:
                slope_of_cap = 1.0 / torch.cosh(z / cap).square()
                z = torch.tanh(z / cap) * cap
            if case["slopes"]:
                z = z - st["slopes"][h].double() * (row - col).abs()
            z = torch.where(hidden, -math.inf, z)
            p = torch.nan_to_num(torch.softmax(z, 1), nan=0.0)               # a row without a key: zeros
            out["o"][b, :, h] = p @ v
            if train:
                go = st["go"][b, :, h].double()
                dz = p * (go @ v.T - (go * out["o"][b, :, h]).sum(1, keepdim=True)) * scale
                if cap:
                    dz = dz * slope_of_cap
                out["gq"][b, :, h] = dz @ k
                out["gk"][b, :, h // G] += dz.T @ q
                out["gv"][b, :, h // G] += p.T @ go
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return (_exact_norm if case["op"] == "norm" else _exact_rotary if case["op"] == "rotary" else _exact_attention)(st, case)
