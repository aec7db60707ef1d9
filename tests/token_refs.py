"""Plain 64-bit restatements of the token operators (residual RMS norm, multi-axis rotary positions, masked attention) on the CPU, and the
element-wise bounds that their kernels' outputs are held to.  Test infrastructure."""
import math

import torch

# a rounding to the type is off by at most half a step, relative; HALF_MIN: half of the smallest subnormal step (fp16 probabilities and score
# gradients below 2^-14 are rounded to a fixed grid)
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
HALF_MIN = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
F32 = 2.0 ** -24


def rnd(t, dtype):
    return t.to(dtype).double()


def norm_ref(x, w, res, eps, gy=None, gs=None):
    """float64 copies of inputs in their type -> dict of results and bounds; `x`, `res`, `w`, `gy`, `gs` are the tensors the kernel gets"""
    T, W = x.dtype, w.dtype
    s = (x.double() + res.double()).to(T).double() if res is not None else x.double()
    C = s.shape[-1]
    r = 1.0 / torch.sqrt(s.pow(2).mean(-1, keepdim=True) + eps)
    wd = w.double()
    y = s * r * wd
    # r: a sum of C squares in any order is off by at most C 2^-24 relative, half of it in the root, some operations on top
    f = F32 * (C / 2 + 8)
    out = {"s": s, "y": y, "y_tol": y.abs() * (HALF[T] + f) + HALF_MIN[T]}
    if gy is not None:
        h, xh = gy.double() * wd, s * r
        m = (h * xh).mean(-1, keepdim=True)
        a = (h * xh).abs().mean(-1, keepdim=True)
        g0 = gs.double() if gs is not None else torch.zeros_like(s)
        gx = g0 + r * (h - xh * m)
        mag = g0.abs() + r * (h.abs() + xh.abs() * (m.abs() + a))
        gw = (gy.double() * xh).reshape(-1, C).sum(0)
        rows = max(1, s.numel() // C)
        out.update(gx=gx, gx_tol=gx.abs() * HALF[T] + mag * 2 * f + HALF_MIN[T], gw=gw,
                   gw_tol=gw.abs() * HALF[W] + (gy.double() * xh).abs().reshape(-1, C).sum(0) * (f + F32 * (rows + 8)) + HALF_MIN[W])
    return out


def rotary_ref(x, pos, freq, pairs, interleaved=False, inverse=False):
    """x [B,S,H,D] -> rotated in 64 bits, bound"""
    B, S, H, D = x.shape
    T, P = x.dtype, sum(pairs)
    axis = [a for a, n in enumerate(pairs) for _ in range(n)]
    ang = pos.double()[..., axis] * freq.double()
    ang = ang if ang.dim() == 3 else ang[None]
    if inverse:
        ang = -ang
    c, s = ang.cos()[:, :, None], ang.sin()[:, :, None]
    xd = x.double()
    ia = torch.arange(0, 2 * P, 2) if interleaved else torch.arange(P)
    ib = ia + (1 if interleaved else P)
    a, b = xd[..., ia], xd[..., ib]
    out, tol = xd.clone(), torch.zeros_like(xd)
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    # the angle: fp64 (and this reference's own reduction: 2^-52 of the angle), its fraction of a turn rounded to fp32 (2^-25 of half a turn's
    # range: below 2^-26 turns = 9.4e-8 rad); sine and cosine to 2 units of 2^-24; three fp32 roundings
    e = (9.4e-8 + 2 * 2.0 ** -24 + 3 * F32 + 2.0 ** -51 * float(ang.abs().max())) * (a.abs() + b.abs())
    tol[..., ia], tol[..., ib] = e, e
    return out, tol + out.abs() * HALF[T] * (1 if T != torch.float32 else 2) + HALF_MIN[T]


def visible(B, Sq, Sk, causal=False, prefix=None, q_docs=None, k_docs=None, k_len=None):
    n = k_len.long().clamp(0, Sk) if k_len is not None else torch.full((B,), Sk)
    j, pos = torch.arange(Sk), torch.arange(Sq)[None] + n[:, None] - Sq
    see = (j[None, None] < n[:, None, None]).expand(B, Sq, Sk).clone()
    if causal:
        early = prefix[:, None, None] if prefix is not None else torch.zeros(B, 1, 1, dtype=torch.long)
        see &= (j <= pos[:, :, None]) | (j < early)
    if q_docs is not None:
        see &= (q_docs[:, :, None] == k_docs[:, None]) & (q_docs[:, :, None] >= 0)
    return see, pos


def attention_ref(q, k, v, scale=None, softcap=0.0, slopes=None, causal=False, prefix=None, q_docs=None, k_docs=None, k_len=None, go=None):
    """CPU tensors in the kernel's type -> dict of 64-bit results and element-wise bounds"""
    T = q.dtype
    B, Sq, Hq, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = scale if scale is not None else D ** -0.5
    see, pos = visible(B, Sq, Sk, causal, prefix, q_docs, k_docs, k_len)
    # keys and queries that nobody pairs with may hold anything
    kv_on, q_on = see.any(1), see.any(2)
    clean = lambda t, on: torch.where(on[..., None, None], t.double(), torch.zeros((), dtype=torch.float64))       # noqa: E731
    k64, v64, q64 = clean(k, kv_on).repeat_interleave(G, 2), clean(v, kv_on).repeat_interleave(G, 2), clean(q, q_on)
    mm = lambda a, b: torch.einsum("bihd,bjhd->bhij", a, b)                                                        # noqa: E731
    av = lambda p, x: torch.einsum("bhij,bjhd->bihd", p, x)                                                        # noqa: E731
    at = lambda p, x: torch.einsum("bhij,bihd->bjhd", p, x)                                                        # noqa: E731
    raw = mm(q64, k64) * scale
    z, t = raw, None
    if softcap:
        t = torch.tanh(raw / softcap)
        z = softcap * t
    dist = (pos[:, :, None] - torch.arange(Sk)).abs().double()[:, None]
    if slopes is not None:
        z = z - slopes.double().view(1, Hq, 1, 1) * dist
    z = z.masked_fill(~see[:, None], -math.inf)
    m = z.amax(-1, keepdim=True) if Sk else torch.zeros(B, Hq, Sq, 1, dtype=torch.float64)
    p = torch.exp(z - torch.where(m.isinf(), torch.zeros_like(m), m))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    o = av(p, v64)
    # fp32 error of a score: D products in any order, the operations behind it on numbers up to |z| and the largest score; tanh is off by
    # 4 2^-24 absolute, i.e. that times the cap.  A probability's relative error is its score's and the largest's together, the hardware
    # exponential's and the sum's (any order) on top
    zabs = float((mm(q64.abs(), k64.abs()) * scale).max()) if Sk and Sq and B else 0.0
    zmax = float(z[z.isfinite()].abs().max()) if bool(z.isfinite().any()) else 0.0
    u, lo = HALF[T], HALF_MIN[T]
    ez = F32 * (D * zabs + 8 * zmax + 8 * softcap + 4)
    e = 2 * ez + F32 * (Sk + 32)
    A = av(p, v64.abs())
    if T == torch.float32:
        u = u * 4
    out = {"o": o, "o_tol": u * o.abs() + (u + e) * A + lo * (1 + v64.abs().sum(1, keepdim=True).repeat(1, Sq, 1, 1))}
    if go is not None:
        g = clean(go, q_on)
        dp = mm(g, v64)
        delta = (g * o).sum(-1).permute(0, 2, 1)[..., None]
        fac = 1.0 - t * t if softcap else torch.ones_like(p)
        ds = p * (dp - delta) * fac
        gq, gk, gv = scale * av(ds, k64), scale * at(ds, q64), at(p, g)
        # dP and delta as sums of D products; delta reads the rounded o, with the forward's error
        dpa = mm(g.abs(), v64.abs())
        ed = ((g.abs() * (out["o_tol"] + F32 * (D + 4) * o.abs())).sum(-1)).permute(0, 2, 1)[..., None]
        efac = F32 * (4 * 4 + 4) + 2 * ez / max(softcap, 1e-30) if softcap else 0.0
        eds = p * ((e + 4 * F32) * (dp - delta).abs() * fac + F32 * (D + 4) * dpa + ed + efac * (dp - delta).abs()) + u * ds.abs() + lo
        # rows whose largest probability is within 2^-22 of one count as saturated: their score gradients are zero
        eds = eds + torch.where(p > 1 - 2.0 ** -21, ds.abs(), torch.zeros_like(ds))
        ep = p * (e + u) + lo
        acc = F32 * (max(Sq * G, Sk) + 8)
        red = lambda x: x.view(B, Sk, Hkv, G, D).sum(3)                                                            # noqa: E731
        out.update(gq=gq, gq_tol=u * gq.abs() + scale * av(eds + acc * ds.abs(), k64.abs()) + lo,
                   gk=red(gk), gk_tol=u * red(gk).abs() + scale * red(at(eds + acc * ds.abs(), q64.abs())) + lo,
                   gv=red(gv), gv_tol=u * red(gv).abs() + red(at(ep + acc * p, g.abs())) + lo)
    return out


def check(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    if bool(bad.any()):
        i = int(((got - want).abs() / tol.clamp_min(1e-300)).nan_to_num(nan=math.inf).argmax())
        raise AssertionError("%s: %d of %d outside; worst at %d: got %r want %r tol %r" % (
            what, int(bad.sum()), bad.numel(), i, float(got.reshape(-1)[i]), float(want.reshape(-1)[i]), float(tol.expand_as(want).reshape(-1)[i])))
