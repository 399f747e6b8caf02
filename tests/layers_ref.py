"""Plain implementations in 64 bits of the operators of layers in training, from their definitions, each with a bound of what an
implementation with 32-bit sums and one rounding of its outputs may be off.

u = 2^-24 is the half step of 32-bit rounding.  A sum of m terms in 32 bits is off by at most m u times the sum of their magnitudes,
whatever its order.
"""
import math

import numpy as np
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}  # step among the subnormals


def rounding(x, dtype):
    return np.abs(x) * HALF[dtype] + LEAST[dtype] / 2


def words(counter, seed):
    """Ten rounds of Philox-4x32 of uint64 arrays that hold 32-bit words."""
    x = [np.asarray(w, dtype=np.uint64) for w in counter]
    low = np.uint64(0xFFFFFFFF)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        p, q = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(q >> np.uint64(32)) ^ x[1] ^ np.uint64(k0), q & low, (p >> np.uint64(32)) ^ x[3] ^ np.uint64(k1), p & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return x


def numbers(counter, seed):
    """The eight 16-bit numbers of every counter, [..., 8]."""
    x = np.broadcast_arrays(*words(counter, seed))
    return np.stack([h for w in x for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], -1).astype(np.int64)


def threshold(p):
    return int(np.rint(float(np.float32(p)) * 65536.0))


def factor(p):
    """What is kept is multiplied by this."""
    t = threshold(p)
    return np.float32(65536.0 / (65536 - t)) if t < 65536 else np.float32(0)


def row_factors(n, F, p, seed, step):
    kept = numbers((np.arange(-(-F // 8))[None, :], np.arange(n)[:, None], step, 0), seed).reshape(n, -(-F // 8) * 8)[:, :F] >= threshold(p)
    return np.where(kept, float(factor(p)), 0.0)


def edge_factors(src, dst, heads, p, seed, step):
    groups = np.arange(-(-heads // 8))[None, :]
    kept = numbers((src[:, None], dst[:, None], step, 1 + groups), seed).reshape(len(src), groups.size * 8)[:, :heads] >= threshold(p)
    return np.where(kept, float(factor(p)), 0.0)


# ---- dense ------------------------------------------------------------------------------------------


def activation(z, act):
    """Value, slope, and how much the two change at most with z."""
    if act == "relu":
        return np.where(z <= 0, 0.0, z), np.where(z <= 0, 0.0, 1.0), 1.0, 0.0
    if act == "gelu":
        below = 0.5 * torch.erfc(torch.from_numpy(-z / math.sqrt(2))).numpy()
        density = np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * below, below + z * density, 1.13, 0.8  # the slope's own is (2 - z^2) density <= 2 / sqrt(2 pi)
    if act == "silu":
        with np.errstate(over="ignore"):
            f = 1 / (1 + np.exp(-z))
        return z * f, f * (1 + z * (1 - f)), 1.1, 0.5
    return z, np.ones_like(z), 1.0, 0.0


def dense(x, w, b, r, g, act, factors, dtype):
    """{name: (value, bound)} of y and, with g, of the gradients x, w, b.  Operands are float64 arrays of values of `dtype`."""
    n, F = x.shape
    N = w.shape[0]
    b0 = np.zeros(N) if b is None else b
    z = x @ w.T + b0
    size = np.abs(x) @ np.abs(w).T + np.abs(b0)
    # F terms, the bias, and for products of three parts what they leave out (2^-25)
    dz = (F + 4) * U * size
    a, slope, grow, bend = activation(z, act)
    # the function itself: 8 steps of its value and of z (erf is added to 1)
    da = grow * dz + 8 * U * (np.abs(a) + np.abs(z))
    y = a * factors
    total = y if r is None else y + r
    out = {"y": (total, da * factors + 3 * U * (np.abs(y) + np.abs(total)) + rounding(total, dtype))}
    if g is None:
        return out
    gz = g * factors * slope
    off = np.abs(g * factors) * (bend * dz + 8 * U * (1 + np.abs(z))) + 3 * U * np.abs(gz)
    if act == "relu":  # on which side of its border a sum lies that is nearer to it than its error
        off = off + np.abs(g * factors) * (np.abs(z) <= dz)
    if b is not None:
        gb = gz.sum(0)
        out["b"] = (gb, off.sum(0) + (n + 2) * U * np.abs(gz).sum(0) + rounding(gb, dtype))
    # in 16 bits the gradient of z is rounded for the products
    held = off + (rounding(np.abs(gz) + off, dtype) if dtype != torch.float32 else 0.0)
    gx, gw = gz @ w, gz.T @ x
    out["x"] = (gx, held @ np.abs(w) + (N + 4) * U * ((np.abs(gz) + held) @ np.abs(w)) + rounding(gx, dtype))
    out["w"] = (gw, held.T @ np.abs(x) + (n + 4) * U * ((np.abs(gz) + held).T @ np.abs(x)) + rounding(gw, dtype))
    return out


# ---- attention --------------------------------------------------------------------------------------


def attention(q, k, v, g, co, ri, H, Hk, scale, dropout, dtype):
    """{name: (value, bound)} of out, lse and, with g, of the gradients q, k, v.  q [Vd, H * D], k and v [Vs, Hk * D] float64;
    dropout: (p, seed, step) or None."""
    Vd, Vs, D = q.shape[0], k.shape[0], q.shape[1] // H
    dst = np.repeat(np.arange(Vd), np.diff(co.astype(np.int64)))
    src = ri[int(co[0]):int(co[-1])].astype(np.int64)
    there = src < Vs
    dst, src = dst[there], src[there]
    head = np.arange(H) // (H // Hk)
    qe, ke, ve = q.reshape(Vd, H, D)[dst], k.reshape(Vs, Hk, D)[src][:, head], v.reshape(Vs, Hk, D)[src][:, head]

    def by(index, count, x):
        out = np.zeros((count,) + x.shape[1:])
        np.add.at(out, index, x)
        return out

    with np.errstate(invalid="ignore", divide="ignore"):
        s = scale * (qe * ke).sum(2)
        ds = (D + 6) * U * abs(scale) * (np.abs(qe) * np.abs(ke)).sum(2)
        top = np.full((Vd, H), -np.inf)
        np.maximum.at(top, dst, s)
        base = np.where(top == -np.inf, 0.0, top)
        e = np.exp(s - base[dst])
        total = by(dst, Vd, e)
        lse = np.where(total > 0, base + np.log(np.where(total > 0, total, 1.0)), -np.inf)
        p = np.where(total[dst] > 0, e / np.where(total > 0, total, 1.0)[dst], 0.0)
    worst = np.zeros((Vd, H))
    np.maximum.at(worst, dst, ds)
    degree = by(dst, Vd, np.ones(len(dst)))[:, None]
    fine = np.where(np.isfinite(lse), np.abs(lse), 0.0)
    m = np.ones((len(src), H)) if dropout is None else edge_factors(src, dst, H, *dropout)
    pm = (p * m)[:, :, None]
    out = by(dst, Vd, pm * ve)
    size = by(dst, Vd, pm * np.abs(ve))
    # twice what the scores are off (numerator and denominator), the sums' and some twenty further roundings; exp2 of a score
    # that was multiplied by log2 e is off by a few steps of the score more, which ds's 6 holds
    rel = (2 * worst + (2 * degree + 20) * U)[:, :, None]
    # a probability below 2^-126 may count as 0: a product with it is off by less than 2^-126 of its other part
    lost = 2.0 ** -126
    size = size * rel + lost * by(dst, Vd, m[:, :, None] * np.abs(ve))
    value = {"out": (out.reshape(Vd, H * D), (size + rounding(out, dtype)).reshape(Vd, H * D)),
             "lse": (lse, worst + (degree + 8) * U + 4 * U * fine)}
    if g is None:
        return value
    ge = g.reshape(Vd, H, D)[dst]
    gv = (ge * ve).sum(2)
    c, dc = m * gv, (D + 4) * U * m * (np.abs(ge) * np.abs(ve)).sum(2)
    # the probabilities once more, from lse: its error on top
    prel = (3 * worst + (2 * degree + 40) * U + 8 * U * fine)
    mean = by(dst, Vd, p * c)
    dmean = by(dst, Vd, p * (np.abs(c) * prel[dst] + dc)) + (degree + 4) * U * by(dst, Vd, p * np.abs(c))
    gs = scale * p * (c - mean[dst])
    # gq = scale (sum p c k - mean sum p k): the error of each product's parts, not of their difference
    apart = abs(scale) * p * (np.abs(c) + np.abs(mean)[dst])
    dgs = apart * (prel[dst] + (degree[dst] + 8) * U) + abs(scale) * (p * (dc + dmean[dst]) + lost * (np.abs(c) + np.abs(mean)[dst]))
    gq = by(dst, Vd, gs[:, :, None] * ke)
    value["q"] = (gq, by(dst, Vd, dgs[:, :, None] * np.abs(ke)) + (degree[:, :, None] + 8) * U * by(dst, Vd, apart[:, :, None] * np.abs(ke))
                  + rounding(gq, dtype))
    uses = by(src, Vs, np.ones(len(src)))[:, None, None] * (H // Hk) + 8

    def shared(x):
        return by(src, Vs, x).reshape(Vs, Hk, H // Hk, D).sum(2)

    gk, gvv = shared(gs[:, :, None] * qe), shared(pm * ge)
    value["k"] = (gk, shared(dgs[:, :, None] * np.abs(qe)) + uses * U * shared(apart[:, :, None] * np.abs(qe)) + rounding(gk, dtype))
    value["v"] = (gvv, shared((pm * prel[dst][:, :, None] + lost * m[:, :, None]) * np.abs(ge)) + uses * U * shared(pm * np.abs(ge)) + rounding(gvv, dtype))
    for name, shape in (("q", (Vd, H * D)), ("k", (Vs, Hk * D)), ("v", (Vs, Hk * D))):
        value[name] = tuple(x.reshape(shape) for x in value[name])
    return value


def by_source(co, ri, Vs):
    """The edges by source, those without one left out: row offsets and destinations."""
    dst = np.repeat(np.arange(len(co) - 1, dtype=np.uint32), np.diff(co.astype(np.int64)))
    src = ri[int(co[0]):int(co[-1])]
    order = np.argsort(src, kind="stable")
    order = order[src[order] < Vs]
    ro = np.zeros(Vs + 1, dtype=np.uint32)
    ro[1:] = np.cumsum(np.bincount(src[order], minlength=Vs))
    return ro, dst[order]


def check(got, expected, what):
    value, bound = expected
    got = got.detach().float().cpu().numpy().astype(np.float64) if isinstance(got, torch.Tensor) else got
    assert got.shape == value.shape, (what, got.shape, value.shape)
    fine = np.isfinite(value)
    assert (np.isnan(got) == np.isnan(value)).all(), f"{what}: NaN at other places"
    assert (got[~fine & ~np.isnan(value)] == value[~fine & ~np.isnan(value)]).all(), f"{what}: infinities"
    off = np.abs(got[fine] - value[fine]) - np.broadcast_to(bound, value.shape)[fine]
    if off.size:
        assert off.max() <= 0, f"{what}: off by {off.max():.3g} more than the bound, at {int(np.argmax(off))} of {off.size}"
