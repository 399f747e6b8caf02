"""Plain implementations in 64 bits of the operators on vertex tables in few bits, from their definitions."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def e4m3_table():
    """Value of every e4m3 byte."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b >> 7, -v, v)


E4M3 = e4m3_table()


def nearest(values, y):
    """Index in the ascending `values` of the one nearest to each y >= 0; ties to the even index."""
    hi = np.clip(np.searchsorted(values, y), 1, len(values) - 1)
    lo = hi - 1
    up, down = values[hi] - y, y - values[lo]
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)


def mx_blocks(F):
    return -(-F // 32)


def mx_quantize(x):
    """x [n, F] float32 -> (codes, scales) as the library lays them out."""
    n, F = x.shape
    B = mx_blocks(F)
    v = np.zeros((n, B * 32))
    v[:, :F] = x
    sign = np.zeros((n, B * 32), dtype=np.uint8)
    sign[:, :F] = np.signbit(x)
    v = v.reshape(n, B, 32)
    a = np.abs(v).max(2)
    bad = ~np.isfinite(a)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(a > 0, np.frexp(np.where(bad, 1.0, a))[1] - 1 - 2, -127)
    e = np.clip(e, -127, 127)
    y = np.ldexp(np.where(bad[:, :, None], 0.0, np.abs(v)), -e[:, :, None])
    code = nearest(E2M1, np.minimum(y, 6.0)).astype(np.uint8) | (sign.reshape(n, B, 32) << 3)
    code[np.broadcast_to(bad[:, :, None], code.shape)] = 0
    codes = (code[:, :, 0::2] | (code[:, :, 1::2] << 4)).reshape(n, B * 16)
    scales = np.zeros((n, -(-B // 4) * 4), dtype=np.uint8)
    scales[:, :B] = np.where(bad, 255, e + 127)
    return codes, scales


def mx_values(codes, scales, F):
    """The 64-bit values of a 4-bit table."""
    n, B = codes.shape[0], mx_blocks(F)
    code = np.stack([codes & 15, codes >> 4], 2).reshape(n, B * 32)
    v = np.where(code & 8, -1.0, 1.0) * E2M1[code & 7]
    s = scales[:, :B].astype(np.int64)
    s = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    return (v.reshape(n, B, 32) * s[:, :, None]).reshape(n, B * 32)[:, :F]


def mx_rows(codes, scales, F, ids=None):
    """Rows by id; one that the table does not have is zeros."""
    v = mx_values(codes, scales, F)
    if ids is None:
        return v
    out = np.zeros((len(ids), F))
    there = ids < v.shape[0]
    out[there] = v[ids[there]]
    return out


def kv8_append(cache, scales, k, v, first, D, block_rows):
    """In place, on numpy arrays laid out as the library's."""
    n, heads = k.shape[0], cache.shape[2]
    new = np.stack([k.reshape(n, heads, D), v.reshape(n, heads, D)], 1).astype(np.float64)
    for block in range(first // block_rows, -(-(first + n) // block_rows)):
        r0, r1 = block * block_rows, min((block + 1) * block_rows, first + n)
        for side in range(2):
            for h in range(heads):
                old = int(scales[block, side, h]) if r0 < first else 0
                kept = E4M3[cache[r0:max(min(first, r1), r0), side, h, :D]] * 2.0 ** (old - 127)
                x = np.concatenate([kept, new[max(r0, first) - first:r1 - first, side, h]])
                a = np.abs(x[np.isfinite(x)]).max(initial=0.0)
                e = -127
                if a > 0:
                    m, ex = np.frexp(a)
                    e = max(-127, ex - 9 + (1 if m > 0.875 else 0))
                byte = max(old, e + 127)
                y = x * 2.0 ** -(byte - 127)
                code = nearest(E4M3[:127], np.minimum(np.abs(np.where(np.isfinite(y), y, 0.0)), 448.0)).astype(np.uint8)
                code |= (np.signbit(y).astype(np.uint8) << 7)
                code = np.where(np.isfinite(y), code, 0x7F)
                cache[r0:r1, side, h, :D] = code
                cache[r0:r1, side, h, D:] = 0
                scales[block, side, h] = byte


def kv8_values(cache, scales, D, block_rows):
    """[capacity, 2, heads, D] values."""
    unit = np.ldexp(1.0, scales.astype(np.int64) - 127)
    return E4M3[cache[:, :, :, :D]] * unit[np.arange(cache.shape[0]) // block_rows][:, :, :, None]


def attention(q, values, co, rows, cache_rows, q_heads, scale):
    """(out, lse, tolerance of out, of lse): q [Vd, q_heads * D], values [capacity, 2, heads, D], rows [E] of uint32.

    Tolerances, in steps u = 2^-24 of 32-bit rounding.  A score of D products summed in 32 bits and two more roundings (the
    scales are powers of two; score_scale * log2 e is rounded once) is off by at most (D + 4) u sum|q K| scale; 2^(s - max)
    adds a rounding of the difference, covered by 2 u (|s| + |max|), and two steps of the exponential.  A weight is off by
    expm1 of that, in the sum and the weighted sum alike; both sums round at most three times for each edge (the product, the
    rescaling, the addition) and a few times where parts are joined: 3 (edges + 64) u."""
    Vd, D = len(co) - 1, values.shape[3]
    heads = values.shape[2]
    share = q_heads // heads
    u = 2.0 ** -24
    out, lse = np.zeros((Vd, q_heads, D)), np.full((Vd, q_heads), -np.inf)
    tol, ltol = np.zeros((Vd, q_heads, D)), np.zeros((Vd, q_heads))
    q = q.reshape(Vd, q_heads, D).astype(np.float64)
    for d in range(Vd):
        r = rows[co[d]:co[d + 1]]
        r = r[r < cache_rows].astype(np.int64)
        if not len(r):
            continue
        kv = values[r]
        for h in range(q_heads):
            k, v = kv[:, 0, h // share], kv[:, 1, h // share]
            s = k @ q[d, h] * scale
            p = np.exp(s - s.max())
            out[d, h] = p @ v / p.sum()
            lse[d, h] = s.max() + np.log(p.sum())
            top = (np.abs(k) @ np.abs(q[d, h]) * abs(scale)).max()
            delta = (D + 4) * u * top + 4 * u * np.abs(s).max() + 4 * u
            rounding = 3 * (len(r) + 64) * u
            tol[d, h] = (p @ np.abs(v) / p.sum()) * (2 * np.expm1(2 * delta) + 2 * rounding) + 2.0 ** -126
            ltol[d, h] = 2 * delta + 2 * rounding + 4 * u * (abs(lse[d, h]) + np.abs(s).max())
    return out.reshape(Vd, -1), lse, tol.reshape(Vd, -1), ltol
