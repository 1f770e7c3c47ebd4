"""Plain 64-bit restatement of the 8-bit paged K/V cache: the number format, the
page layout and the attention over it, from their definitions in numpy."""
import numpy as np

TILE = 16


def e4m3_values():
    v = np.empty(256)
    for code in range(256):
        e, m = (code >> 3) & 15, code & 7
        x = np.nan if (e, m) == (15, 7) else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[code] = -x if code & 128 else x
    return v


E4M3 = e4m3_values()


def quantise(x):
    """x [..., d] fp32 values: (codes uint8 [..., d], bytes uint8 [...])."""
    x = np.asarray(x, np.float64)
    fine = np.isfinite(x).all(-1)
    x = np.where(fine[..., None], x, 0.0)
    m, e = np.frexp(np.abs(x).max(-1))  # max |x| = m 2^e; 448 = 0.875 * 2^9
    e = np.where(m == 0, -126, np.maximum(np.where(m > 0.875, e - 8, e - 9), -126))
    y = np.ldexp(x, -e[..., None])
    quantum = np.ldexp(1.0, np.maximum(np.frexp(y)[1] - 1, -6) - 3)
    y = np.round(y / quantum) * quantum  # half to even
    codes = np.searchsorted(E4M3[:127], np.abs(y)).astype(np.uint8)
    assert np.array_equal(E4M3[codes], np.abs(y))
    codes |= np.where(np.signbit(y), 128, 0).astype(np.uint8)
    codes = np.where(fine[..., None], codes, 0).astype(np.uint8)
    return codes, np.where(fine, e + 127, 255).astype(np.uint8)


def dequantise(codes, byte):
    b = byte.astype(np.int64)
    scale = np.where(b == 255, np.nan, np.where(b == 0, 0.0, np.ldexp(1.0, b - 127)))
    with np.errstate(invalid="ignore"):
        return E4M3[codes] * scale[..., None]


def page_bytes(kv_heads, d, page_size):
    return page_size * kv_heads * (d + 1)


def slot_index(kv_heads, d, page_size, is_v, page, offset):
    """Byte positions in the pool of a slot: codes [kv_heads, d], bytes [kv_heads]."""
    tile = page * page_bytes(kv_heads, d, page_size) + offset // TILE * page_bytes(kv_heads, d, TILE)
    s = offset % TILE
    h, i = np.arange(kv_heads)[:, None], np.arange(d)[None]
    code = (h * d + i) * TILE + s if is_v else (h * TILE + s) * d + i
    return tile + code, tile + kv_heads * d * TILE + h[:, 0] * TILE + s


def store(pool, is_v, kv_heads, d, page_size, page, offset, x):
    """pool: flat uint8 array; x [kv_heads, d]."""
    code, byte = slot_index(kv_heads, d, page_size, is_v, page, offset)
    pool[code], pool[byte] = quantise(x)


def fetch(pool, is_v, kv_heads, d, page_size, page, offset):
    code, byte = slot_index(kv_heads, d, page_size, is_v, page, offset)
    return dequantise(pool[code], pool[byte])


def attend(q, k, v):
    """One row over its keys: q [heads, d], k and v [n, kv_heads, d] -> the
    outputs [heads, d], sum p |v| [heads, d], and per head the largest
    sum |q_i k_i| / sqrt(d)."""
    heads, d = q.shape
    n, kv_heads = k.shape[:2]
    out, mag, big = np.zeros((heads, d)), np.zeros((heads, d)), np.zeros(heads)
    if n == 0:
        return out, mag, big
    for h in range(heads):
        kk, vv = k[:, h * kv_heads // heads], v[:, h * kv_heads // heads]
        s = kk @ q[h] / np.sqrt(d)
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h], mag[h] = p @ vv, p @ np.abs(vv)
        big[h] = (np.abs(kk) @ np.abs(q[h])).max() / np.sqrt(d)
    return out, mag, big


def tolerance(out, mag, big, n, d, vmax, q_dtype, out_dtype):
    """How far a result may be off, element by element, in 32-bit arithmetic.

    A score is a sum of d products in fp32, scaled by a few fp32 factors: off
    by (d + 8) 2^-24 sum|q k| / sqrt(d) =: es, and e^s by that relatively (and
    as much again through the sum it is divided by).  fp32 q with a bf16 result
    is used to 16 bits: 2^-17 more of the same sum.  The probabilities enter
    with 11 bits (2^-12) for a bf16 result and 22 (2^-23) for fp32, and where
    they fall below f16's normal range with an absolute 2^-25 against a
    largest of at least 2^8.  Sums over n keys, exponentials and the joins add
    (n / 16 + 64) 2^-24.  The result is rounded once."""
    es = (d + 8) * 2.0 ** -24 * big
    if q_dtype == "f32" and out_dtype == "bf16":
        es = es + 2.0 ** -17 * big
    p = 2.0 ** -12 if out_dtype == "bf16" else 2.0 ** -23
    rel = 2 * es + p + (n / 16 + 64) * 2.0 ** -24
    half_step = 2.0 ** -8 if out_dtype == "bf16" else 2.0 ** -24
    tol = mag * rel[:, None] + n * 2.0 ** -32 * vmax
    return tol + half_step * (np.abs(out) + tol)
