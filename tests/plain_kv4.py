"""Keys and values held in 4 bits, plainly: blocks of 32 elements as codes and a scale, the pages' bytes, attention in float64."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def block(x):
    """32 numbers (float32) -> (codes 0..15, scale byte)."""
    x = np.asarray(x, dtype=np.float64)
    if not np.isfinite(x).all():
        return np.zeros(32, dtype=np.uint8), 255
    big = np.abs(x).max()
    e = -124
    if big > 0:
        e = max(-124, int(np.frexp(big)[1]) - 1 - 2)
    y = x * 2.0 ** -e
    d = np.abs(np.abs(y)[:, None] - GRID)
    near = np.where(d == d.min(-1, keepdims=True), np.arange(8) % 2, 2)       # the nearest, among two of them the even code
    return (near.argmin(-1) | np.where(np.signbit(y), 8, 0)).astype(np.uint8), e + 127


def value(codes, byte):
    """What codes and a scale byte stand for, float64."""
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    return np.full(len(codes), np.nan) if byte == 255 else v * 2.0 ** (int(byte) - 127)


def held(rows):
    """Rows [..., hd] as the cache holds them: `value` of `block` of every 32 elements, in one go."""
    rows = np.asarray(rows, dtype=np.float64)
    x = rows.reshape(rows.shape[:-1] + (-1, 32))
    fine = np.isfinite(x).all(-1, keepdims=True)
    x = np.where(fine, x, 0.0)
    big = np.abs(x).max(-1, keepdims=True)
    e = np.where(big > 0, np.maximum(-124, np.frexp(big)[1] - 3), -124)
    y = x * 2.0 ** -e.astype(np.float64)
    d = np.abs(np.abs(y)[..., None] - GRID)
    even = np.where(d == d.min(-1, keepdims=True), np.arange(8) % 2, 2)       # the nearest, among two of them the even code
    v = np.where(np.signbit(y), -1.0, 1.0) * GRID[even.argmin(-1)] * 2.0 ** e.astype(np.float64)
    return np.where(fine, v, np.nan).reshape(rows.shape)


def put(part, t, k, v):
    """Token t's key and value rows [hd] into the bytes of one head's part of a page (uint8 [68 hd])."""
    hd = len(k)
    m = hd // 32
    kc, ks = part[:1024 * m].reshape(64, 16 * m), part[1024 * m:1088 * m].reshape(16, m, 4)
    vc, vs = part[1088 * m:2112 * m].reshape(8, 4 * m, 8, 4), part[2112 * m:].reshape(8, m, 8)
    for b in range(m):
        codes, s = block(k[32 * b:32 * b + 32])
        kc[t, 16 * b:16 * b + 16] = codes[0::2] | codes[1::2] << 4
        half, octet, four, r = t // 32, t % 32 // 8, t % 8 // 4, t % 4
        ks[4 * octet + r, b, 2 * half + four] = s
        codes, s = block(v[32 * b:32 * b + 32])
        vc[t // 8, 4 * b:4 * b + 4, t % 8] = (codes[0::2] | codes[1::2] << 4).reshape(4, 4)
        vs[t // 8, b, t % 8] = s


def attention(q, k, v, scale, first, window=None):
    """Rows q [n, nq, hd] of the tokens at first.. over k, v [tokens, nkv, hd], float64.  Returns the output, the same sum with
    |v|, and the largest scale * sum |q k| of a row: what roundings are counted against."""
    n, nq, hd = q.shape
    G = nq // k.shape[1]
    out, size, most = np.zeros_like(q, dtype=np.float64), np.zeros_like(q, dtype=np.float64), 0.0
    for h in range(nq if n else 0):
        kk, vv = k[:first + n, h // G], v[:first + n, h // G]
        at, key = np.arange(first, first + n)[:, None], np.arange(first + n)[None, :]
        seen = (key <= at) & ((key > at - window) if window is not None else True)
        with np.errstate(invalid="ignore"):
            s = np.where(seen, q[:, h] @ kk.T * scale, -np.inf)
            e = np.exp(s - s.max(-1, keepdims=True))
            e = np.where(np.isnan(s).any(-1, keepdims=True), np.nan, e)
            # what a row does not see has no part in it, NaN or not: 0 there, the rest as it is
            clean, bad = np.where(np.isnan(vv), 0.0, vv), np.isnan(vv)
            out[:, h] = np.where(seen.astype(float) @ bad.astype(float) > 0, np.nan, e @ clean / e.sum(-1, keepdims=True))
            size[:, h] = e @ np.abs(clean) / e.sum(-1, keepdims=True)
            most = max(most, float((np.abs(np.nan_to_num(kk)) @ np.abs(q[:, h]).T).max()) * scale)
    return out, size, most
