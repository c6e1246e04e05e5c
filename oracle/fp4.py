"""Microscaled 4-bit floating point and the norms around a block, restated in numpy for the tests:
decisions in 64 bits, the f32 roundings that the operators define made one by one.

A quantised matrix is (elements, scales, row scales): f64 element values [M, K], stored scale bytes [M, blocks],
f32 [M] or None."""
import numpy as np

VALUES = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], np.float64)
BLOCK = {"mx": 32, "nv": 16}


def e2m1(v):
    """Codes of the nearest elements, ties to the even code, saturating."""
    d = np.abs(np.abs(v)[..., None] - VALUES)
    best = d.min(-1, keepdims=True)
    # of two elements at the same distance the one with the even code
    order = np.where(d == best, np.arange(8) % 2, 2)
    return (order.argmin(-1) | (np.signbit(v).astype(np.int64) << 3)).astype(np.uint8)


def element(codes):
    return np.where(codes & 8, -1.0, 1.0) * VALUES[codes & 7]


def e4m3_values():
    """The 256 values of e4m3 (no infinities, 0x7F and 0xFF NaN)."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v[[0x7F, 0xFF]] = np.nan
    return np.where(b & 128, -v, v)


def to_e4m3(t):
    """Codes of non-negative f64 numbers, nearest, ties to even."""
    table = e4m3_values()[:0x7F]
    hi = np.clip(np.searchsorted(table, t), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = t - table[lo], table[hi] - t
    return np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)


def floor_log2(v):
    return np.frexp(v)[1] - 1


def quantise(x, fmt):
    """x [M, K] of f16 or f32 values (any float array) -> codes [M, K], scale bytes [M, K / B], row scales."""
    x = np.asarray(x, np.float64)
    m, k = x.shape
    b = x.reshape(m, k // BLOCK[fmt], BLOCK[fmt])
    amax = np.abs(b).max(-1)
    bad = ~np.isfinite(b).all(-1)
    safe = np.where(np.isfinite(amax), amax, 0.0)
    if fmt == "mx":
        e = np.where(safe > 0, floor_log2(np.where(safe > 0, safe, 1.0)) - 2, -127).clip(-127, 127)
        codes = e2m1(np.where(bad[..., None], 0.0, b) * 2.0 ** -e.astype(np.float64)[..., None])
        codes = np.where(bad[..., None], 0, codes)
        return codes.reshape(m, k).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8), None
    row = safe.max(-1)
    row_bad = bad.any(-1)
    least = np.ceil(np.log2(np.where(row > 0, row, 1.0) / 2688.0))
    least = np.where(row > 2688.0 * 2.0 ** least, least + 1, least)
    least = np.where(row <= 2688.0 * 2.0 ** (least - 1), least - 1, least)
    g = np.where(row > 0, 2.0 ** np.maximum(least, -100), 1.0)
    t = (safe.astype(np.float32) / (6 * g).astype(np.float32)[:, None]).astype(np.float64)
    s8 = to_e4m3(t)
    s = (e4m3_values()[s8] * g[:, None])[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(s > 0, (np.where(np.isfinite(b), b, 0.0).astype(np.float32) / s.astype(np.float32)).astype(np.float64), np.copysign(0.0, b))
    codes = np.where(row_bad[:, None, None] | (s == 0), 0, e2m1(q))
    return (codes.reshape(m, k).astype(np.uint8), np.where(row_bad[:, None], 0x7F, s8).astype(np.uint8),
            np.where(row_bad, np.nan, g).astype(np.float32))


def scale_values(scales, fmt):
    if fmt == "mx":
        return np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return e4m3_values()[scales]


def values(codes, scales, row, fmt):
    """f64 [M, K], exactly."""
    v = element(codes) * np.repeat(scale_values(scales, fmt), BLOCK[fmt], axis=1)
    return v if row is None else v * row.astype(np.float64)[:, None]


def pack(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def tile_scales(scales, fill=0):
    """[M, blocks] bytes -> [ceil(M / 128), ceil(blocks / 4), 512]; `fill` in the rows behind the last."""
    m, blocks = scales.shape
    tiles = np.zeros((-(-m // 128), -(-blocks // 4), 512), np.uint8)
    for r in range(tiles.shape[0] * 128):
        for c in range(tiles.shape[1] * 4):
            tiles[r // 128, c // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + c % 4] = scales[r, c] if r < m and c < blocks else fill if r >= m else 0
    return tiles


def untile_scales(tiles, m, blocks):
    t = tiles.reshape(tiles.shape[0], tiles.shape[1], 32, 4, 4).transpose(0, 3, 2, 1, 4).reshape(tiles.shape[0] * 128, -1)
    return t[:m, :blocks]


def rmsnorm_block(x, residual, post, gate, pre, alpha, eps, seqlen, round16):
    """(stream, next input before it is rounded or quantised) in f32; round16 rounds an f32 array to the 16-bit type and back."""
    f = np.float32

    def unit(v):
        mean = (v.astype(np.float64) ** 2).mean(-1, keepdims=True)
        with np.errstate(divide="ignore", invalid="ignore"):
            return v * (1.0 / np.sqrt(mean + np.float64(f(eps)))).astype(f)

    with np.errstate(invalid="ignore", over="ignore"):
        u = x.astype(f)
        if post is not None:
            u = unit(u) * post.astype(f)
        if gate is not None:
            rows = np.arange(len(x)) // seqlen if seqlen > 0 else np.zeros(len(x), int)
            u = gate.reshape(-1, x.shape[1]).astype(f)[rows] * u
        stream = round16(f(alpha) * residual.astype(f) + u)
        return stream, None if pre is None else unit(stream) * pre.astype(f)
