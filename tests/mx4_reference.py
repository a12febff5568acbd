"""The MXFP4 operators in 64 bits with numpy, for the tests: codes one at a time from the definition."""
import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantize(x, rule="floor"):
    """x [rows, cols] float64 -> (codes [rows, cols] 0..15, scale bytes [rows, cols / 32])."""
    v = np.asarray(x, np.float64).reshape(x.shape[0], -1, 32)
    codes = np.zeros(v.shape, np.uint8)
    scales = np.zeros(v.shape[:2], np.uint8)
    finite = np.isfinite(v).all(-1)
    top = np.where(finite, np.abs(v).max(-1), 0)
    part, e = np.frexp(top)
    e = np.where(top > 0, e - 1, -1000)  # top in [2^e, 2^(e+1))
    if rule == "noclip":
        e = e + (part > 0.75)
    e = np.clip(e - 2, -126, 125)
    scales[:] = np.where(finite, e + 127, 255)
    a = np.abs(np.ldexp(np.where(finite[..., None], v, 0), -e[..., None]))
    # nearest of the eight magnitudes, ties to the even code: the number of borders that lie below
    for border, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5, False)):
        codes += (a >= border if up else a > border).astype(np.uint8)
    codes |= np.where(np.signbit(v) & finite[..., None], 8, 0).astype(np.uint8)
    return codes.reshape(x.shape), scales


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def tile(scales, k):
    """[..., rows, k / 32] -> [..., ceil(k / 128), rows, 4]."""
    words = (k + 127) // 128
    full = np.zeros((*scales.shape[:-1], 4 * words), np.uint8)
    full[..., : scales.shape[-1]] = scales
    return np.ascontiguousarray(np.moveaxis(full.reshape(*scales.shape[:-1], words, 4), -2, -3))


def values(blocks, scales):
    """Packed blocks [..., k / 2] and scale rows [..., k / 32] as the products read them, in 64 bits."""
    table = np.concatenate([E2M1, -E2M1])
    codes = np.empty((*blocks.shape[:-1], 2 * blocks.shape[-1]), np.uint8)
    codes[..., 0::2], codes[..., 1::2] = blocks & 15, blocks >> 4
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return table[codes] * np.repeat(s, 32, -1)


def swiglu(gate_up, alpha, limit):
    g, u = np.asarray(gate_up, np.float64)[..., 0::2], np.asarray(gate_up, np.float64)[..., 1::2]
    g = np.where(g > limit, limit, g)
    u = np.where(u > limit, limit, np.where(u < -limit, -limit, u))
    with np.errstate(over="ignore", invalid="ignore"):
        return g * (1 / (1 + np.exp(-float(np.float32(alpha)) * g))) * (u + 1)
