"""The 4-bit block-scaled formats in 64 bits (numpy), from their definition."""
import numpy as np

from rocwmma_b200 import MXF4, NVF4

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
BLOCK = {MXF4: 32, NVF4: 16}
# every finite, non-negative E4M3 value by its byte
E4M3 = np.array([(8 + b % 8) * 2.0 ** (b // 8 - 10) if b >= 8 else b * 2.0 ** -9 for b in range(127)])


def nearest(values, x):
    """Index of the nearest of ascending `values`, ties to the even index; beyond the last: the last."""
    hi = np.clip(np.searchsorted(values, x), 1, len(values) - 1)
    lo = hi - 1
    below, above = x - values[lo], values[hi] - x
    return np.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)


def quantize(fmt, x, exponent=0):
    """x [rows, k] -> (codes [rows, k] 0..15, scale bytes [rows, blocks], values [rows, k])."""
    rows, k = x.shape
    block = BLOCK[fmt]
    blocks = -(-k // block)
    y = np.zeros((rows, blocks * block))
    with np.errstate(invalid="ignore"):
        y[:, :k] = x.astype(np.float64) * 2.0 ** -exponent
        y = y.reshape(rows, blocks, block)
        top = np.abs(y).max(2)
    bad = ~np.isfinite(top)
    top = np.where(bad, 0, top)
    y = np.where(bad[..., None], 0, y)
    if fmt == MXF4:
        e = np.maximum(np.frexp(top)[1] - 1 - 2, -127)
        e = np.where(top == 0, -127, e)
        byte, scale = e + 127, 2.0 ** e
        byte = np.where(bad, 255, byte)
    else:
        byte = nearest(E4M3, top / 6)
        scale = E4M3[byte]
        byte = np.where(bad, 127, byte)
    with np.errstate(invalid="ignore", divide="ignore"):
        v = np.where(scale[..., None] > 0, y / scale[..., None], 0)
    code = nearest(E2M1, np.abs(v))
    values = np.where(v < 0, -1, 1) * E2M1[code] * scale[..., None] * 2.0 ** exponent
    values = np.where(bad[..., None], np.nan, values)
    code = code + 8 * (v < 0)
    return code.reshape(rows, -1)[:, :k], byte.astype(np.uint8), values.reshape(rows, -1)[:, :k]


def pack(fmt, codes, scale_bytes):
    """(codes, scales) as the library holds them."""
    rows, k = codes.shape
    full = np.zeros((rows, -(-k // 32) * 32), np.uint8)
    full[:, :k] = codes
    packed = full[:, 0::2] | (full[:, 1::2] << 4)
    tiles, groups = -(-rows // 128), -(-scale_bytes.shape[1] // 4)
    s = np.zeros((tiles * 128, groups * 4), np.uint8)
    s[:rows, :scale_bytes.shape[1]] = scale_bytes
    s = s.reshape(tiles, 4, 32, groups, 4).transpose(0, 3, 2, 1, 4)
    return packed.reshape(-1), np.ascontiguousarray(s).reshape(-1)


def unpack(fmt, rows, k, codes, scales):
    """(codes [rows, k], scale bytes [rows, blocks]) of a packed operand."""
    c = codes.reshape(rows, -1)
    full = np.stack((c & 15, c >> 4), 2).reshape(rows, -1)
    blocks = -(-k // BLOCK[fmt])
    tiles, groups = -(-rows // 128), -(-blocks // 4)
    s = scales.reshape(tiles, groups, 32, 4, 4).transpose(0, 3, 2, 1, 4).reshape(tiles * 128, groups * 4)
    return full[:, :k], s[:rows, :blocks]


def values(fmt, codes, scale_bytes):
    """What codes and scale bytes stand for."""
    if fmt == MXF4:
        scale = np.where(scale_bytes == 255, np.nan, 2.0 ** (scale_bytes.astype(np.float64) - 127))
    else:
        scale = np.append(E4M3, np.nan)[np.minimum(scale_bytes, 127)]
    v = np.where(codes >= 8, -1, 1) * E2M1[codes % 8]
    return v * np.repeat(scale, BLOCK[fmt], 1)[:, :codes.shape[1]]
