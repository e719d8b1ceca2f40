"""The microscaled 4-bit formats in 64 bits, written from their definitions with numpy: what the tests compare with."""
import numpy as np
import torch

E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
E4M3 = np.array([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)])[:127]
BLOCK = {"mxfp4": 32, "nvfp4": 16}


def nearest(a, grid):
    """Index of the grid value nearest to each a >= 0 (beyond the end: the last); of two equally near, the even index."""
    up = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    mid = (grid[up - 1] + grid[up]) / 2
    return np.where((a > mid) | ((a == mid) & (up % 2 == 0)), up, up - 1)


def bf16(v):
    """A positive double rounded to 8 bits."""
    with np.errstate(divide="ignore"):
        step = np.exp2(np.floor(np.log2(np.where(v > 0, v, 1))) - 7)
    return np.round(v / step) * step


def quantize(fmt, x):
    """x [rows, cols] (doubles holding 16-bit values) -> (codes 0..15, block scale bytes, row scales or None)."""
    rows, cols = x.shape
    b = x.reshape(rows, cols // BLOCK[fmt], BLOCK[fmt])
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    row = None
    if fmt == "mxfp4":
        _, e = np.frexp(top)
        byte = np.where(top > 0, np.maximum(e - 3 + 127, 0), 0)
        scale = np.exp2(byte - 127.0)
        byte = np.where(bad, 0xFF, byte)
    else:
        row = np.maximum(bf16(top.max(1) / 2688), 2.0 ** -110)
        byte = nearest(top / (6 * row[:, None]), E4M3)
        scale = E4M3[byte] * row[:, None]
        byte = np.where(bad, 0x7F, byte)
    q = nearest(np.abs(b) / np.where(scale > 0, scale, 1)[..., None], E2M1)
    q = np.where((scale > 0)[..., None], q, 0)
    codes = q + 8 * np.signbit(b)
    return np.where(bad[..., None], 0, codes).reshape(rows, cols).astype(np.uint8), byte.astype(np.uint8), row


def values(fmt, codes, byte, row=None):
    """Quantized parts -> doubles."""
    v = E2M1[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    if fmt == "mxfp4":
        s = np.where(byte == 0xFF, np.nan, np.exp2(byte.astype(np.float64) - 127))
    else:
        s = np.where(byte == 0x7F, np.nan, E4M3[np.minimum(byte, 126)]) * (1.0 if row is None else np.asarray(row, np.float64)[:, None])
    return v * np.repeat(s, BLOCK[fmt], 1)


def pack(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    return np.stack([packed & 15, packed >> 4], -1).reshape(packed.shape[0], -1)


def tile(byte):
    """Row-major block scales -> the tiled order, byte by byte from its definition (unnamed places: 0)."""
    rows, blocks = byte.shape
    tiles = -(-blocks // 4)
    out = np.zeros(-(-rows // 128) * tiles * 512, np.uint8)
    for r in range(rows):
        for k in range(blocks):
            out[(r // 128 * tiles + k // 4) * 512 + 16 * (r % 32) + 4 * (r % 128 // 32) + k % 4] = byte[r, k]
    return out


def untile(tiled, rows, blocks):
    tiles = -(-blocks // 4)
    r, k = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    return tiled[(r // 128 * tiles + k // 4) * 512 + 16 * (r % 32) + 4 * (r % 128 // 32) + k % 4]


def random_operand(fmt, rows, cols, seed, row_scales=True):
    """A quantized tensor of random codes and scales, and its values: (packed, tiled, row scales or None, doubles)."""
    g = np.random.default_rng(seed)
    codes = g.integers(0, 16, (rows, cols), dtype=np.uint8)
    byte = (g.integers(120, 130, (rows, cols // 32)) if fmt == "mxfp4" else g.integers(8, 0x7F, (rows, cols // 16))).astype(np.uint8)
    row = (0.25 + g.random(rows)).astype(np.float32) * np.float32(1.0 if fmt == "mxfp4" else 0.01) if row_scales else None
    v = values(fmt, codes, byte, row if fmt == "nvfp4" else None)
    if fmt == "mxfp4" and row is not None:
        v = v * row[:, None].astype(np.float64)
    return pack(codes), tile(byte), row, v


def cuda(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()
