"""A quantised KV cache in numpy, element by element from the header's description of it."""
import numpy as np

Q4_0, Q8_0 = 3, 4
BITS = {Q4_0: 4, Q8_0: 8}


def block_bytes(kv, hd):
    return 16 * hd // 32 * (18 if kv == Q4_0 else 34)


def code_place(kind, kv, hd, p, e):
    """(byte, shift) of the code of position p, dim e in a block."""
    bits = BITS[kv]
    if kind == "k":
        lane = 4 * (p % 8) + e % 32 // 8
        if bits == 4:
            i, byte, shift = (p // 8) * (hd // 32) + e // 32, e % 8 // 2, 4 * (e % 2)
        else:
            i, byte, shift = 2 * ((p // 8) * (hd // 32) + e // 32) + e % 8 // 4, e % 4, 0
    else:
        lane, byte = 4 * (e % 16 // 2) + p % 8 // 2, 2 * (p % 2) + p // 8
        i, shift = (e // 16, 4 * (e % 2)) if bits == 4 else (2 * (e // 16) + e % 2, 0)
    words = hd * bits // 64
    at = 512 * (i // 4) + (16 if i < words // 4 * 4 else 8) * lane + 4 * (i % 4)
    return at + byte, shift


def tables(kind, kv, hd):
    """Bytes and shifts [16][hd], and byte offsets of the scales [16][hd / 32]."""
    at = np.array([[code_place(kind, kv, hd, p, e) for e in range(hd)] for p in range(16)])
    start = 16 * hd * BITS[kv] // 8
    scale = np.array([[start + 2 * ((2 * (p % 8) + p // 8) * (hd // 32) + k) for k in range(hd // 32)] for p in range(16)])
    return at[..., 0], at[..., 1], scale


def quantise(kv, x):
    """x [..., hd] fp32 -> codes and f16 scales, in 64 bits from the definition."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32).astype(np.float32)
    mag = np.abs(g)
    with np.errstate(all="ignore"):
        if kv == Q4_0:
            first = np.argmax(mag == mag.max(-1, keepdims=True), -1)[..., None]
            d = np.take_along_axis(g, first, -1) / np.float32(-8)
        else:
            d = mag.max(-1, keepdims=True) * (np.float32(1) / np.float32(127))
        scale = np.clip(d, -65504, 65504).astype(np.float16)
        bad = ~np.isfinite(g).all(-1, keepdims=True)
        s = scale.astype(np.float64)
        q = np.where(bad | (s == 0), 0.0, np.rint(g.astype(np.float64) / np.where(s == 0, 1.0, s)))
    lo, hi, zero = (-8, 7, 8) if kv == Q4_0 else (-127, 127, 128)
    codes = (np.clip(np.nan_to_num(q), lo, hi) + zero).astype(np.uint8)
    scale = np.where(bad, np.array(0x7FFF, np.uint16).view(np.float16), scale)
    return codes.reshape(x.shape), scale[..., 0]


def write(cache, kind, kv, hd, slot, head, pos, codes, scales):
    """One row's codes [hd] and scales [hd / 32] into cache [slots][heads][cap / 16][bytes] (uint8)."""
    at, shift, sat = tables(kind, kv, hd)
    blk, p = cache[slot, head, pos // 16], pos % 16
    mask = 15 if BITS[kv] == 4 else 255
    for e in range(hd):
        blk[at[p, e]] = (int(blk[at[p, e]]) & ~(mask << shift[p, e]) & 255) | (int(codes[e]) << shift[p, e])
    for k in range(hd // 32):
        blk[sat[p, k]:sat[p, k] + 2] = np.frombuffer(np.float16(scales[k]).tobytes(), np.uint8)


def values(blocks, kind, kv, hd):
    """blocks [n][bytes] -> [n][16][hd] in 64 bits."""
    at, shift, sat = tables(kind, kv, hd)
    bits = BITS[kv]
    codes = (blocks[:, at] >> shift.astype(np.uint8)) & (2 ** bits - 1)
    scale = (blocks[:, sat].astype(np.uint16) | blocks[:, sat + 1].astype(np.uint16) << 8).view(np.float16).astype(np.float64)
    with np.errstate(invalid="ignore"):
        return (codes.astype(np.float64) - 2 ** (bits - 1)) * np.repeat(scale, 32, -1)
