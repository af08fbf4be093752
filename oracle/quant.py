"""64-bit plain forms of the 4-bit cache: its numbers, its bytes, and the head norms with rotation.

Rows are float64 arrays [..., D]; codes uint8 [..., D], scale bytes uint8 [..., D / 32]; pages uint8
[pages, H, block * (D + D / 16)].
"""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
LARGEST_EXPONENT = {'bf16': 127, 'fp16': 15}


def quantize(x, dtype):
    """(codes, scale bytes) of rows x [..., D]."""
    x = np.asarray(x, np.float64)
    blocks = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = np.abs(blocks).max(-1)
    bad = ~np.isfinite(top)
    mantissa, exponent = np.frexp(np.where(bad | (top == 0), 1.0, top))       # top = mantissa 2^exponent, in [0.5, 1)
    e = exponent - 1 + (2 * mantissa >= 1.75) - 2
    e = np.where(top == 0, -127, np.clip(e, -127, LARGEST_EXPONENT[dtype] - 2))
    y = np.abs(np.where(bad[..., None], 0.0, blocks)) / 2.0 ** e[..., None]
    # the nearest level; of two as near the one with the even code
    distance = np.abs(y[..., None] - LEVELS)
    near = distance == distance.min(-1, keepdims=True)
    first = near.argmax(-1)
    last = 7 - near[..., ::-1].argmax(-1)
    codes = np.where(first % 2 == 0, first, last) + 8 * np.signbit(blocks)
    codes = np.where(bad[..., None], 0, codes).astype(np.uint8).reshape(x.shape)
    return codes, np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, scales):
    """The numbers that codes and scale bytes stand for."""
    size = np.where(codes & 8, -1.0, 1.0) * LEVELS[codes & 7]
    factor = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return size * np.repeat(factor, 32, -1)


def _places(block, D):
    """Byte and half (0 low, 1 high) of every (row, element) of K and V in a page of one head, bytes of every (row, block)
    of their scales; written element by element from the format."""
    half = block * D // 2
    byte, high = np.zeros((2, block, D), np.int64), np.zeros((2, block, D), np.int64)
    scale = np.zeros((2, block, D // 32), np.int64)
    for r in range(block):
        group, g, j = r // 16, r % 16 // 4, r % 4
        for d in range(D):
            byte[0, r, d], high[0, r, d] = r * D // 2 + d // 2, d % 2
            p, m = d // 32, d % 16
            byte[1, r, d] = half + group * 8 * D + ((16 * g + m) * 4 + j) * (D // 32) + p
            high[1, r, d] = d % 32 // 16
        for p in range(D // 32):
            scale[0, r, p] = 2 * half + r * (D // 32) + p
            scale[1, r, p] = 2 * half + block * (D // 32) + r * (D // 32) + p
    return byte, high, scale


def write_page(page, rows, k, v, D):
    """Writes (codes, scale bytes) k and v [n, ...] of one head into rows `rows` of its bytes `page`."""
    byte, high, scale = _places(page.size // (D + D // 16), D)
    for which, (codes, scales) in enumerate((k, v)):
        for i, r in enumerate(rows):
            for half in (0, 1):
                at = high[which, r] == half
                place = byte[which, r][at]
                keep = 0xf0 if half == 0 else 0x0f
                page[place] = (page[place] & keep) | (codes[i][at] << (4 * half))
            page[scale[which, r]] = scales[i]


def read_pages(pages, D):
    """K and V rows [pages, block, H, D] of a pool as the numbers they stand for."""
    block = pages.shape[2] // (D + D // 16)
    byte, high, scale = _places(block, D)
    out = []
    for which in (0, 1):
        codes = (pages[:, :, byte[which]] >> (4 * high[which]).astype(np.uint8)) & 15
        out.append(values(codes, pages[:, :, scale[which]]).transpose(0, 2, 1, 3))
    return out


def norm_rope(x, weight, cos, sin, eps):
    """(out, terms): x [..., D] normalised (weight None: as it is) and rotated by cos, sin [..., D]; terms bounds the sum
    of the magnitudes of the two products of each element."""
    half = x.shape[-1] // 2
    y = x if weight is None else x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * weight
    turned = np.concatenate([-y[..., half:], y[..., :half]], -1)
    return y * cos + turned * sin, np.abs(y * cos) + np.abs(turned * sin)
