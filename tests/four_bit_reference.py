"""The 4-bit format in numpy and float64: codes and scales of values, pages of a cache, and their append."""
from __future__ import annotations

import numpy as np

PAGE, D, GROUP, PAGE_BYTES = 16, 128, 32, 2176
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def encode(x):
    """Codes and scale bytes of x [..., n], by search: every scale that is written, every level."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, GROUP)
    top = np.abs(g).max(-1)
    e = np.full(top.shape, 13)
    for k in range(13, -24, -1):
        e = np.where(top <= 7 * 2.0 ** k, k, e)
    y = np.minimum(np.abs(g) / (2.0 ** e)[..., None], 8)  # beyond 6 the nearest is 6, however far
    far = np.abs(y[..., None] - LEVELS)
    best = far.min(-1, keepdims=True)
    tied = far == best  # of two levels as near, the one with the even code
    code = np.where(tied[..., ::2].any(-1), 2 * tied[..., ::2].argmax(-1), tied.argmax(-1))
    code = code + 8 * np.signbit(g)
    return code.reshape(x.shape).astype(np.uint8), (e + 127).astype(np.uint8)


def decode(code, scale):
    with np.errstate(over="ignore"):
        value = LEVELS[code % 8] * np.where(code > 7, -1.0, 1.0)
        power = np.where(scale == 255, np.nan, 2.0 ** (scale.astype(np.float64) - 127))
        return value * np.repeat(power, GROUP, -1)


def pack(code):
    return (code[..., ::2] | code[..., 1::2] << 4).astype(np.uint8)


def unpack(b):
    return np.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], -1)


def write_slot(page, slot, k, v):
    """Puts K and V [128] of one token into a kv head's page [PAGE_BYTES]."""
    (kc, ks), (vc, vs) = encode(k), encode(v)
    page[64 * slot:64 * slot + 64] = pack(kc)
    vb = pack(vc)
    for piece in range(16):
        at = 1024 + 256 * (slot // 4) + 16 * piece + 4 * (slot % 4)
        page[at:at + 4] = vb[4 * piece:4 * piece + 4]
    page[2048 + 4 * slot:2048 + 4 * slot + 4] = ks
    page[2112 + slot::16][:4] = vs


def read_pages(pages):
    """K and V [..., 16, 128] in float64 of pages [..., PAGE_BYTES]."""
    lead = pages.shape[:-1]
    k = decode(unpack(pages[..., :1024].reshape(*lead, PAGE, 64)), pages[..., 2048:2112].reshape(*lead, PAGE, 4))
    vb = np.swapaxes(pages[..., 1024:2048].reshape(*lead, 4, 16, 4, 4), -3, -2).reshape(*lead, PAGE, 64)
    v = decode(unpack(vb), np.swapaxes(pages[..., 2112:].reshape(*lead, 4, PAGE), -1, -2))
    return k, v


def to_pages(k, v):
    """Pages [n, KV, PAGE_BYTES] of K and V [n, KV, 16, 128]."""
    (kc, ks), (vc, vs) = encode(k), encode(v)
    lead = k.shape[:-2]
    vb = np.swapaxes(pack(vc).reshape(*lead, 4, 4, 16, 4), -3, -2)
    return np.concatenate([pack(kc).reshape(*lead, -1), vb.reshape(*lead, -1), ks.reshape(*lead, -1),
                           np.swapaxes(vs, -1, -2).reshape(*lead, -1)], -1)
