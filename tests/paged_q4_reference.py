"""Plain restatement of the 4-bit pages for the tests: a row's codes and words from fp32 values, step by
step in numpy's fp32, and a page's values from its bytes."""
import numpy as np
import torch

import paged_reference as ref

Q4_GROUP = 0x400
MOST = 2112.0      # the largest scale
NAN_WORD = 0x7FE0


def page_bytes(hkv, hd, page):
    return -(-(2 * hkv * page * (hd // 2 + hd // 16)) // 128) * 128


def encode(x):
    """(codes, scales, zeros) of fp32 x [..., hd]: codes [..., hd], one scale (NaN: not held) and one zero
    point per 32 values."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    with np.errstate(invalid="ignore", over="ignore"):
        lo, hi = np.minimum(g.min(-1), np.float32(0)), np.maximum(g.max(-1), np.float32(0))
        f = (hi - lo) * np.float32(1 / 15)
        good = np.isfinite(g).all(-1) & (f <= MOST)
        f = np.where(good, f, np.float32(0))
        _, e = np.frexp(f)
        k = np.maximum(e, -13) - 6
        d = np.ldexp(np.ceil(np.ldexp(f, -k)), k).astype(np.float32)
        by = np.where(d > 0, d, np.float32(1))
        z = np.where(good, np.rint(-lo / by), 0)
        code = np.clip(np.rint(g / by[..., None]) + z[..., None], 0, 15)
        code = np.where(good[..., None], code, 0)
    return code.reshape(x.shape).astype(np.int64), np.where(good, d, np.nan), z.astype(np.int64)


def values(code, scale, zero):
    """What they stand for, float64 [..., hd]."""
    g = code.reshape(*code.shape[:-1], code.shape[-1] // 32, 32) - zero[..., None]
    with np.errstate(invalid="ignore"):
        return (g * np.asarray(scale, np.float64)[..., None]).reshape(code.shape)


def places(hd):
    """(byte, shift) of each dim's code inside a row."""
    d = np.arange(hd)
    groups = min(hd // 32, 4)
    r = d % 128
    dword = 16 * (d // 128) + r % 32 // 8 * groups + r // 32
    bit = 16 * (d % 2) + 4 * (d % 8 // 2)
    return 4 * dword + bit // 8, bit % 8


def split(hkv, hd, page, raw):
    """(codes [.., 2, kv heads, page, hd], words [.., 2, kv heads, page, hd / 32]) of page bytes (a CPU tensor)."""
    rows, lead = 2 * hkv * page, raw.shape[:-1]
    b = raw.numpy()
    byte, shift = places(hd)
    code = b[..., : rows * hd // 2].reshape(*lead, 2, hkv, page, hd // 2)[..., byte] >> shift.astype(np.uint8) & 15
    word = np.ascontiguousarray(b[..., rows * hd // 2 : rows * (hd // 2 + hd // 16)]).view(np.uint16)
    return code.astype(np.int64), word.reshape(*lead, 2, hkv, page, hd // 32).astype(np.int64)


def decode(fmt, hkv, hd, page, raw, plain=ref.decode):
    """paged_reference.decode that knows this format too."""
    if fmt != Q4_GROUP:
        return plain(fmt, hkv, hd, page, raw)
    code, word = split(hkv, hd, page, raw)
    scale = (word & 0xFFE0).astype(np.uint16).view(np.float16).astype(np.float64)
    return torch.from_numpy(values(code, scale, word & 15))
