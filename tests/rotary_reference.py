"""Plain 64-bit restatement of rotary positions for the tests."""
import math

import numpy as np


def turns(dims, theta=1e6, scaling="plain", factor=1.0, original=0, low=1.0, high=32.0):
    half = dims // 2
    if scaling == "base" and half > 1:
        theta = theta * factor ** (dims / (dims - 2))
    out = []
    for j in range(half):
        f = theta ** (-2 * j / dims)
        if scaling == "linear":
            f = f / factor
        if scaling == "ramp":
            pair = lambda r: dims * math.log(original / (r * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
            a, b = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), dims - 1)
            b = max(b, a + 0.001)
            away = min(max((j - a) / (b - a), 0), 1)
            f = f * (1 - away) + f / factor * away
        if scaling == "bands":
            keep = min(max((original * f / (2 * math.pi) - low) / (high - low), 0), 1)
            f = f * keep + f / factor * (1 - keep)
        out.append(f / (2 * math.pi))
    return np.array(out)


def rotate(x, positions, table, layout, amplitude=1.0):
    """(y, bound): x [rows, heads, hd] turned in 64 bits, and how far an fp32 result may be off: one rounding
    (2^-24 of the value, which is at most its pair's sum) and the angle's, 2^-53 of the turns made, here and there."""
    x = np.asarray(x, np.float64)
    half = len(table)
    made = np.asarray(positions, np.float64)[:, None] * table
    angle = 2 * np.pi * (made - np.rint(made))[:, None]
    c, s = np.cos(angle) * amplitude, np.sin(angle) * amplitude
    i = (np.arange(half) * 2, np.arange(half) * 2 + 1) if layout == "neighbours" else (np.arange(half), np.arange(half) + half)
    y, bound = x.copy(), np.zeros_like(x)
    a, b = x[..., i[0]], x[..., i[1]]
    y[..., i[0]], y[..., i[1]] = a * c - b * s, a * s + b * c
    size = (np.abs(a) + np.abs(b)) * abs(amplitude)
    off = size * (2.0**-24 + 4 * np.pi * 2.0**-53 * (np.abs(made)[:, None] + 4))
    bound[..., i[0]], bound[..., i[1]] = off, off
    return y, bound
