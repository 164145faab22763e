"""Rotary positions over librta.so's rta_rotary_turns and rta_rotate: pairs of neighbours or of half a
head's distance, the whole head or its first values, frequencies as trained or scaled for longer
contexts.  PagedCache.append_rotary takes the same rotation on the way into the pages.
"""
import ctypes

import torch

from . import _lib
from ._lib import check

LAYOUTS = {"neighbours": 0, "halves": 1}
SCALINGS = {"plain": 0, "linear": 1, "base": 2, "ramp": 3, "bands": 4}


def turns(dims, theta=1e6, scaling="plain", factor=1.0, original=0, low=1.0, high=32.0):
    """(turns per position of each of the dims / 2 pairs as a float64 CPU tensor, amplitude); the formulas
    of `scaling` are rta_rotary_turns's in include/rta.h."""
    if scaling not in SCALINGS:
        raise ValueError(f"scaling is one of {', '.join(SCALINGS)}")
    got = torch.empty(max(dims, 0) // 2, dtype=torch.float64)
    amplitude = ctypes.c_double()
    check(_lib.load().rta_rotary_turns(dims, theta, SCALINGS[scaling], factor, original, low, high, got.data_ptr(),
                                       ctypes.byref(amplitude)), "rta_rotary_turns")
    return got, amplitude.value


class Rotary:
    """A rotation: layout "neighbours" (pairs 2 j, 2 j + 1) or "halves" (j, j + dims / 2), over the first
    `dims` (None: all) of head_dim values.  amplitude: None for the scaling's own."""

    def __init__(self, head_dim, dims=None, layout="neighbours", theta=1e6, scaling="plain", factor=1.0, original=0,
                 low=1.0, high=32.0, amplitude=None, device="cuda:0"):
        if layout not in LAYOUTS:
            raise ValueError(f"layout is one of {', '.join(LAYOUTS)}")
        dims = head_dim if dims is None else dims
        if not 0 < dims <= head_dim or head_dim > 512:
            raise ValueError(f"dims lies in 2 .. head_dim, and head_dim in 2 .. 512 ({dims}, {head_dim})")
        table, own = turns(dims, theta, scaling, factor, original, low, high)
        self.head_dim, self.dims, self.layout = head_dim, dims, layout
        self.amplitude = own if amplitude is None else float(amplitude)
        self.turns = table.to(device)
        self.device = self.turns.device
        self._c = _lib.Rotary(LAYOUTS[layout], head_dim, dims, self.amplitude, self.turns.data_ptr())
        self._at = ctypes.byref(self._c)
        self._rotate = _lib.load().rta_rotate

    def _check_rows(self, t, name, heads=None):
        if not isinstance(t, torch.Tensor) or t.device != self.device or t.dtype != torch.float32:
            raise TypeError(f"{name} must be a float32 tensor on {self.device}")
        hd = self.head_dim
        if t.dim() != 3:
            raise ValueError(f"{name} must be [rows, heads, {hd}]")
        (rows, heads, width), (row, head, one) = t.shape, t.stride()
        if width != hd or one != 1 or (heads > 1 and head != hd):
            raise ValueError(f"{name} must be [rows, heads, {hd}] with contiguous rows")
        return row if rows > 1 else max(row, heads * hd)

    def rotate(self, x, positions, out=None):
        """x [rows, heads, head_dim] fp32 (rows may be strided) turned to positions [rows] (int64, any
        sign: negated positions take gradients back).  out may be x."""
        stride = self._check_rows(x, "x")
        rows, heads, _ = x.shape
        if not isinstance(positions, torch.Tensor) or positions.device != self.device or positions.dtype != torch.int64:
            raise TypeError(f"positions must be an int64 tensor on {self.device}")
        if positions.shape != (rows,) or not positions.is_contiguous():
            raise ValueError(f"positions must be contiguous of shape ({rows},)")
        if out is None:
            out = torch.empty(x.shape, dtype=torch.float32, device=self.device)
            out_stride = heads * self.head_dim
        else:
            out_stride = self._check_rows(out, "out")
            if out.shape != x.shape:
                raise ValueError(f"out must be of shape {tuple(x.shape)}")
        fn, index = self._rotate, self.device.index
        args = (self._at, x.data_ptr(), stride, rows, heads, positions.data_ptr(), out.data_ptr(), out_stride,
                torch._C._cuda_getCurrentRawStream(index))
        if torch.cuda.current_device() == index:
            status = fn(*args)
        else:
            with torch.cuda.device(index):
                status = fn(*args)
        if status:
            check(status, "rta_rotate")
        return out


__all__ = ["LAYOUTS", "SCALINGS", "Rotary", "turns"]
