"""Root-mean-square norm of rows, with the residual's addition in front or a SiLU gate
before or after, in the input's type or in 8 bits with scales:

    h = x (+ residual)                     residual_out = h, rounded once
    y = h / sqrt(mean(h^2) + eps) * weight (* silu(gate))
    with gate_first: h = x silu(gate), y = h / sqrt(mean(h^2) + eps) * weight
    8 bits (e4m3): scale = max |y| / 448 of the row or of each 128 columns, y / scale

The norm before a layer's projections (residual, 8 bits for an fp8 product) and the gated
norm of a gated delta rule's or a selective scan's output.  y is fp32 up to its one
rounding.  C ABI: ``gdn_rms_norm`` (include/gdn_b200.h).  No reference counterpart.
"""
from __future__ import annotations

import torch

from . import _native as N
from ._checks import dtype16, expect


def _run(x, weight, eps, residual, gate, gate_first, fp8, group, output, residual_out):
    ext = N.torch_ext()
    if ext is not None:
        return ext.rms_norm(x, weight, eps, residual, gate, gate_first, fp8, group, output, residual_out)
    dt = dtype16(x)
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    D = x.shape[-1]
    if D == 0 or D % 8 or D > 16384:
        raise ValueError("the rows of x must hold a multiple of 8 values, at most 16384")
    if residual is not None and gate is not None:
        raise ValueError("residual and gate cannot both be given")
    if residual is None and residual_out is not None:
        raise ValueError("residual_out goes with residual")
    if group not in (0, 128) or (group and D % 128):
        raise ValueError("group_size must be 0, or 128 with rows of a multiple of 128")
    rows = x.numel() // D

    def row_stride(name, t):
        if t is None:
            return D
        if t.device != x.device:
            raise ValueError(f"x and {name} must be on the same device")
        if t.dtype != x.dtype:
            raise TypeError(f"{name} must have the type of x")
        if t.shape != x.shape:
            raise ValueError(f"{name} must have the shape of x")
        if t.is_contiguous():
            return D
        if t.dim() != 2 or t.stride(1) != 1:
            raise ValueError(f"{name} must be contiguous, or 2D with contiguous rows")
        return t.stride(0) if rows > 1 else D

    strides = [row_stride(n, t) for n, t in (("x", x), ("residual", residual), ("gate", gate))]
    expect(x, "weight", weight, x.dtype, (D,))
    odt = torch.float8_e4m3fn if fp8 else x.dtype
    if output is None:
        output = torch.empty(x.shape, dtype=odt, device=x.device)
    expect(x, "output", output, odt, x.shape)
    ret, scale = [output], None
    if fp8:
        shape = (*x.shape[:-1], D // group) if group else x.shape[:-1]
        scale = torch.empty(shape, dtype=torch.float32, device=x.device)
        ret.append(scale)
    if residual is not None:
        if residual_out is None:
            residual_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        expect(x, "residual_out", residual_out, x.dtype, x.shape)
        ret.append(residual_out)
    with torch.cuda.device(x.device):
        rc = N.lib().gdn_rms_norm(N.ptr(x), strides[0], N.ptr(weight), N.ptr(residual), strides[1], N.ptr(gate),
                                  strides[2], float(eps), N.ptr(output), N.ptr(scale), group, N.ptr(residual_out),
                                  rows, D, dt, int(gate_first), N.stream_handle(x.device))
    N.check(rc, "gdn_rms_norm")
    return ret


def run(x, weight, eps: float = 1e-6, residual=None, gate=None, gate_first: bool = False, output=None,
        residual_out=None):
    """Norm in x's type; returns the output, with ``residual`` (output, residual_out).

    x [..., D] bf16 or fp16, contiguous or 2D with a row stride; residual, gate of
    x's shape (not both); weight [D] of x's type; D a multiple of 8 up to 16384.
    ``output`` and ``residual_out`` may each be an input that is contiguous (in place),
    but overlap nothing in part."""
    r = _run(x, weight, eps, residual, gate, gate_first, False, 0, output, residual_out)
    return tuple(r) if residual is not None else r[0]


def run_fp8(x, weight, eps: float = 1e-6, residual=None, gate=None, gate_first: bool = False, group_size: int = 0,
            output=None, residual_out=None):
    """Norm to e4m3; returns (output float8_e4m3fn [..., D], scale fp32), with
    ``residual`` (output, scale, residual_out).  The value an element stands for is
    output * scale; scales are per row ([...], group_size 0) or per 128 columns
    ([..., D / 128], group_size 128).  Other arguments as ``run``."""
    return tuple(_run(x, weight, eps, residual, gate, gate_first, True, group_size, output, residual_out))
