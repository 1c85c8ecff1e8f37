"""Short causal depthwise convolution: the operator in front of a gated delta rule or a
selective-scan layer.

``run`` takes packed prompts (``cu_seqlens``, as ``prefill.run``), ``run_pool`` the
tokens of a decode batch over a pool of convolution states with read/write slots (as
``decode.run_pool``):

    out[t, d] = silu(bias[d] + sum_j weight[d, j] x~[t - W + 1 + j, d])

where x~ before a sequence's first token is its state: its last W - 1 inputs, oldest
first (zeros without one).  ``splits`` cuts the channels into up to four separate
contiguous outputs (q | k | v, or x | B | C), so that the operator that follows takes
them as they are.  C ABI: ``gdn_conv``, ``gdn_conv_pool`` (include/gdn_b200.h).  No
reference counterpart: the reference's solutions stop at the delta rule.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as N
from ._checks import dim, dtype16, expect
from .prefill import _widen


def _plan(x, weight, bias, splits, outputs):
    """Checks of what both forms share (the ctypes path): (dtype, D, W, splits, outputs)."""
    dt = dtype16(x)
    D = x.shape[-1]
    dim("weight", weight, 2)
    W = weight.shape[1]
    if not 2 <= W <= 4:
        raise ValueError("the convolution's width must be 2, 3 or 4")
    if D == 0 or D % 8:
        raise ValueError("the channels of x must be a positive multiple of 8")
    expect(x, "weight", weight, x.dtype, (D, W))
    if bias is not None:
        expect(x, "bias", bias, x.dtype, (D,))
    if x.stride(-1) != 1:
        raise ValueError("the channels of x must be contiguous")
    splits = list(splits) or [D]
    if len(splits) > 4:
        raise ValueError("at most 4 splits")
    if any(s <= 0 or s % 8 for s in splits):
        raise ValueError("splits must be positive multiples of 8")
    if sum(splits) != D:
        raise ValueError("splits must sum to the channels of x")
    if outputs is None:
        outputs = [torch.empty((*x.shape[:-1], s), dtype=x.dtype, device=x.device) for s in splits]
    elif len(outputs) != len(splits):
        raise ValueError("outputs must hold one tensor per split")
    for s, o in zip(splits, outputs):
        expect(x, "outputs", o, x.dtype, (*x.shape[:-1], s))
    return dt, D, W, splits, list(outputs)


def _pointers(splits, outputs):
    return ((ctypes.c_void_p * len(outputs))(*[o.data_ptr() for o in outputs]),
            (ctypes.c_int64 * len(splits))(*splits))


def run(x, weight, bias, state, cu_seqlens, silu: bool = True, splits=None, outputs=None, new_state=None):
    """Convolution of packed prompts; returns (output, new_state), with ``splits``
    ([outputs], new_state).

    x [T, D] bf16 or fp16 (rows may be strided: a slice of a wider projection);
    weight [D, W] and bias [D] (or None) of x's dtype, W = 2, 3 or 4; state
    [N, W-1, D] or None (zeros); cu_seqlens [N+1] int64 (int32 is widened).
    ``splits``: channel counts (multiples of 8) of separate contiguous outputs.
    Rows of no sequence are left as they were in given ``outputs``, which may not
    overlap x or one another; a sequence of length 0 keeps its state."""
    cu_seqlens = _widen(cu_seqlens)
    ext = N.torch_ext()
    if ext is not None:
        outs, new_state = ext.conv(x, weight, bias, state, cu_seqlens, silu, list(splits or ()), outputs, new_state)
        return (outs if splits else outs[0]), new_state
    dt, D, W, parts, outs = _plan(x, weight, bias, splits or (), outputs)
    dim("x", x, 2)
    dim("cu_seqlens", cu_seqlens, 1)
    T, n = x.shape[0], cu_seqlens.shape[0] - 1
    if n <= 0:
        raise ValueError("must have at least one sequence")
    expect(x, "cu_seqlens", cu_seqlens, torch.int64, (n + 1,))
    if state is not None:
        expect(x, "state", state, x.dtype, (n, W - 1, D))
    if new_state is None:
        new_state = torch.empty((n, W - 1, D), dtype=x.dtype, device=x.device)
    expect(x, "new_state", new_state, x.dtype, (n, W - 1, D))
    ptrs, widths = _pointers(parts, outs)
    with torch.cuda.device(x.device):
        rc = N.lib().gdn_conv(N.ptr(x), x.stride(0) if T > 1 else D, N.ptr(weight), N.ptr(bias), N.ptr(state),
                              N.ptr(cu_seqlens), ptrs, widths, len(parts), N.ptr(new_state), T, n, D, W, dt,
                              int(silu), N.stream_handle(x.device))
    N.check(rc, "gdn_conv")
    return (outs if splits else outs[0]), new_state


def run_pool(x, weight, bias, state_pool, in_slots, out_slots=None, silu: bool = True, splits=None, outputs=None):
    """Convolution of T >= 1 tokens of each sequence of a decode batch over a pool of
    states, updated in place; returns the output, with ``splits`` the list of outputs.

    x [B, T, D] (batch and token strides are free); state_pool [P, W-1, D];
    sequence i starts from slot in_slots[i] (int32 [B]; negative or >= P: zeros) and
    its new state goes to out_slots[i] (default in_slots; negative or >= P: not
    written)."""
    ext = N.torch_ext()
    if ext is not None:
        outs = ext.conv_pool(x, weight, bias, state_pool, in_slots, out_slots, silu, list(splits or ()), outputs)
        return outs if splits else outs[0]
    dt, D, W, parts, outs = _plan(x, weight, bias, splits or (), outputs)
    dim("x", x, 3)
    B, T, _ = x.shape
    if T < 1:
        raise ValueError("need at least one token per sequence")
    dim("state_pool", state_pool, 3)
    expect(x, "state_pool", state_pool, x.dtype, (state_pool.shape[0], W - 1, D))
    for name, s in (("in_slots", in_slots), ("out_slots", out_slots)):
        if s is not None or name == "in_slots":
            expect(x, name, s, torch.int32, (B,))
    ptrs, widths = _pointers(parts, outs)
    with torch.cuda.device(x.device):
        rc = N.lib().gdn_conv_pool(N.ptr(x), x.stride(0) if B > 1 else 0, x.stride(1) if T > 1 else D,
                                   N.ptr(weight), N.ptr(bias), N.ptr(state_pool), state_pool.shape[0],
                                   N.ptr(in_slots), N.ptr(out_slots), ptrs, widths, len(parts), B, T, D, W,
                                   dt, int(silu), N.stream_handle(x.device))
    N.check(rc, "gdn_conv_pool")
    return outs if splits else outs[0]
