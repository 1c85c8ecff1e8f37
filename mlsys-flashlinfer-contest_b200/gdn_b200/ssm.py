"""Selective state-space scan with one decay per head and token, the sibling of the gated
delta rule without its correction term:

    dt = softplus(a + dt_bias)
    S <- exp(-exp(A_log) dt) S + (dt x) B^T        y = S C + D x

``run`` takes packed prompts (``cu_seqlens``, initial states in, final states out, as
``prefill.run``), ``run_pool`` the tokens of a decode batch over a pool of states (as
``decode.run_pool``).  States are k-last, [.., H, P, state_dim]; head h reads B and C of
group h // (H / G).  Head and state sizes are 64 or 128.  C ABI: ``gdn_ssm``,
``gdn_ssm_pool`` (include/gdn_b200.h).  No reference counterpart.
"""
from __future__ import annotations

import torch

from . import _native as N
from ._checks import dim, expect
from .prefill import _widen


def _inputs(x, B, C, A_log, a, dt_bias, D, lead):
    """Checks of the inputs both forms share (the ctypes path): (H, P, G, state_dim)."""
    dim("x", x, lead + 2)
    dim("B", B, lead + 2)
    H, P = x.shape[lead:]
    G, Ns = B.shape[lead:]
    if H <= 0 or G <= 0 or H % G:
        raise ValueError("the heads of x must be a positive multiple of B's groups")
    if P not in (64, 128):
        raise ValueError("the head size of x must be 64 or 128")
    if Ns not in (64, 128):
        raise ValueError("the state size of B and C must be 64 or 128")
    first = tuple(x.shape[:lead])
    for name, t, dt, shape in (("x", x, torch.bfloat16, (*first, H, P)), ("B", B, torch.bfloat16, (*first, G, Ns)),
                               ("C", C, torch.bfloat16, (*first, G, Ns)), ("a", a, torch.bfloat16, (*first, H)),
                               ("A_log", A_log, torch.float32, (H,)), ("dt_bias", dt_bias, torch.float32, (H,)),
                               ("D", D, torch.float32, (H,))):
        if t is not None or name != "D":
            expect(x, name, t, dt, shape)
    return H, P, G, Ns


def workspace_bytes(T: int, Nseq: int, H: int, G: int, P: int, state_dim: int) -> int:
    return int(N.lib().gdn_ssm_workspace_bytes(T, Nseq, H, G, P, state_dim))


def run(x, B, C, state, A_log, a, dt_bias, D, cu_seqlens, output=None, new_state=None):
    """Scan of packed prompts; returns (output [T,H,P] bf16, new_state [N,H,P,state_dim] fp32).

    x [T,H,P], B and C [T,G,state_dim], a [T,H] bf16; state [N,H,P,state_dim] fp32 or
    None (zeros); A_log, dt_bias [H] fp32; D [H] fp32 or None (no skip term);
    cu_seqlens [N+1] int64 (int32 is widened).  Rows of no sequence are left as they
    were in a given ``output``, which may not overlap an input; a sequence of length 0
    keeps its state.  Outputs are off by their rounding and 2^-16 of the sums' terms
    (tensor-core products of two bf16 terms; up to 16 tokens a sequence on average, and
    ``run_pool``: fp32 sums, so that the same tokens may give other bits), states by
    fp32 arithmetic."""
    cu_seqlens = _widen(cu_seqlens)
    ext = N.torch_ext()
    if ext is not None:
        return ext.ssm(x, B, C, state, A_log, a, dt_bias, D, cu_seqlens, output, new_state)
    H, P, G, Ns = _inputs(x, B, C, A_log, a, dt_bias, D, 1)
    T = x.shape[0]
    dim("cu_seqlens", cu_seqlens, 1)
    n = cu_seqlens.shape[0] - 1
    if n <= 0:
        raise ValueError("must have at least one sequence")
    expect(x, "cu_seqlens", cu_seqlens, torch.int64, (n + 1,))
    if state is not None:
        expect(x, "state", state, torch.float32, (n, H, P, Ns))
    if output is None:
        output = torch.empty_like(x)
    if new_state is None:
        new_state = torch.empty((n, H, P, Ns), dtype=torch.float32, device=x.device)
    expect(x, "output", output, torch.bfloat16, x.shape)
    expect(x, "new_state", new_state, torch.float32, (n, H, P, Ns))
    with torch.cuda.device(x.device):
        ws_bytes = workspace_bytes(T, n, H, G, P, Ns)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
        rc = N.lib().gdn_ssm(N.ptr(x), N.ptr(B), N.ptr(C), N.ptr(state), N.ptr(A_log), N.ptr(a), N.ptr(dt_bias),
                             N.ptr(D), N.ptr(cu_seqlens), N.ptr(output), N.ptr(new_state), T, n, H, G, P, Ns,
                             N.ptr(ws), ws_bytes, N.stream_handle(x.device))
    N.check(rc, "gdn_ssm")
    return output, new_state


def run_pool(x, B, C, A_log, a, dt_bias, D, state_pool, in_slots, out_slots=None, no_state_update: bool = False,
             output=None):
    """Scan of T >= 1 tokens of each sequence of a decode batch over a pool of states,
    updated in place; returns output [B,T,H,P] bf16.

    x [B,T,H,P], B and C [B,T,G,state_dim], a [B,T,H] bf16; state_pool
    [pool,H,P,state_dim] fp32 or bf16: sequence i starts from slot in_slots[i] (int32;
    negative or out of range: zeros) and its state goes to out_slots[i] (default
    in_slots; negative or out of range: not written).  ``no_state_update`` leaves the
    pool as it is."""
    ext = N.torch_ext()
    if ext is not None:
        return ext.ssm_pool(x, B, C, A_log, a, dt_bias, D, state_pool, in_slots, out_slots, no_state_update, output)
    H, P, G, Ns = _inputs(x, B, C, A_log, a, dt_bias, D, 2)
    batch, T = x.shape[:2]
    if T < 1:
        raise ValueError("need at least one token per sequence")
    if state_pool.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("state_pool must be float32 or bfloat16")
    dim("state_pool", state_pool, 4)
    expect(x, "state_pool", state_pool, state_pool.dtype, (state_pool.shape[0], H, P, Ns))
    expect(x, "in_slots", in_slots, torch.int32, (batch,))
    if out_slots is not None:
        expect(x, "out_slots", out_slots, torch.int32, (batch,))
    if output is None:
        output = torch.empty_like(x)
    expect(x, "output", output, torch.bfloat16, x.shape)
    with torch.cuda.device(x.device):
        rc = N.lib().gdn_ssm_pool(N.ptr(x), N.ptr(B), N.ptr(C), N.ptr(A_log), N.ptr(a), N.ptr(dt_bias), N.ptr(D),
                                  N.ptr(state_pool), int(state_pool.dtype == torch.bfloat16), state_pool.shape[0],
                                  N.ptr(in_slots), N.ptr(out_slots), 2 if no_state_update else 0, N.ptr(output),
                                  batch, T, H, G, P, Ns, N.stream_handle(x.device))
    N.check(rc, "gdn_ssm_pool")
    return output
