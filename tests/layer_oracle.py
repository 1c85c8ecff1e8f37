"""64-bit definitions of the convolution, the selective scan and the norm, with the bounds
their tests hold the kernels to.

``*_ref`` return the exact result and a magnitude: the same sums over absolute values.  A
kernel that adds n fp32 terms is off by at most about n 2^-24 times that magnitude; a
rounding to a type is off by half a step, ``HALF[dtype]`` relative to the value.
"""
import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def d(t):
    return None if t is None else t.detach().cpu().double()


def within(got, ref, slack):
    """|got - ref| <= half a step of got's type at the reference (plus slack, absolute)."""
    g, r = d(got), ref
    assert g.shape == r.shape, (g.shape, r.shape)
    bound = HALF[got.dtype] * (r.abs() + slack) + TINY[got.dtype] + slack
    bad = ~((g - r).abs() <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} outside the bound, worst ratio "
                           f"{float(((g - r).abs() / bound).nan_to_num(nan=1e30).max()):.3g}")


def silu(x):
    return x * torch.sigmoid(x)


def conv_ref(x, weight, bias, before, act=True):
    """One sequence: x [t, D] after the rows ``before`` [W-1, D] -> (out, magnitude, state)."""
    x, w = d(x), d(weight)
    full = torch.cat([d(before), x])
    t, W = x.shape[0], w.shape[1]
    out = torch.zeros_like(x)
    mag = torch.zeros_like(x)
    for j in range(W):
        out += w[:, j] * full[j:j + t]
        mag += (w[:, j] * full[j:j + t]).abs()
    if bias is not None:
        out += d(bias)
        mag += d(bias).abs()
    return (silu(out) if act else out), mag, full[full.shape[0] - (W - 1):]


def scan_ref(x, B, C, a, A_log, dt_bias, D, S):
    """One sequence: x [t, H, P], B, C [t, G, Ns], a [t, H], S [H, P, Ns] -> (y, its magnitude,
    state, its magnitude)."""
    x, B, C, a, A_log, dt_bias, D, S = (d(v) for v in (x, B, C, a, A_log, dt_bias, D, S))
    S = S.clone()
    H, G = x.shape[1], B.shape[1]
    B, C = (v.repeat_interleave(H // G, 1) for v in (B, C))
    dt = torch.nn.functional.softplus(a + dt_bias, threshold=1e9)
    Sa = S.abs()
    y, ya = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(x.shape[0]):
        dec = torch.exp(-torch.exp(A_log) * dt[t])[:, None, None]
        add = (dt[t][:, None] * x[t])[..., None] * B[t][:, None]
        S, Sa = dec * S + add, dec * Sa + add.abs()
        skip = D[:, None] * x[t] if D is not None else torch.zeros_like(x[t])
        y[t] = (S * C[t][:, None]).sum(-1) + skip
        ya[t] = (Sa * C[t][:, None].abs()).sum(-1) + skip.abs()
    return y, ya, S, Sa


def norm_ref(x, weight, eps, residual=None, gate=None, gate_first=False):
    """(y, h before the gate) in 64 bits."""
    h = d(x)
    if residual is not None:
        h = h + d(residual)
    raw = h
    if gate is not None and gate_first:
        h = h * silu(d(gate))
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * d(weight)
    if gate is not None and not gate_first:
        y = y * silu(d(gate))
    return y, raw


def gates(H, device, g):
    """A_log, dt_bias of the magnitudes a trained layer has (steps of 1e-3 to 0.1, decays of 1 to 16)."""
    u = torch.rand(2, H, generator=g, device=device)
    step = torch.exp(u[0] * 4.6 - 6.9)
    return torch.log(1 + 15 * u[1]), step + torch.log(-torch.expm1(-step))
