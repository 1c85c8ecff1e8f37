"""The operators of a layer run together, as a serving stack runs them (GPU): norm, projection,
short convolution with its outputs split, gated delta rule or selective scan, gated norm; prompts,
then tokens over the slot pools, eagerly, captured and replayed, and on another stream."""
import pytest
import torch

import layer_oracle as L

pytestmark = pytest.mark.gpu
HID, W = 256, 4


def rand(g, *s, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*s, generator=g, device="cuda") * scale).to(dtype)


class ScanLayer:
    """x|B|C convolution, selective scan, gated norm; four heads of 64, two groups, state size 128."""
    H, P, G, N = 4, 64, 2, 128

    def __init__(self, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.inner, self.bc = self.H * self.P, self.G * self.N
        self.parts = [self.inner, self.bc, self.bc]
        dim = sum(self.parts)
        self.w_norm = 1 + rand(g, HID, scale=0.1)
        self.w_in = rand(g, HID, dim + self.inner + 8, scale=HID ** -0.5)  # (rows of a multiple of 8)
        self.w_conv, self.b_conv = rand(g, dim, W, scale=0.5), rand(g, dim, scale=0.1)
        self.A_log, self.dt_bias = L.gates(self.H, "cuda", g)
        self.D = torch.rand(self.H, generator=g, device="cuda")
        self.w_out = 1 + rand(g, self.inner, scale=0.1)
        self.dim = dim

    def front(self, x, residual):
        from gdn_b200 import norm
        h, residual = norm.run(x, self.w_norm, residual=residual)
        z = h @ self.w_in
        wide, gate, a = z[..., :self.dim], z[..., self.dim:self.dim + self.inner].contiguous(), z[..., -8:-8 + self.H].contiguous()
        return wide, gate, a, residual

    def back(self, y, gate):
        from gdn_b200 import norm
        return norm.run_fp8(y.reshape(gate.shape), self.w_out, gate=gate, gate_first=True, group_size=128)

    def prompts(self, x, residual, cu, conv_state=None, state=None):
        from gdn_b200 import conv, ssm
        wide, gate, a, residual = self.front(x, residual)
        (xs, B, C), conv_state = conv.run(wide, self.w_conv, self.b_conv, conv_state, cu, splits=self.parts)
        T = x.shape[0]
        y, state = ssm.run(xs.view(T, self.H, self.P), B.view(T, self.G, self.N), C.view(T, self.G, self.N), state,
                           self.A_log, a, self.dt_bias, self.D, cu)
        return (*self.back(y, gate), residual, conv_state, state, (wide, xs, B, C, a, y, gate))

    def tokens(self, x, residual, conv_pool, pool, slots):
        from gdn_b200 import conv, ssm
        b, t = x.shape[:2]
        wide, gate, a, residual = self.front(x.reshape(b * t, HID), residual.reshape(b * t, HID))
        xs, B, C = conv.run_pool(wide.unflatten(0, (b, t)), self.w_conv, self.b_conv, conv_pool, slots, splits=self.parts)
        y = ssm.run_pool(xs.view(b, t, self.H, self.P), B.view(b, t, self.G, self.N), C.view(b, t, self.G, self.N),
                         self.A_log, a.view(b, t, self.H), self.dt_bias, self.D, pool, slots)
        return (*self.back(y.reshape(b * t, self.inner), gate), residual)


def prompts(lens, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(lens)
    return rand(g, T, HID), rand(g, T, HID), torch.tensor([0] + lens, device="cuda").cumsum(0)


def test_scan_layer_prompts_against_the_definitions():
    """Every stage on what the stage before it gave, against its 64-bit definition."""
    lens = [70, 0, 130, 1]
    x, res, cu = prompts(lens, 1)
    lay = ScanLayer()
    q, scale, residual, conv_state, state, (wide, xs, B, C, a, y, gate) = lay.prompts(x, res, cu)
    _, h = L.norm_ref(x, lay.w_norm, 1e-6, residual=res)
    L.within(residual, h, 2.0 ** -24 * h.abs())
    at = 0
    for i, n in enumerate(lens):
        ref, mag, st = L.conv_ref(wide[at:at + n], lay.w_conv, lay.b_conv, torch.zeros(W - 1, lay.dim))
        L.within(torch.cat([xs, B, C], -1)[at:at + n], ref, 2.0 ** -16 * mag)
        assert torch.equal(L.d(conv_state[i]), st)
        seq = lambda v, *s: v[at:at + n].view(n, *s)  # noqa: E731
        yr, ya, S, Sa = L.scan_ref(seq(xs, 4, 64), seq(B, 2, 128), seq(C, 2, 128), a[at:at + n], lay.A_log, lay.dt_bias,
                                   lay.D, torch.zeros(4, 64, 128))
        L.within(y[at:at + n], yr, (2.0 ** -8 + (8 * n + 200) * 2.0 ** -24) * ya)
        L.within(state[i], S, (2.0 ** -16 + (8 * n + 200) * 2.0 ** -24) * Sa)
        at += n
    want, _ = L.norm_ref(y.reshape(gate.shape), lay.w_out, 1e-6, gate=gate, gate_first=True)
    amax = want.view(sum(lens), 2, 128).abs().amax(-1)
    assert ((L.d(scale) - amax / 448).abs() <= 2.0 ** -12 * amax / 448).all()
    got = L.d(q.float()) * L.d(scale).repeat_interleave(128, -1)
    bound = 2.0 ** -4 * want.abs() * (1 + 2.0 ** -8) + (2.0 ** -10 + 2.0 ** -10) * (amax / 448).repeat_interleave(128, -1)
    assert ((got - want).abs() <= bound).all()


def test_scan_layer_prompt_then_tokens_captured_and_on_another_stream():
    """A prompt, then tokens over the pools: eager, replayed from a graph, and on a side stream give the same bits."""
    lay = ScanLayer()
    lens = [90, 33, 64]
    x, res, cu = prompts(lens, 2)
    _, _, _, conv_state, state, _ = lay.prompts(x, res, cu)
    g = torch.Generator(device="cuda").manual_seed(3)
    steps = [(rand(g, 3, t, HID), rand(g, 3, t, HID)) for t in (1, 1, 1, 1)]
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")

    def pools():
        cp, sp = torch.zeros(5, W - 1, lay.dim, dtype=torch.bfloat16, device="cuda"), torch.zeros(5, 4, 64, 128, device="cuda")
        cp[slots.long()], sp[slots.long()] = conv_state, state
        return cp, sp

    cp, sp = pools()
    eager = [lay.tokens(*s, cp, sp, slots) for s in steps]

    cp2, sp2 = pools()
    bx, br = (torch.empty_like(v) for v in steps[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lay.tokens(bx.zero_(), br.zero_(), cp2, sp2, slots)  # (one-time set-up outside the capture)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lay.tokens(bx, br, cp2, sp2, slots)
    for dst, src in zip((cp2, sp2), pools()):
        dst.copy_(src)
    for (tx, tr), want in zip(steps, eager):
        bx.copy_(tx)
        br.copy_(tr)
        graph.replay()
        for o, w in zip(out, want):
            assert torch.equal(o.float(), w.float())
    assert torch.equal(cp, cp2) and torch.equal(sp, sp2)

    cp3, sp3 = pools()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [lay.tokens(*s, cp3, sp3, slots) for s in steps]
    side.synchronize()
    for o, w in zip(other, eager):
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(o, w))
    assert torch.equal(cp, cp3) and torch.equal(sp, sp3)


def test_two_captured_prompt_calls():
    """Two graphs of calls that are cut into pieces (each with a workspace), replayed in turn and together."""
    lay = ScanLayer()
    calls = []
    for seed, n in ((5, 3000), (6, 2500)):
        x, res, cu = prompts([n], seed)
        want = lay.prompts(x, res, cu)[:5]
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            got = lay.prompts(x, res, cu)[:5]
        calls.append((graph, side, got, want, (x, res, cu)))  # (a graph reads its inputs where they were)
    torch.cuda.synchronize()
    for graph, side, *_ in calls * 2:
        with torch.cuda.stream(side):
            graph.replay()
    torch.cuda.synchronize()
    for _, _, got, want, _ in calls:
        for a, b in zip(got, want):
            assert torch.equal(a.float(), b.float())


def test_delta_rule_layer_prompt_and_tokens():
    """q|k|v convolution, gated delta rule, gated norm: a prompt and then tokens against the whole prompt."""
    from gdn_b200 import conv, decode, norm, prefill
    g = torch.Generator(device="cuda").manual_seed(7)
    Hq, Hv, T, n = 2, 4, 90, 84
    parts = [Hq * 128, Hq * 128, Hv * 128]
    dim = sum(parts)
    x = rand(g, T, dim)
    w, gate, wn = rand(g, dim, W, scale=0.5), rand(g, T, Hv, 128), 1 + rand(g, 128, scale=0.1)
    a, b = rand(g, T, Hv), rand(g, T, Hv)
    A_log, dt_bias = L.gates(Hv, "cuda", g)
    scale = 0.0

    def run(t0, t1, conv_state=None, state=None):
        cu = torch.tensor([0, t1 - t0], device="cuda")
        (q, k, v), cs = conv.run(x[t0:t1], w, None, conv_state, cu, splits=parts)
        o, st = prefill.run(q.view(-1, Hq, 128), k.view(-1, Hq, 128), v.view(-1, Hv, 128), state, A_log, a[t0:t1], dt_bias,
                            b[t0:t1], cu, scale, use_qk_l2norm=True)
        return norm.run(o, wn, gate=gate[t0:t1]), cs, st

    whole, cs_all, st_all = run(0, T)
    head, cs, st = run(0, n)
    slot = torch.zeros(1, dtype=torch.int32, device="cuda")
    outs = [head]
    for t in range(n, T, 2):
        q, k, v = conv.run_pool(x[None, t:t + 2], w, None, cs, slot, splits=parts)
        o = decode.run_pool(q.view(1, 2, Hq, 128), k.view(1, 2, Hq, 128), v.view(1, 2, Hv, 128), A_log, a[None, t:t + 2],
                            dt_bias, b[None, t:t + 2], scale, st, slot, qk_l2norm=True)
        outs.append(norm.run(o[0], wn, gate=gate[t:t + 2]))
    assert torch.equal(cs, cs_all)
    got = torch.cat(outs)
    # the delta rule's own bounds (bf16 outputs within 1e-2, the state within 1e-3), seen through a norm that
    # divides by the rows' root mean square
    rel = (got.float() - whole.float()).norm() / whole.float().norm()
    assert rel < 1e-2 and (st - st_all).norm() / st_all.norm() < 1e-3


def test_the_ctypes_path_gives_the_same(monkeypatch):
    """Without the torch binding the entry points make the same calls through ctypes."""
    from gdn_b200 import _native as N, conv, norm, ssm
    lay = ScanLayer()
    x, res, cu = prompts([2000, 40], 8)
    want = lay.prompts(x, res, cu)[:5]
    cp, sp = want[3].clone(), want[4].clone()
    slots = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    tok = (x[:4].view(2, 2, HID), res[:4].view(2, 2, HID))
    want_t = lay.tokens(*tok, cp, sp, slots)
    monkeypatch.setattr(N, "_ext", None)
    got = lay.prompts(x, res, cu)[:5]
    cp2, sp2 = got[3].clone(), got[4].clone()
    got_t = lay.tokens(*tok, cp2, sp2, slots)
    for a, b in zip((*got, *got_t, cp2, sp2), (*want, *want_t, cp, sp)):
        assert a.dtype == b.dtype and torch.equal(a.float(), b.float())
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    for exc, call in ((ValueError, lambda: conv.run(z(4, 60), z(60, 4), None, None, cu)),
                      (ValueError, lambda: conv.run(z(4, 64), z(64, 4), None, None, cu, splits=[32])),
                      (TypeError, lambda: norm.run(z(4, 64).float(), z(64))),
                      (ValueError, lambda: norm.run(z(4, 64), z(64), residual=z(4, 64), gate=z(4, 64))),
                      (ValueError, lambda: ssm.run(z(4, 2, 32), z(4, 1, 64), z(4, 1, 64), None, z(2).float(), z(4, 2),
                                                   z(2).float(), None, cu))):
        with pytest.raises(exc):
            call()
