"""The convolution, scan and norm past 2^31 elements, and scans on several streams at once (GPU)."""
import pytest
import torch

import layer_oracle as L
from test_ssm_gpu import make, no_timeouts, s_slack, y_slack  # noqa: F401 (the fixture is used by all)

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def free():
    yield
    torch.cuda.empty_cache()


def rand(*s, seed=0):
    return torch.randn(*s, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(BF16)


def test_convolution_of_many_tokens():
    from gdn_b200 import conv
    T, D, tail = (1 << 18) + 200, 8192 + 8, 100
    x = torch.zeros(T, D, dtype=BF16, device="cuda")
    x[-2 * tail:] = rand(2 * tail, D)
    w, st = rand(D, 4, seed=1), rand(2, 3, D, seed=2)
    cu = torch.tensor([0, T - tail, T], device="cuda")
    out, new = conv.run(x, w, None, st, cu)
    o2, n2 = conv.run(x[-tail:].clone(), w, None, st[1:], torch.tensor([0, tail], device="cuda"))
    assert torch.equal(out[-tail:], o2) and torch.equal(new[1:], n2)
    o3, n3 = conv.run(x[-2 * tail:-tail].clone(), w, None, torch.zeros_like(st[:1]), torch.tensor([0, tail], device="cuda"))
    assert torch.equal(out[-2 * tail:-tail], o3) and torch.equal(new[:1], n3)


def test_convolution_in_a_far_slot():
    from gdn_b200 import conv
    P, D = (1 << 31) // (3 * 8192) + 100, 8192
    pool = torch.zeros(P, 3, D, dtype=BF16, device="cuda")
    x, w, st = rand(2, 2, D), rand(D, 4, seed=1), rand(3, D, seed=2)
    pool[P - 1] = st
    small = torch.stack([st, torch.zeros_like(st)])
    out = conv.run_pool(x, w, None, pool, torch.tensor([P - 1, P], dtype=torch.int32, device="cuda"),
                        torch.tensor([P - 2, -1], dtype=torch.int32, device="cuda"))
    want = conv.run_pool(x, w, None, small, torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    assert torch.equal(out, want) and torch.equal(pool[P - 2], small[0]) and torch.equal(pool[P - 1], st)
    assert not pool[:P - 2].any()


def test_norm_of_many_rows():
    from gdn_b200 import norm
    R, D = (1 << 18) + 100, 8192
    x = torch.zeros(R, D, dtype=BF16, device="cuda")
    x[-50:] = rand(50, D)
    w = rand(D, seed=1)
    assert torch.equal(norm.run(x, w)[-60:], norm.run(x[-60:].clone(), w))
    q, s = norm.run_fp8(x, w, group_size=128)
    q2, s2 = norm.run_fp8(x[-60:].clone(), w, group_size=128)
    assert torch.equal(q[-60:].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s[-60:], s2)


def test_scan_of_many_tokens():
    from gdn_b200 import ssm
    H, T, tail = 64, (1 << 19) + 300, 150
    m = make((tail,), H, 64, 1, 128, seed=3)
    x, B, C, a = (torch.zeros(T, *m[k].shape[1:], dtype=BF16, device="cuda") for k in ("x", "B", "C", "a"))
    for t, k in ((x, "x"), (B, "B"), (C, "C"), (a, "a")):
        t[-tail:] = m[k]
    st = torch.randn(3, H, 64, 128, device="cuda")
    cu = torch.tensor([0, T // 2, T - tail, T], device="cuda")
    out, new = ssm.run(x, B, C, st, m["A_log"], a, m["dt_bias"], m["D"], cu)
    y, ya, S, Sa = L.scan_ref(m["x"], m["B"], m["C"], m["a"], m["A_log"], m["dt_bias"], m["D"], st[2])
    L.within(out[-tail:], y, y_slack(ya, tail))
    L.within(new[2], S, s_slack(Sa, tail))
    assert out[:T - tail].isfinite().all() and new.isfinite().all()


def test_scan_in_a_far_slot():
    from gdn_b200 import ssm
    H, P = 64, (1 << 31) // (64 * 64 * 128) + 10
    pool = torch.zeros(P, H, 64, 128, dtype=BF16, device="cuda")
    st = rand(H, 64, 128, seed=4)
    pool[P - 1] = st
    for T in (1, 3):
        m = make((1, T), H, 64, 2, 128, seed=T)
        small = st[None].clone()
        args = (m["x"], m["B"], m["C"], m["A_log"], m["a"], m["dt_bias"], m["D"])
        out = ssm.run_pool(*args, pool, torch.tensor([P - 1], dtype=torch.int32, device="cuda"),
                           torch.tensor([P - 2], dtype=torch.int32, device="cuda"))
        want = ssm.run_pool(*args, small, torch.zeros(1, dtype=torch.int32, device="cuda"))
        assert torch.equal(out, want) and torch.equal(pool[P - 2], small[0]) and torch.equal(pool[P - 1], st)
    assert not pool[:P - 2].any()


def test_states_of_many_sequences():
    """Final states past 2^31 elements, from prompts of one token and of some."""
    from gdn_b200 import ssm
    H, P, Ns = 64, 128, 128
    N = (1 << 31) // (H * P * Ns) + 3
    for n in (1, 40):
        m = make((n,), H, P, 8, Ns, seed=n)
        x, B, C, a = (m[k].repeat(N, *[1] * (m[k].dim() - 1)) for k in ("x", "B", "C", "a"))
        cu = torch.arange(N + 1, device="cuda") * n
        out, new = ssm.run(x, B, C, None, m["A_log"], a, m["dt_bias"], m["D"], cu)
        assert (new == new[:1]).all() and torch.equal(out.view(N, n, H, P), out[:n].expand(N, n, H, P))
        y, ya, S, Sa = L.scan_ref(m["x"], m["B"], m["C"], m["a"], m["A_log"], m["dt_bias"], m["D"], torch.zeros(H, P, Ns))
        L.within(out[-n:], y, y_slack(ya, n))
        L.within(new[-1], S, s_slack(Sa, n))


def test_scans_side_by_side():
    """Cut and whole calls, eager and replayed, side by side: the bits of each alone."""
    from gdn_b200 import ssm
    sets = []
    for k, (lens, H) in enumerate((([5000], 16), ([300, 700, 64], 32), ([40] * 70 + [4000], 8))):
        m = make((sum(lens),), H, 64, 1, 128, seed=k)
        st = torch.randn(len(lens), H, 64, 128, device="cuda")
        cu = torch.tensor([0] + lens, device="cuda").cumsum(0)
        sets.append((m["x"], m["B"], m["C"], st, m["A_log"], m["a"], m["dt_bias"], m["D"], cu))
    want = [ssm.run(*s) for s in sets]
    torch.cuda.synchronize()
    g, held = torch.cuda.CUDAGraph(), None
    with torch.cuda.graph(g):
        held = ssm.run(*sets[0])
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[] for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i in range(8):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(ssm.run(*sets[k]))
        g.replay()
    torch.cuda.synchronize()
    for k, w in enumerate(want):
        for o, n in got[k]:
            assert torch.equal(o, w[0]) and torch.equal(n, w[1])
    assert torch.equal(held[0], want[0][0]) and torch.equal(held[1], want[0][1])
