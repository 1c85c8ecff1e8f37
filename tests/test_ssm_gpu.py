"""The selective scan against its 64-bit definition (GPU)."""
import pytest
import torch

import layer_oracle as L

pytestmark = pytest.mark.gpu


def make(lead, H, P, G, Ns, seed=0, skip=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*lead, *s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    A_log, dt_bias = L.gates(H, "cuda", g)
    return dict(x=r(H, P), B=r(G, Ns), C=r(G, Ns), A_log=A_log, a=r(H), dt_bias=dt_bias,
                D=torch.rand(H, generator=g, device="cuda") if skip else None)


# Bounds.  fp32 arithmetic on a state that t tokens went into: every token multiplies it by a
# decay whose relative error is a few 2^-24 (its exponent rounded, expf) and adds a product
# of dt (log1pf, expf: a few 2^-24) -- 8 2^-24 a token, and 200 2^-24 for the rest, times
# the magnitude.  Matrix products over chunks round two operands to bf16, the weights within the
# chunk and the state that C reads (half a step, 2^-8, of each term), and split the
# state's update into two bf16 terms (2^-8 of 2^-8).
def y_slack(ya, n):
    return (2.0 ** -8 + (8 * n + 200) * 2.0 ** -24) * ya


def s_slack(Sa, n):
    return (2.0 ** -16 + (8 * n + 200) * 2.0 ** -24) * Sa


def f32_slack(mag, n):
    return (8 * n + 200) * 2.0 ** -24 * mag


def check_packed(m, lens, state, out, new, cu0=0):
    H, P = m["x"].shape[1:]
    Ns = m["B"].shape[2]
    at = cu0
    for i, n in enumerate(lens):
        S0 = state[i] if state is not None else torch.zeros(H, P, Ns)
        seq = {k: m[k][at:at + n] for k in ("x", "B", "C", "a")}
        y, ya, S, Sa = L.scan_ref(**seq, A_log=m["A_log"], dt_bias=m["dt_bias"], D=m["D"], S=S0)
        L.within(out[at:at + n], y, y_slack(ya, n))
        L.within(new[i], S, s_slack(Sa, n))
        at += n


@pytest.mark.parametrize("H,P,G,Ns", [(2, 64, 1, 128), (3, 64, 1, 128), (6, 64, 2, 64), (2, 128, 1, 128),
                                      (4, 128, 2, 64), (1, 64, 1, 64)])
@pytest.mark.parametrize("lens,state", [([1], False), ([1, 0, 2, 63, 64, 65], True), ([0, 200, 1, 0, 130], True),
                                        ([127, 128, 129], False), ([700], True)])
def test_packed(lens, state, H, P, G, Ns):
    from gdn_b200 import ssm
    m = make((sum(lens),), H, P, G, Ns, seed=sum(lens) + H, skip=H != 3)
    st = torch.randn(len(lens), H, P, Ns, device="cuda") if state else None
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0)
    out, new = ssm.run(m["x"], m["B"], m["C"], st, m["A_log"], m["a"], m["dt_bias"], m["D"], cu)
    check_packed(m, lens, st, out, new)


def test_rows_of_no_sequence_stay():
    from gdn_b200 import ssm
    m = make((300,), 4, 64, 1, 128)
    out = torch.full((300, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([5, 80, 80, 281], dtype=torch.int32, device="cuda")
    _, new = ssm.run(m["x"], m["B"], m["C"], None, m["A_log"], m["a"], m["dt_bias"], m["D"], cu, output=out)
    assert (out[:5] == 7).all() and (out[281:] == 7).all()
    check_packed(m, [75, 0, 201], None, out, new, cu0=5)
    assert (new[1] == 0).all()


def test_no_tokens_keeps_the_states():
    from gdn_b200 import ssm
    m = make((0,), 2, 64, 1, 128)
    st = torch.randn(2, 2, 64, 128, device="cuda")
    cu = torch.zeros(3, dtype=torch.int64, device="cuda")
    out, new = ssm.run(m["x"], m["B"], m["C"], st, m["A_log"], m["a"], m["dt_bias"], m["D"], cu)
    assert out.shape == (0, 2, 64) and torch.equal(new, st)


def test_strong_and_absent_decay():
    """Decays from none (dt near 0) to complete within a token (dt A of thousands) leave no infinity or NaN."""
    from gdn_b200 import ssm
    lens = [150, 90]
    m = make((240,), 4, 64, 1, 128, seed=5)
    m["A_log"] = torch.tensor([-20.0, 0.0, 5.0, 12.0], device="cuda")
    m["dt_bias"] = torch.tensor([30.0, -30.0, 3.0, 1.0], device="cuda")
    st = torch.randn(2, 4, 64, 128, device="cuda")
    cu = torch.tensor([0, 150, 240], device="cuda")
    out, new = ssm.run(m["x"], m["B"], m["C"], st, m["A_log"], m["a"], m["dt_bias"], m["D"], cu)
    check_packed(m, lens, st, out, new)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,P,G,Ns", [(4, 64, 2, 128), (3, 64, 1, 64), (2, 128, 1, 128), (2, 128, 2, 64)])
@pytest.mark.parametrize("B,T", [(1, 1), (5, 1), (3, 4), (2, 17)])
def test_pool(B, T, H, P, G, Ns, dtype):
    from gdn_b200 import ssm
    m = make((B, T), H, P, G, Ns, seed=B * 100 + T, skip=T != 4)
    pool = torch.randn(B + 3, H, P, Ns, device="cuda").to(dtype)
    slots = torch.randperm(B + 3, device="cuda")[:B].to(torch.int32)
    was = pool.clone()
    args = (m["x"], m["B"], m["C"], m["A_log"], m["a"], m["dt_bias"], m["D"], pool, slots)
    dry = ssm.run_pool(*args, no_state_update=True)
    assert torch.equal(pool, was)
    out = ssm.run_pool(*args)
    assert torch.equal(out, dry)
    for i, at in enumerate(slots.tolist()):
        y, ya, S, Sa = L.scan_ref(*(m[k][i] for k in ("x", "B", "C", "a")), m["A_log"], m["dt_bias"], m["D"], was[at])
        L.within(out[i], y, f32_slack(ya, T))
        L.within(pool[at], S, f32_slack(Sa, T))
        was[at] = pool[at]
    assert torch.equal(pool, was), "a slot of no sequence changed"


def test_pool_slots():
    from gdn_b200 import ssm
    m = make((4, 2), 2, 64, 1, 128)
    pool = torch.randn(6, 2, 64, 128, device="cuda")
    was = pool.clone()
    reads = torch.tensor([-1, 6, 2, 3], dtype=torch.int32, device="cuda")
    writes = torch.tensor([0, 1, -1, 5], dtype=torch.int32, device="cuda")
    out = ssm.run_pool(m["x"], m["B"], m["C"], m["A_log"], m["a"], m["dt_bias"], m["D"], pool, reads, writes)
    for i, (r, w) in enumerate(zip([None, None, 2, 3], [0, 1, None, 5])):
        S0 = was[r] if r is not None else torch.zeros(2, 64, 128)
        y, ya, S, Sa = L.scan_ref(*(m[k][i] for k in ("x", "B", "C", "a")), m["A_log"], m["dt_bias"], m["D"], S0)
        L.within(out[i], y, f32_slack(ya, 2))
        if w is not None:
            L.within(pool[w], S, f32_slack(Sa, 2))
    assert torch.equal(pool[2:5], was[2:5])


def test_tokens_after_a_prompt():
    """A prompt, then tokens over the pool, against the whole sequence."""
    from gdn_b200 import ssm
    T = 150
    m = make((T,), 4, 64, 2, 128, seed=9)
    n = 141
    cu = torch.tensor([0, n], device="cuda")
    head, state = ssm.run(m["x"][:n], m["B"][:n], m["C"][:n], None, m["A_log"], m["a"][:n], m["dt_bias"], m["D"], cu)
    slot = torch.zeros(1, dtype=torch.int32, device="cuda")
    outs = [ssm.run_pool(*(m[k][None, t:e] for k in ("x", "B", "C")), m["A_log"], m["a"][None, t:e], m["dt_bias"],
                         m["D"], state, slot) for t, e in ((n, n + 1), (n + 1, n + 6), (n + 6, T))]
    y, ya, S, Sa = L.scan_ref(*(m[k] for k in ("x", "B", "C", "a")), m["A_log"], m["dt_bias"], m["D"],
                              torch.zeros(4, 64, 128))
    L.within(torch.cat([head] + [o[0] for o in outs]), y, y_slack(ya, T))
    L.within(state[0], S, s_slack(Sa, T))


def test_refusals():
    from gdn_b200 import ssm
    m = make((10,), 4, 64, 2, 128)
    cu = torch.tensor([0, 10], device="cuda")
    ok = dict(x=m["x"], B=m["B"], C=m["C"], state=None, A_log=m["A_log"], a=m["a"], dt_bias=m["dt_bias"], D=m["D"],
              cu_seqlens=cu)
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    for exc, match, kw in [
            (TypeError, "x must", dict(x=m["x"].half())),
            (ValueError, "head size", dict(x=z(10, 4, 32))),
            (ValueError, "state size", dict(B=z(10, 2, 32), C=z(10, 2, 32))),
            (ValueError, "multiple", dict(B=z(10, 3, 128), C=z(10, 3, 128))),
            (ValueError, "C must", dict(C=z(10, 1, 128))),
            (ValueError, "contiguous", dict(x=z(10, 4, 128)[..., :64])),
            (TypeError, "A_log", dict(A_log=z(4))),
            (ValueError, "a must", dict(a=z(9, 4))),
            (TypeError, "state", dict(state=z(1, 4, 64, 128))),
            (ValueError, "at least one", dict(cu_seqlens=cu[:1])),
            (ValueError, "CUDA|same device", dict(B=m["B"].cpu()))]:
        with pytest.raises(exc, match=match):
            ssm.run(**{**ok, **kw})
    st = z(1, 4, 64, 128, dt=torch.float32)
    with pytest.raises(ValueError, match="overlaps"):
        ssm.run(**{**ok, "state": st}, new_state=st)


@pytest.fixture(autouse=True)
def no_timeouts():
    """No kernel of a test gave up on a bounded wait."""
    import ctypes
    from gdn_b200 import _native as N
    yield
    status = ctypes.c_uint32()
    assert N.lib().gdn_read_status(ctypes.byref(status), 1) == N.GDN_OK and status.value == 0


@pytest.mark.parametrize("what", ["x nan", "x inf", "a nan", "a inf", "B nan", "C inf"])
def test_values_that_are_not_finite_stay_where_they_belong(what):
    """Row h, p from token j on (x), head h from token j on (a), everything of the group from token j on (B), token
    j of the group (C): nothing earlier, no other head, no other sequence."""
    from gdn_b200 import ssm
    H, P, G, Ns = 4, 64, 2, 128
    lens = [100, 137, 50]
    m = make((287,), H, P, G, Ns, seed=3)
    cu = torch.tensor([0, 100, 237, 287], device="cuda")
    run = lambda m: ssm.run(m["x"], m["B"], m["C"], None, m["A_log"], m["a"], m["dt_bias"], m["D"], cu)  # noqa: E731
    want, want_s = run(m)
    for j in (100, 100 + 63, 100 + 70, 236):
        name, value = what.split()
        bad = {k: (v.clone() if v is not None else None) for k, v in m.items()}
        bad[name][(j, 1, 5) if name in ("x", "B", "C") else (j, 1)] = float(value)
        got, got_s = run(bad)
        y = torch.zeros(287, H, P, dtype=torch.bool, device="cuda")   # what may (and has to) differ
        s = torch.zeros(3, H, P, Ns, dtype=torch.bool, device="cuda")
        if name == "x":
            y[j:237, 1, 5], s[1, 1, 5] = True, True
        elif name == "a":
            y[j:237, 1], s[1, 1] = True, True
        elif name == "B":
            y[j:237, 2:], s[1, 2:, :, 5] = True, True
        else:
            y[j, 2:] = True
        assert torch.equal(got[~y], want[~y]), f"{what} at {j} reached other outputs"
        assert torch.equal(got_s[~s], want_s[~s]), f"{what} at {j} reached other states"
        assert not got_s[s].isfinite().any()
        if name != "a" or value == "nan":
            assert not got[y].isfinite().any()


def test_same_answer_twice_and_beside_other_sequences():
    """Bitwise: no order of execution enters the sums, and a sequence's results do not depend on its neighbours."""
    from gdn_b200 import ssm
    lens = [300, 65, 0, 190]
    m = make((sum(lens),), 6, 64, 2, 128, seed=11)
    st = torch.randn(4, 6, 64, 128, device="cuda")
    cu = torch.tensor([0, 300, 365, 365, 555], device="cuda")
    run = lambda t0, t1, st, cu: ssm.run(m["x"][t0:t1], m["B"][t0:t1], m["C"][t0:t1], st, m["A_log"],  # noqa: E731
                                         m["a"][t0:t1], m["dt_bias"], m["D"], cu)
    y, s = run(0, 555, st, cu)
    y2, s2 = run(0, 555, st, cu)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    y3, s3 = run(300, 365, st[1:2], torch.tensor([0, 65], device="cuda"))
    assert torch.equal(y[300:365], y3) and torch.equal(s[1:2], s3)


@pytest.mark.parametrize("H,P,G,Ns,lens,state", [
    (2, 64, 1, 128, [1900], True),               # few pairs: pieces of a few chunks
    (2, 128, 2, 64, [3300, 0, 2700, 5], True),
    (3, 64, 1, 64, [2048 + 33], False),
    (4, 64, 1, 128, [64 * 32, 64 * 30 + 1], True),  # a last piece of one token
])
def test_sequences_cut_into_pieces(H, P, G, Ns, lens, state):
    """Calls of few (sequence, head) pairs, whose sequences run as pieces joined by their decays."""
    from gdn_b200 import ssm
    assert ssm.workspace_bytes(sum(lens), len(lens), H, G, P, Ns) > 0
    m = make((sum(lens),), H, P, G, Ns, seed=sum(lens))
    st = torch.randn(len(lens), H, P, Ns, device="cuda") if state else None
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0)
    out, new = ssm.run(m["x"], m["B"], m["C"], st, m["A_log"], m["a"], m["dt_bias"], m["D"], cu)
    check_packed(m, lens, st, out, new)


def test_one_long_sequence_among_many():
    """A batch that fills the GPU, one of whose sequences is long enough to be cut."""
    from gdn_b200 import ssm
    lens = [40] * 70 + [9000] + [33] * 40
    H, G = 8, 1
    assert ssm.workspace_bytes(sum(lens), len(lens), H, G, 64, 128) > 0
    m = make((sum(lens),), H, 64, G, 128, seed=2)
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0)
    out, new = ssm.run(m["x"], m["B"], m["C"], None, m["A_log"], m["a"], m["dt_bias"], m["D"], cu)
    # the sequences on both sides, and the whole long one
    for i in (0, 69, 70, 71, 110):
        a, b = int(cu[i]), int(cu[i + 1])
        y, ya, S, Sa = L.scan_ref(*(m[k][a:b] for k in ("x", "B", "C", "a")), m["A_log"], m["dt_bias"], m["D"],
                                  torch.zeros(H, 64, 128))
        L.within(out[a:b], y, y_slack(ya, b - a))
        L.within(new[i], S, s_slack(Sa, b - a))


def test_many_sequences_equal_one_call_each():
    """More (sequence, tile) pairs than SMs: what runs beside a sequence changes no bit of it."""
    from gdn_b200 import ssm
    lens = [130, 0, 64, 700, 1, 65, 700, 320]
    H = 64
    m = make((sum(lens),), H, 64, 2, 128, seed=4)
    st = torch.randn(len(lens), H, 64, 128, device="cuda")
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0)
    out, new = ssm.run(m["x"], m["B"], m["C"], st, m["A_log"], m["a"], m["dt_bias"], m["D"], cu)
    for i, n in enumerate(lens):
        a, b = int(cu[i]), int(cu[i + 1])
        # (a short one alone takes the token-by-token kernel, a long one alone runs in pieces)
        if n > 16 and ssm.workspace_bytes(n, 1, H, 2, 64, 128) == 0:
            o, s = ssm.run(m["x"][a:b], m["B"][a:b], m["C"][a:b], st[i:i + 1], m["A_log"], m["a"][a:b], m["dt_bias"],
                           m["D"], torch.tensor([0, n], device="cuda"))
            assert torch.equal(out[a:b], o) and torch.equal(new[i:i + 1], s)
    assert torch.equal(new[1], st[1])


def test_one_long_sequence_among_some():
    from gdn_b200 import ssm
    lens = [40] * 20 + [4500] + [33] * 20
    H = 8
    assert ssm.workspace_bytes(sum(lens), len(lens), H, 1, 64, 128) > 0
    m = make((sum(lens),), H, 64, 1, 128, seed=6)
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0)
    out, new = ssm.run(m["x"], m["B"], m["C"], None, m["A_log"], m["a"], m["dt_bias"], m["D"], cu)
    for i in (0, 19, 20, 21, 40):
        a, b = int(cu[i]), int(cu[i + 1])
        y, ya, S, Sa = L.scan_ref(*(m[k][a:b] for k in ("x", "B", "C", "a")), m["A_log"], m["dt_bias"], m["D"],
                                  torch.zeros(H, 64, 128))
        L.within(out[a:b], y, y_slack(ya, b - a))
        L.within(new[i], S, s_slack(Sa, b - a))


def test_long_sequences_among_hundreds():
    """More sequences than one round of the search for a piece covers (128), with several cut ones."""
    from gdn_b200 import ssm
    lens = [20 + i % 50 for i in range(400)]
    lens[3], lens[140], lens[399], lens[200] = 4000, 5001, 2500, 0
    H = 8
    assert ssm.workspace_bytes(sum(lens), len(lens), H, 1, 64, 128) > 0
    m = make((sum(lens) + 70,), H, 64, 1, 128, seed=7)
    st = torch.randn(len(lens), H, 64, 128, device="cuda")
    cu = torch.tensor([6] + lens, device="cuda").cumsum(0)
    out = torch.full_like(m["x"], 7.0)
    _, new = ssm.run(m["x"], m["B"], m["C"], st, m["A_log"], m["a"], m["dt_bias"], m["D"], cu, output=out)
    assert (out[:6] == 7).all() and (out[int(cu[-1]):] == 7).all()
    assert torch.equal(new[200], st[200])
    for i in (0, 2, 3, 4, 127, 128, 139, 140, 141, 199, 201, 255, 256, 398, 399):
        a, b = int(cu[i]), int(cu[i + 1])
        y, ya, S, Sa = L.scan_ref(*(m[k][a:b] for k in ("x", "B", "C", "a")), m["A_log"], m["dt_bias"], m["D"], st[i])
        L.within(out[a:b], y, y_slack(ya, b - a))
        L.within(new[i], S, s_slack(Sa, b - a))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,P,G,Ns", [(4, 64, 2, 128), (3, 64, 1, 64), (2, 128, 1, 128), (2, 128, 2, 64)])
@pytest.mark.parametrize("T", [2, 3, 5, 33])
def test_pool_of_few_tokens(T, H, P, G, Ns, dtype):
    from gdn_b200 import ssm
    B = 3
    m = make((B, T), H, P, G, Ns, seed=T + H)
    pool = torch.randn(B + 2, H, P, Ns, device="cuda").to(dtype)
    before = pool.clone()
    ins, outs = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([4, 0, -1], [1, 3, 2]))
    out = ssm.run_pool(m["x"], m["B"], m["C"], m["A_log"], m["a"], m["dt_bias"], m["D"], pool, ins, outs)
    for i in range(B):
        S0 = before[int(ins[i])] if ins[i] >= 0 else torch.zeros(H, P, Ns)
        y, ya, S, Sa = L.scan_ref(*(m[k][i] for k in ("x", "B", "C", "a")), m["A_log"], m["dt_bias"], m["D"], S0)
        L.within(out[i], y, f32_slack(ya, T))
        L.within(pool[int(outs[i])], S, f32_slack(Sa, T))
    assert torch.equal(pool[0], before[0]) and torch.equal(pool[4], before[4])
