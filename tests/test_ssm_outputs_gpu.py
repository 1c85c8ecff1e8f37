"""What the scan of prompts owes its outputs beyond the elementwise bounds of its other tests (GPU):
one rounding, and values that are not finite only where the recurrence has them."""
import ctypes

import pytest
import torch

import layer_oracle as L
from test_ssm_gpu import make

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_timeouts():
    """No kernel of a test gave up on a bounded wait."""
    from gdn_b200 import _native as N
    yield
    status = ctypes.c_uint32()
    assert N.lib().gdn_read_status(ctypes.byref(status), 1) == N.GDN_OK and status.value == 0


def rounded_once(got, ref, slack):
    """``got`` is the rounding of a value v with |v - ref| <= slack.  rn(v) is the nearest to v, so
    |rn(v) - v| <= |rn(ref) - v| <= |rn(ref) - ref| + slack, and |rn(v) - ref| <= |rn(ref) - ref| + 2 slack.
    (rn(ref) itself goes through fp32: 2^-23 of ref.)"""
    own = (ref.to(got.dtype).double() - ref).abs()
    err = (L.d(got) - ref).abs()
    bound = own + 2 * slack + 2.0 ** -23 * ref.abs() + L.TINY[got.dtype]
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside the bound, worst {float((err - bound).max()):.3g}"


def out_slack(ya, n):
    """Operands of two bf16 terms leave half a step of half a step, 2^-16, of a term; the fp32 arithmetic of n tokens
    is off by (8 n + 200) 2^-24 of the magnitude."""
    return (2.0 ** -16 + (8 * n + 200) * 2.0 ** -24) * ya


def run(m, lens, state=None):
    from gdn_b200 import ssm
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0)
    return ssm.run(m["x"], m["B"], m["C"], state, m["A_log"], m["a"], m["dt_bias"], m["D"], cu)


def reference(m, lens, state=None):
    H, P = m["x"].shape[1:]
    refs, at = [], 0
    for i, n in enumerate(lens):
        S0 = state[i] if state is not None else torch.zeros(H, P, m["B"].shape[2])
        refs.append(L.scan_ref(*(m[k][at:at + n] for k in ("x", "B", "C", "a")), m["A_log"], m["dt_bias"], m["D"], S0))
        at += n
    return [torch.cat([r[0] for r in refs]), torch.cat([r[1] for r in refs]),
            torch.stack([r[2] for r in refs]), torch.stack([r[3] for r in refs])]


@pytest.mark.parametrize("H,P,G,Ns", [(3, 64, 1, 128), (2, 128, 1, 128), (4, 64, 2, 64), (2, 128, 2, 64)])
@pytest.mark.parametrize("lens", [[150, 64, 65], [1900]])
def test_skip_term_is_rounded_once(lens, H, P, G, Ns):
    """With steps that are next to nothing the output is D x, of a D between two bf16 values."""
    m = make((sum(lens),), H, P, G, Ns, seed=21)
    m["dt_bias"].fill_(-40.0)
    m["D"] = torch.tensor([1.0038, -3.0131, 0.7515], device="cuda").repeat(2)[:H].contiguous()
    out, _ = run(m, lens)
    y, ya, _, _ = reference(m, lens)
    rounded_once(out, y, out_slack(ya, 1))


@pytest.mark.parametrize("H,P,G,Ns", [(3, 64, 1, 128), (2, 128, 1, 128), (4, 64, 2, 64), (2, 128, 2, 64)])
def test_outputs_within_a_chunk_are_rounded_once(H, P, G, Ns):
    lens = [64, 63, 17, 40]
    m = make((sum(lens),), H, P, G, Ns, seed=20, skip=H != 4)
    out, _ = run(m, lens)
    y, ya, _, _ = reference(m, lens)
    rounded_once(out, y, out_slack(ya, 64))


@pytest.mark.parametrize("H,P,G,Ns,lens,state", [
    (3, 64, 1, 128, [200, 65, 130], True), (2, 128, 1, 128, [129, 0, 400], True), (4, 64, 2, 64, [700], True),
    (2, 128, 2, 64, [64, 100], True),
    (6, 128, 2, 128, [150, 64], False),            # three heads of 128 a group
    (2, 64, 1, 128, [1900], True), (2, 128, 2, 64, [3300, 5], False)])  # in pieces
def test_outputs_and_states_of_long_sequences(H, P, G, Ns, lens, state):
    """Outputs rounded once.  States as fp32 sums give them, by their norm too: three bf16 terms of W leave 2^-24 of a
    term; each token's decay and product are off by 8 2^-24 at most, and such errors, of either sign, come to less
    than a millionth of the whole (two terms of W left 2.6e-6)."""
    m = make((sum(lens),), H, P, G, Ns, seed=24 + H)
    st = torch.randn(len(lens), H, P, Ns, device="cuda") if state else None
    out, new = run(m, lens, st)
    y, ya, S, _ = reference(m, lens, st)
    rounded_once(out, y, out_slack(ya, max(lens)))
    own = (y.to(torch.bfloat16).double() - y).norm()
    assert (L.d(out) - y).norm() <= 1.02 * own
    for i, n in enumerate(lens):
        if n or st is not None:
            assert (L.d(new[i]) - S[i]).norm() <= 1e-6 * S[i].norm()


@pytest.mark.parametrize("value", ["nan", "inf", "-inf", "3e38"])
@pytest.mark.parametrize("P,lens", [(64, [100, 70]), (128, [100, 70]), (64, [1900])])
def test_a_skip_that_is_not_finite_stays_in_its_head(P, lens, value):
    """Two heads of 64 share a tile's products."""
    m = make((sum(lens),), 4, P, 2, 128, seed=22)
    want, want_s = run(m, lens)
    for head in (1, 2):
        bad = dict(m, D=m["D"].clone())
        bad["D"][head] = float(value)
        got, got_s = run(bad, lens)
        rest = [h for h in range(4) if h != head]
        assert torch.equal(got[:, rest], want[:, rest]) and torch.equal(got_s, want_s)
        if value == "3e38":  # (finite, and so are its products with x below 1)
            y, ya, _, _ = reference(bad, lens)
            small = bad["x"][:, head].abs().cpu() < 1
            rounded_once(got[:, head][small.cuda()], y[:, head][small], out_slack(ya[:, head][small], max(lens)))
        else:
            assert not got[:, head].isfinite().any()


@pytest.mark.parametrize("lens", [[100, 70], [1900]])
def test_a_step_that_overflows_stays_in_its_head(lens):
    """A step of 3e38 at one token: the weights of its head within the chunk overflow."""
    m = make((sum(lens),), 4, 64, 2, 128, seed=25)
    want, want_s = run(m, lens)
    for head in (1, 2):
        bad = dict(m, a=m["a"].clone())
        bad["a"][40, head] = 3e38
        got, got_s = run(bad, lens)
        rest = [h for h in range(4) if h != head]
        assert torch.equal(got[:, rest], want[:, rest]) and torch.equal(got_s[:, rest], want_s[:, rest])
        assert torch.equal(got[:40], want[:40]) and torch.equal(got[lens[0]:], want[lens[0]:])


@pytest.mark.parametrize("what", ["x nan", "x inf", "a nan", "B nan", "C inf"])
def test_values_that_are_not_finite_in_a_cut_sequence(what):
    """A bad value in a piece that is not the last: later pieces of what it reaches, nothing else."""
    from gdn_b200 import ssm
    lens = [1900, 300]
    T, H, P, G, Ns = sum(lens), 4, 64, 2, 128
    assert ssm.workspace_bytes(T, len(lens), H, G, P, Ns) > 0
    m = make((T,), H, P, G, Ns, seed=23)
    want, want_s = run(m, lens)
    name, value = what.split()
    for j in (0, 70, 1000):
        bad = dict(m, **{name: m[name].clone()})
        bad[name][(j, 1, 5) if name in ("x", "B", "C") else (j, 1)] = float(value)
        got, got_s = run(bad, lens)
        y = torch.zeros(T, H, P, dtype=torch.bool, device="cuda")
        s = torch.zeros(2, H, P, Ns, dtype=torch.bool, device="cuda")
        if name == "x":
            y[j:1900, 1, 5], s[0, 1, 5] = True, True
        elif name == "a":
            y[j:1900, 1], s[0, 1] = True, True
        elif name == "B":
            y[j:1900, 2:], s[0, 2:, :, 5] = True, True
        else:
            y[j, 2:] = True
        assert torch.equal(got[~y], want[~y]) and torch.equal(got_s[~s], want_s[~s])
        assert not got[y].isfinite().any() and not got_s[s].isfinite().any()


@pytest.mark.parametrize("P", [64, 128])
@pytest.mark.parametrize("lens", [[64, 40], [200, 333], [1900]])
def test_resets_between_weak_decays(P, lens):
    """Tokens that end a head's memory between tokens that keep it: decays of e^-96 and e^-0.005 within a chunk.  What
    the weak ones leave is a difference of sums that the strong ones have made large."""
    T, H = sum(lens), 4
    m = make((T,), H, P, 2, 128, seed=26)
    g = torch.Generator(device="cuda").manual_seed(27)
    strong = torch.rand(T, H, generator=g, device="cuda") < 0.3
    m["a"] = torch.where(strong, 6.0, -8.0).to(torch.bfloat16)
    m["A_log"] = torch.full((H,), 2.7726, device="cuda")
    m["dt_bias"] = torch.zeros(H, device="cuda")
    m["x"] = torch.where(strong[..., None], 2.0 ** -10 * m["x"], 4 * m["x"])
    st = torch.randn(len(lens), H, P, 128, device="cuda")
    out, new = run(m, lens, st)
    y, ya, S, Sa = reference(m, lens, st)
    rounded_once(out, y, out_slack(ya, 64))
    for i in range(len(lens)):
        L.within(new[i], S[i], (8 * 64 + 200) * 2.0 ** -24 * Sa[i])


def weak_decays(T, bias):
    """Decays of 1 - 3e-4 and 1 - 2e-3: a state that remembers thousands of tokens."""
    H, P, Ns = 4, 64, 64
    m = make((T,), H, P, 1, Ns, seed=28, skip=False)
    m["a"] = (0.5 * m["a"].float()).to(torch.bfloat16)
    m["A_log"], m["dt_bias"] = torch.zeros(H, device="cuda"), torch.full((H,), bias, device="cuda")
    st = torch.randn(1, H, P, Ns, device="cuda")
    S = st[0].double()
    dt = torch.nn.functional.softplus(m["a"].double() + bias, threshold=1e9)
    for t in range(T):
        S = S * torch.exp(-dt[t])[:, None, None] + (dt[t][:, None] * m["x"][t].double())[..., None] * m["B"][t].double()[:, None]
    return m, st, S


@pytest.mark.parametrize("bias", [-8.0, -6.0])
def test_long_memory_token_by_token(bias):
    """Each token's decay is rounded to fp32, to either side: T tokens add up to sqrt(T) 2^-24, 3.3e-6 for 3000.  An
    exponential that errs to one side adds up to T times that (4.6e-5)."""
    from gdn_b200 import ssm
    T = 3000
    m, st, S = weak_decays(T, bias)
    pool, slot = st.clone(), torch.zeros(1, dtype=torch.int32, device="cuda")
    for t0, t1 in ((0, 1000), (1000, 1001), (1001, 1003), (1003, T)):
        ssm.run_pool(*(m[k][None, t0:t1] for k in ("x", "B", "C")), m["A_log"], m["a"][None, t0:t1], m["dt_bias"], None, pool, slot)
    assert (pool[0].double() - S).norm() <= 3.3e-6 * S.norm()


@pytest.mark.parametrize("bias", [-8.0, -6.0])
def test_long_memory_of_a_prompt(bias):
    """A rounding a chunk: 47 of them, sqrt(47) 2^-24, and the sums' own, a few 2^-24."""
    T = 3000
    m, st, S = weak_decays(T, bias)
    _, new = run(m, [T], st)
    assert (new[0].double() - S).norm() <= 1e-6 * S.norm()
