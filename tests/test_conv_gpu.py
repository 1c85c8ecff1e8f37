"""The short convolution against its 64-bit definition (GPU)."""
import pytest
import torch

import layer_oracle as L

pytestmark = pytest.mark.gpu

# fp32: at most 5 products and additions (5 2^-24 of the magnitude), and silu, whose 2^x sees its
# argument rounded: |x| 2^-23 relative.  At the magnitudes here (below 64) 2^-16 covers both.
SLACK = 2.0 ** -16


def make(lens, D, W, dtype, bias, state, seed=0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, T = len(lens), sum(lens)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    return dict(x=r(T, D + pad)[:, :D], weight=r(D, W), bias=r(D) if bias else None,
                state=r(n, W - 1, D) if state else None,
                cu=torch.tensor([0] + lens, device="cuda").cumsum(0))


def check(m, lens, out, new, act=True):
    W, D = m["weight"].shape[1], m["x"].shape[1]
    at = 0
    for i, n in enumerate(lens):
        before = m["state"][i] if m["state"] is not None else torch.zeros(W - 1, D)
        ref, mag, st = L.conv_ref(m["x"][at:at + n], m["weight"], m["bias"], before, act)
        L.within(out[at:at + n], ref, SLACK * mag)
        assert torch.equal(L.d(new[i]), st), f"state of sequence {i}"
        at += n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("lens,state", [([1], False), ([1, 1, 2, 3, 5], True), ([0, 4, 0, 0, 70, 0], True),
                                        ([31, 33, 32, 64, 1], False), ([200], True)])
def test_packed(lens, state, W, dtype):
    from gdn_b200 import conv
    m = make(lens, 72, W, dtype, bias=W != 3, state=state)
    out, new = conv.run(m["x"], m["weight"], m["bias"], m["state"], m["cu"])
    check(m, lens, out, new)


@pytest.mark.parametrize("D,pad", [(8, 0), (1024, 8), (1032, 0), (2056, 40)])
def test_channels_strides_and_no_activation(D, pad):
    from gdn_b200 import conv
    lens = [40, 3, 90]
    m = make(lens, D, 4, torch.bfloat16, True, True, seed=D, pad=pad)
    out, new = conv.run(m["x"], m["weight"], m["bias"], m["state"], m["cu"].to(torch.int32), silu=False)
    check(m, lens, out, new, act=False)


def test_many_sequences():
    """More sequences than one round of the search for a tile's sequence covers (32), and than two (1024)."""
    from gdn_b200 import conv
    for n in (33, 1100):
        lens = [(7 * i) % 5 for i in range(n)]
        m = make(lens, 8, 4, torch.bfloat16, False, True, seed=n)
        out, new = conv.run(m["x"], m["weight"], m["bias"], m["state"], m["cu"])
        check(m, lens, out, new)


def test_splits_equal_the_whole():
    from gdn_b200 import conv
    m = make([50, 20], 2048 + 72 + 8, 4, torch.bfloat16, True, True)
    whole, new = conv.run(m["x"], m["weight"], m["bias"], m["state"], m["cu"])
    for parts in ([2128], [2048, 80], [8, 2048, 72], [1024, 1024, 72, 8]):
        outs, new2 = conv.run(m["x"], m["weight"], m["bias"], m["state"], m["cu"], splits=parts)
        assert all(o.is_contiguous() for o in outs)
        assert torch.equal(torch.cat(outs, -1), whole) and torch.equal(new, new2)


def test_rows_of_no_sequence_stay():
    from gdn_b200 import conv
    m = make([60], 64, 4, torch.bfloat16, False, False)
    cu = torch.tensor([5, 20, 20, 41], device="cuda")
    out = torch.full((60, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    conv.run(m["x"], m["weight"], None, None, cu, outputs=[out])
    assert (out[:5] == 7).all() and (out[41:] == 7).all()
    ref, mag, _ = L.conv_ref(m["x"][20:41], m["weight"], None, torch.zeros(3, 64))
    L.within(out[20:41], ref, SLACK * mag)


def test_no_tokens_keeps_the_states():
    from gdn_b200 import conv
    m = make([0, 0], 64, 4, torch.bfloat16, False, True)
    out, new = conv.run(m["x"], m["weight"], None, m["state"], m["cu"])
    assert out.shape == (0, 64) and torch.equal(new, m["state"])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("B,T", [(1, 1), (3, 1), (5, 2), (2, 9)])
def test_pool(B, T, W, dtype):
    from gdn_b200 import conv
    g = torch.Generator(device="cuda").manual_seed(B * 10 + T)
    D = 1096
    x = torch.randn(B, T + 1, D + 16, generator=g, device="cuda").to(dtype)[:, :T, :D]
    weight = torch.randn(D, W, generator=g, device="cuda").to(dtype)
    bias = torch.randn(D, generator=g, device="cuda").to(dtype)
    pool = torch.randn(B + 4, W - 1, D, generator=g, device="cuda").to(dtype)
    slots = torch.randperm(B + 4, generator=g, device="cuda")[:B].to(torch.int32)
    was = pool.clone()
    outs = conv.run_pool(x, weight, bias, pool, slots, splits=[1024, 72])
    out = torch.cat(outs, -1)
    for i in range(B):
        ref, mag, st = L.conv_ref(x[i], weight, bias, was[slots[i].item()])
        L.within(out[i], ref, SLACK * mag)
        assert torch.equal(L.d(pool[slots[i].item()]), st)
        was[slots[i].item()] = pool[slots[i].item()]
    assert torch.equal(pool, was), "a slot of no sequence changed"


def test_pool_slots():
    """Negative and too large read slots are zero states, such write slots are not written; other slots move."""
    from gdn_b200 import conv
    D, W = 64, 4
    x = torch.randn(4, 2, D, device="cuda").to(torch.bfloat16)
    weight = torch.randn(D, W, device="cuda").to(torch.bfloat16)
    pool = torch.randn(6, W - 1, D, device="cuda").to(torch.bfloat16)
    was = pool.clone()
    reads = torch.tensor([-1, 6, 2, 3], dtype=torch.int32, device="cuda")
    writes = torch.tensor([0, 1, -1, 5], dtype=torch.int32, device="cuda")
    out = conv.run_pool(x, weight, None, pool, reads, writes)
    for i, (r, w) in enumerate(zip([None, None, 2, 3], [0, 1, None, 5])):
        before = was[r] if r is not None else torch.zeros(W - 1, D)
        ref, mag, st = L.conv_ref(x[i], weight, None, before)
        L.within(out[i], ref, SLACK * mag)
        if w is not None:
            assert torch.equal(L.d(pool[w]), st)
    assert torch.equal(pool[2:5], was[2:5])


def test_tokens_after_a_prompt_equal_the_whole_prompt():
    from gdn_b200 import conv
    m = make([37], 128, 4, torch.bfloat16, True, False)
    cu = torch.tensor([0, 30], device="cuda")
    whole, end = conv.run(m["x"], m["weight"], m["bias"], None, m["cu"])
    head, state = conv.run(m["x"][:30], m["weight"], m["bias"], None, cu)
    slot = torch.zeros(1, dtype=torch.int32, device="cuda")
    outs = [conv.run_pool(m["x"][None, t:e], m["weight"], m["bias"], state, slot)
            for t, e in ((30, 31), (31, 35), (35, 37))]
    assert torch.equal(torch.cat([head] + [o[0] for o in outs]), whole) and torch.equal(state, end)


def test_extremes():
    """Infinities and NaN stay in the rows and channels that read them."""
    from gdn_b200 import conv
    m = make([12], 16, 4, torch.bfloat16, False, False)
    x = m["x"].clone()
    x[5, 3] = float("nan")
    x[5, 4] = float("inf")
    got, _ = conv.run(x, m["weight"], None, None, m["cu"])
    want, _ = conv.run(m["x"], m["weight"], None, None, m["cu"])
    reach = torch.zeros_like(got, dtype=torch.bool)
    reach[5:9, 3:5] = True
    assert torch.equal(got[~reach], want[~reach])
    assert got[5:9, 3].isnan().all() and not got[5:9, 4].isfinite().any()


def test_refusals():
    from gdn_b200 import conv
    m = make([10], 64, 4, torch.bfloat16, False, False)
    ok = (m["x"], m["weight"], None, None, m["cu"])

    def bad(exc, match, i=None, v=None, **kw):
        args = list(ok)
        if i is not None:
            args[i] = v
        with pytest.raises(exc, match=match):
            conv.run(*args, **kw)

    bad(TypeError, "bfloat16 or float16", 0, m["x"].float())
    bad(ValueError, "contiguous", 0, m["x"].t().contiguous().t())
    bad(ValueError, "multiple of 8", 0, m["x"][:, :60])
    bad(ValueError, "at least dim apart", 0, m["x"][:1].expand(10, 64))
    bad(TypeError, "weight", 1, m["weight"].half())
    bad(ValueError, "width", 1, torch.zeros(64, 5, dtype=torch.bfloat16, device="cuda"))
    bad(ValueError, "state", 3, torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda"))
    bad(ValueError, "at least one sequence", 4, m["cu"][:1])
    bad(ValueError, "sum", splits=[32])
    bad(ValueError, "multiples of 8", splits=[60, 4])
    bad(ValueError, "at most 4", splits=[8] * 8)
    bad(ValueError, "one tensor per split", outputs=[])
    bad(ValueError, "same device|CUDA", 1, m["weight"].cpu())
    new = torch.zeros(1, 3, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        conv.run(*ok[:3], new, m["cu"], new_state=new)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("pool", [False, True])
def test_lowest_values(pool, dtype):
    """silu of sums at the bottom of the range is 0, of -inf NaN, and the neighbouring channels see neither."""
    from gdn_b200 import conv
    m = make([40], 64, 4, dtype, True, True, seed=9)
    m["x"][3, ::2] = torch.finfo(dtype).min
    m["x"][20, 1] = -1e4
    m["x"][30, 2::2] = -float("inf")
    w = m["weight"].abs().clamp(0.1, 1.0)
    if pool:
        pl = m["state"].clone()
        out = conv.run_pool(m["x"][None], w, m["bias"], pl, torch.zeros(1, dtype=torch.int32, device="cuda"))[0]
    else:
        out, _ = conv.run(m["x"], w, m["bias"], m["state"], m["cu"])
    ref, mag, _ = L.conv_ref(m["x"].clamp(min=torch.finfo(dtype).min), w, m["bias"], m["state"][0])
    inf = torch.zeros(40, 64, dtype=torch.bool)
    inf[30:34, 2::2] = True
    low = (mag > 1e3) & ~inf
    got = L.d(out)
    assert low[3:7, ::2].all() and (got[low] == 0).all() and got[inf].isnan().all()
    L.within(out[~(low | inf).to(out.device)], ref[~(low | inf)], SLACK * mag[~(low | inf)])
