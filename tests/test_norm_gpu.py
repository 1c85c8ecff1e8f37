"""The root-mean-square norm against its 64-bit definition (GPU)."""
import pytest
import torch

import layer_oracle as L

pytestmark = pytest.mark.gpu
DIMS = [8, 64, 72, 128, 200, 256, 264, 1024, 1032, 2048, 4096, 4104, 8192, 16384]


def make(rows, D, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return r(rows, D).to(dtype), (1 + 0.1 * r(D)).to(dtype), (3 * r(rows, D)).to(dtype), r(rows, D).to(dtype)


def slack(y, D):
    """fp32: D squares and additions under a square root (D / 2 2^-24 at most), and a handful of products."""
    return (D / 2 + 64) * 2.0 ** -24 * y.abs()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", DIMS)
def test_plain_and_residual(D, dtype):
    from gdn_b200 import norm
    for rows in (1, 37):
        x, w, res, _ = make(rows, D, dtype, D)
        y, _ = L.norm_ref(x, w, 1e-6)
        L.within(norm.run(x, w, 1e-6), y, slack(y, D))
        y, h = L.norm_ref(x, w, 1e-5, residual=res)
        out, new = norm.run(x, w, 1e-5, residual=res)
        L.within(out, y, slack(y, D))
        L.within(new, h, 2.0 ** -24 * h.abs())
        same = res.clone()
        out2, new2 = norm.run(x, w, 1e-5, residual=same, residual_out=same)  # in place
        assert new2.data_ptr() == same.data_ptr() and torch.equal(out, out2) and torch.equal(new, same)


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("D", [64, 128, 136, 4096])
def test_gate(D, first):
    from gdn_b200 import norm
    x, w, _, gate = make(65, D, torch.bfloat16, D)
    y, _ = L.norm_ref(x, w, 1e-6, gate=gate, gate_first=first)
    # silu's 2^x sees its argument rounded: |gate| 2^-23, with |gate| < 8
    L.within(norm.run(x, w, 1e-6, gate=gate, gate_first=first), y, slack(y, D) + 2.0 ** -20 * y.abs())
    x3, g3 = x.view(5, 13, D), gate.view(5, 13, D)
    assert torch.equal(norm.run(x3, w, 1e-6, gate=g3, gate_first=first).view(65, D),
                       norm.run(x, w, 1e-6, gate=gate, gate_first=first))


@pytest.mark.parametrize("mode", ["plain", "residual", "after", "before"])
@pytest.mark.parametrize("D,group", [(8, 0), (128, 0), (128, 128), (200, 0), (384, 128), (640, 128), (1152, 128),
                                     (4096, 0), (4096, 128), (5120, 128), (16384, 0), (16384, 128)])
def test_e4m3(D, group, mode):
    from gdn_b200 import norm
    rows = 19
    x, w, res, gate = make(rows, D, torch.bfloat16, D + group)
    kw = dict(residual=res) if mode == "residual" else dict(gate=gate, gate_first=mode == "before") \
        if mode != "plain" else {}
    y, h = L.norm_ref(x, w, 1e-6, **kw)
    out = norm.run_fp8(x, w, 1e-6, group_size=group, **kw)
    q, scale = out[0], out[1]
    assert q.dtype == torch.float8_e4m3fn and scale.shape == ((rows, D // group) if group else (rows,))
    blocks = y.view(rows, D // group if group else 1, -1)
    want = blocks.abs().amax(-1) / 448
    rel = (D / 2 + 96) * 2.0 ** -24 + 2.0 ** -20
    s = L.d(scale).view(rows, -1)
    assert ((s - want).abs() <= rel * want).all()
    # the quotient is off by `rel`, then rounded: half a step is 2^-4 relative, or 2^-10 below the normal range
    quo = blocks / want[..., None]
    got = q.float().cpu().double().view_as(quo)
    assert ((got - quo).abs() <= 2.0 ** -4 * quo.abs() * (1 + 4 * rel) + 2.0 ** -10 + 4 * rel * quo.abs()).all()
    if mode == "residual":
        L.within(out[2], h, 2.0 ** -24 * h.abs())


def test_strides():
    from gdn_b200 import norm
    wide = torch.randn(21, 1024, device="cuda").to(torch.bfloat16)
    w = torch.randn(256, device="cuda").to(torch.bfloat16)
    x, res, gate = wide[:, :256], wide[:, 264:520], wide[:, 640:896]
    out, new = norm.run(x, w, residual=res)
    out2, new2 = norm.run(x.contiguous(), w, residual=res.contiguous())
    assert torch.equal(out, out2) and torch.equal(new, new2)
    assert torch.equal(norm.run(x, w, gate=gate), norm.run(x.contiguous(), w, gate=gate.contiguous()))


def test_zero_tiny_and_nan_rows():
    from gdn_b200 import norm
    D = 256
    x = torch.randn(6, D, device="cuda").to(torch.bfloat16)
    w = torch.ones(D, device="cuda", dtype=torch.bfloat16)
    x[1] = 0
    x[2] = 1e-30
    x[3, 200] = float("nan")
    x[4, 7] = float("inf")
    clean = torch.tensor([0, 1, 2, 5], device="cuda")
    out = norm.run(x, w)
    assert out[clean].isfinite().all() and (out[1] == 0).all()
    assert out[3].isnan().all() and out[4, 7].isnan()
    for group in (0, 128):
        q, scale = norm.run_fp8(x, w, group_size=group)
        assert q[clean].float().isfinite().all() and scale[clean].isfinite().all()
        assert (scale[1] == 1).all() and (q[1].float() == 0).all()
        assert q[3].float().isnan().all() and scale[3].isnan().all()
        assert (scale[4, 0] if group else scale[4]).isnan()
    # a weight of zero in a whole group: scale 1, zeros
    w[128:] = 0
    q, scale = norm.run_fp8(x[:1], w, group_size=128)
    assert scale[0, 1] == 1 and (q[0, 128:].float() == 0).all() and scale[0, 0] != 1


def test_no_rows_and_many_rows():
    from gdn_b200 import norm
    w = torch.ones(128, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(0, 128, device="cuda").to(torch.bfloat16)
    assert norm.run(x, w).shape == (0, 128)
    out, new = norm.run(x, w, residual=x)
    assert new.shape == (0, 128)
    q, s, new = norm.run_fp8(x, w, residual=x)
    assert q.shape == (0, 128) and s.shape == (0,)
    x = torch.randn(70001, 128, device="cuda").to(torch.bfloat16)
    y, _ = L.norm_ref(x, w, 1e-6)
    L.within(norm.run(x, w), y, slack(y, 128))


def test_refusals():
    from gdn_b200 import norm
    x, w, res, gate = make(4, 256, torch.bfloat16)
    for exc, match, args, kw in [
            (TypeError, "bfloat16 or float16", (x.float(), w), {}),
            (TypeError, "residual", (x, w), dict(residual=res.half())),
            (ValueError, "multiple of 8", (x[:, :250], w), {}),
            (ValueError, "weight", (x, w[:128]), {}),
            (ValueError, "shape", (x, w), dict(gate=gate[:3])),
            (ValueError, "both", (x, w), dict(residual=res, gate=gate)),
            (ValueError, "residual_out", (x, w), dict(residual_out=res)),
            (ValueError, "contiguous", (x.t().contiguous().t(), w), {}),
            (ValueError, "overlaps", (x, w), dict(residual=torch.zeros(5, 256, dtype=x.dtype, device="cuda")[1:],
                                                  residual_out="shifted"))]:
        if kw.get("residual_out") == "shifted":
            base = torch.zeros(5, 256, dtype=x.dtype, device="cuda")
            kw = dict(residual=base[1:], residual_out=base[:4])
        with pytest.raises(exc, match=match):
            norm.run(*args, **kw)
    with pytest.raises(ValueError, match="group_size"):
        norm.run_fp8(x[:, :136].contiguous(), w[:136].contiguous(), group_size=128)
    with pytest.raises(ValueError, match="group_size"):
        norm.run_fp8(x, w, group_size=64)


@pytest.mark.parametrize("D", [72, 128, 1000, 4096, 8192])
def test_in_place(D):
    """The output or residual_out in the place of a contiguous input."""
    from gdn_b200 import norm
    g = torch.Generator(device="cuda").manual_seed(D)
    x, res, gate = (torch.randn(37, D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(3))
    w = torch.rand(D, generator=g, device="cuda").to(torch.bfloat16)
    want = norm.run(x, w)
    y = x.clone()
    assert norm.run(y, w, output=y).data_ptr() == y.data_ptr() and torch.equal(y, want)
    want = norm.run(x, w, gate=gate)
    y = gate.clone()
    norm.run(x, w, gate=y, output=y)
    assert torch.equal(y, want)
    want, wr = norm.run(x, w, residual=res)
    y, r = x.clone(), res.clone()
    norm.run(y, w, residual=r, output=y, residual_out=r)
    assert torch.equal(y, want) and torch.equal(r, wr)
    y, r = x.clone(), res.clone()
    norm.run(y, w, residual=r, output=r, residual_out=y)
    assert torch.equal(r, want) and torch.equal(y, wr)
