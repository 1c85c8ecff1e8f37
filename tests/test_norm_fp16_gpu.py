"""The norm's gates and 8-bit outputs from fp16 (GPU); its other tests hold the same kernels to bf16."""
import pytest
import torch

import layer_oracle as L
from test_norm_gpu import make, slack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("D", [64, 128, 136, 1000, 4096, 8192])
def test_gate(D, first):
    from gdn_b200 import norm
    x, w, _, gate = make(33, D, torch.float16, D)
    y, _ = L.norm_ref(x, w, 1e-6, gate=gate, gate_first=first)
    # silu's 2^x sees its argument rounded: |gate| 2^-23, with |gate| < 8
    L.within(norm.run(x, w, 1e-6, gate=gate, gate_first=first), y, slack(y, D) + 2.0 ** -20 * y.abs())


@pytest.mark.parametrize("mode", ["plain", "residual", "after", "before"])
@pytest.mark.parametrize("D,group", [(8, 0), (128, 128), (200, 0), (1152, 128), (4096, 0), (4096, 128), (16384, 128)])
def test_e4m3(D, group, mode):
    from gdn_b200 import norm
    rows = 11
    x, w, res, gate = make(rows, D, torch.float16, D + group)
    kw = dict(residual=res) if mode == "residual" else dict(gate=gate, gate_first=mode == "before") \
        if mode != "plain" else {}
    y, h = L.norm_ref(x, w, 1e-6, **kw)
    out = norm.run_fp8(x, w, 1e-6, group_size=group, **kw)
    q, scale = out[0], out[1]
    assert q.dtype == torch.float8_e4m3fn and scale.shape == ((rows, D // group) if group else (rows,))
    blocks = y.view(rows, D // group if group else 1, -1)
    want = blocks.abs().amax(-1) / 448
    # fp32: squares and additions under a root, a handful of products, and silu's rounded argument
    rel = (D / 2 + 96) * 2.0 ** -24 + 2.0 ** -20
    assert ((L.d(scale).view(rows, -1) - want).abs() <= rel * want).all()
    # the quotient is off by `rel`, then rounded: half a step is 2^-4 relative, or 2^-10 below the normal range
    quo = blocks / want[..., None]
    got = q.float().cpu().double().view_as(quo)
    assert ((got - quo).abs() <= 2.0 ** -4 * quo.abs() * (1 + 4 * rel) + 2.0 ** -10 + 4 * rel * quo.abs()).all()
    if mode == "residual":
        L.within(out[2], h, 2.0 ** -24 * h.abs())
