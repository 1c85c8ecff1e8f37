"""silu of the short convolution over its whole range (GPU)."""
import pytest
import torch

import layer_oracle as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("form", ["prompt", "one token", "tokens"])
def test_silu_from_the_smallest_to_the_largest_sums(form, dtype):
    """The only tap with a weight is the current token's, so that the sum is x itself.  silu x = x / (1 + e^-x) down to
    the type's smallest values: the exponent is off by half a step of fp32 at 128 (2^-18), which e^x shows as such,
    and the exponential, the reciprocal and the products by 2^-21."""
    from gdn_b200 import conv
    T, D = 64, 256
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.linspace(-120, 100, T * D, device="cuda")[torch.randperm(T * D, generator=g, device="cuda")].view(T, D).to(dtype)
    w = torch.zeros(D, 4, device="cuda", dtype=dtype)
    w[:, 3] = 1
    if form == "prompt":
        out, _ = conv.run(x, w, None, None, torch.tensor([0, T], device="cuda"))
    else:
        xs = x.view(T, 1, D) if form == "one token" else x.view(T // 4, 4, D)
        pool = torch.zeros(xs.shape[0], 3, D, device="cuda", dtype=dtype)
        out = conv.run_pool(xs, w, None, pool, torch.arange(xs.shape[0], dtype=torch.int32, device="cuda")).view(T, D)
    v = L.d(x)
    ref = v / (1 + torch.exp(-v))
    L.within(out, ref, 2.0 ** -17 * ref.abs())
    if dtype is torch.bfloat16:
        assert (out[(x < -42) & (x > -80)] < 0).all()
