"""The norm's 8-bit output against its formula in fp32, bit by bit (GPU).

Every eight values of the rows are integers whose squares sum to 512, so the root mean square is 8 exactly, in any order
of summation: h / 8 * weight is one rounding, max |y| / 448 and y / scale one each, and nothing is left to a
tolerance."""
import pytest
import torch

pytestmark = pytest.mark.gpu
EIGHTS = [[20, 8, 6, 2, 2, 2, 0, 0], [17, 13, 7, 2, 1, 0, 0, 0], [15, 11, 9, 7, 5, 3, 1, 1], [12, 12, 10, 8, 6, 4, 2, 2],
          [19, 11, 5, 2, 1, 0, 0, 0], [14, 14, 10, 4, 2, 0, 0, 0], [8, 8, 8, 8, 8, 8, 8, 8], [22, 4, 2, 2, 2, 0, 0, 0]]


def rows_of(rows, D, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    assert all(sum(v * v for v in e) == 512 for e in EIGHTS)
    e = torch.tensor(EIGHTS, device="cuda")[torch.randint(0, len(EIGHTS), (rows, D // 8), generator=g, device="cuda")].view(rows, D)
    e = e.gather(1, torch.rand(rows, D, generator=g, device="cuda").argsort(1))
    return torch.where(torch.rand(rows, D, generator=g, device="cuda") < 0.5, -e, e).float()


def formula(h, w, group):
    """(q, scale) of fp32 rows h of root mean square 8, on the CPU."""
    y = h.cpu() / 8 * w.cpu().float()
    blocks = y.reshape(y.shape[0], y.shape[1] // group if group else 1, -1)
    scale = blocks.abs().amax(-1) / torch.full((), 448.0)
    scale = torch.where(scale == 0, 1.0, scale)
    q = (blocks / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).reshape(y.shape)
    return q, scale if group else scale[:, 0]


def same(got, want):
    g, w = got.cpu().float(), want.float()
    return bool(((g == w) | (g.isnan() & w.isnan())).all())


@pytest.mark.parametrize("D,group", [(64, 0), (256, 128), (1024, 0), (2048, 128), (4096, 0), (4096, 128), (16384, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_e4m3_is_the_formula(D, group, dtype):
    from gdn_b200 import norm
    rows = (1 << 22) // D
    g = torch.Generator(device="cuda").manual_seed(D)
    w = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(dtype)
    h = rows_of(rows, D, D + 1)
    q2, scale2 = formula(h, w, group)
    q, scale = norm.run_fp8(h.to(dtype), w, 0.0, group_size=group)
    assert torch.equal(scale.cpu(), scale2) and same(q, q2)
    res = (h / 2).round().to(dtype)  # (halves of integers below 64: exact)
    q, scale, new = norm.run_fp8((h - res.float()).to(dtype), w, 0.0, residual=res, group_size=group)
    assert torch.equal(new.float(), h) and torch.equal(scale.cpu(), scale2) and same(q, q2)


@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("power", [-90, -99, -100, -101, -118, -126, -133, 100, 127])
def test_e4m3_of_tiny_and_huge_rows(power, group):
    """Scales down to fp32's smallest values, and one that is infinite (finite values are 0 then, infinite ones NaN)."""
    from gdn_b200 import norm
    D = 1024
    h = rows_of(40, D, 3)
    w = torch.full((D,), 2.0 ** power, device="cuda").to(torch.bfloat16)
    w[::3] *= 1.5
    q, scale = norm.run_fp8(h.to(torch.bfloat16), w, 0.0, group_size=group)
    q2, scale2 = formula(h, w, group)
    assert torch.equal(scale.cpu(), scale2) and same(q, q2)
    assert power != 127 or scale.isinf().any()
