"""Refusals of the convolution, scan and norm entry points at the C ABI, before anything
touches the GPU (CPU)."""
import ctypes

import pytest
import torch

from gdn_b200 import _native as N

P = ctypes.c_void_p
BASE = 1 << 20


def call(fn, args, over):
    names = list(args)
    vals = {**args, **over}
    return getattr(N.lib(), fn)(*[P(v) if isinstance(v, int) and n.startswith("p_") else v
                                  for n, v in ((n, vals[n]) for n in names)])


def rejects(fn, args, over, msg, code=N.GDN_ERR_VALUE):
    assert call(fn, args, over) == code
    assert msg in N.lib().gdn_last_error().decode()


def arr(t, *v):
    return (t * len(v))(*v)


CONV = dict(p_x=BASE, xs=64, p_w=BASE, p_b=BASE, p_st=BASE, p_cu=BASE, outs=arr(P, BASE), widths=arr(ctypes.c_int64, 64),
            n=1, p_new=1 << 24, T=10, N=1, D=64, W=4, dt=0, flags=1, p_stream=0)
CONV_POOL = dict(p_x=BASE, xb=64, xs=64, p_w=BASE, p_b=BASE, p_pool=BASE, pool=4, p_in=BASE, p_out=0, outs=arr(P, BASE),
                 widths=arr(ctypes.c_int64, 64), n=1, B=2, T=1, D=64, W=4, dt=0, flags=1, p_stream=0)
SSM = dict(p_x=BASE, p_B=BASE, p_C=BASE, p_st=BASE, p_A=BASE, p_a=BASE, p_dt=BASE, p_D=BASE, p_cu=BASE, p_y=BASE,
           p_new=1 << 26, T=10, N=1, H=4, G=2, Pd=64, Ns=128, p_ws=0, ws=0, p_stream=0)
SSM_POOL = dict(p_x=BASE, p_B=BASE, p_C=BASE, p_A=BASE, p_a=BASE, p_dt=BASE, p_D=BASE, p_pool=BASE, sdt=0, pool=4,
                p_in=BASE, p_out=0, flags=0, p_y=BASE, B=2, T=1, H=4, G=2, Pd=64, Ns=128, p_stream=0)
NORM = dict(p_x=BASE, xs=256, p_w=BASE, p_res=BASE, rs=256, p_gate=0, gs=256, eps=1e-6, p_out=1 << 22, p_scale=0, group=0,
            p_ro=1 << 23, rows=4, D=256, dt=0, flags=0, p_stream=0)


@pytest.mark.parametrize("over,msg", [
    (dict(W=1), "width"), (dict(W=5), "width"), (dict(D=60), "multiple of 8"), (dict(T=-1), "non-negative"),
    (dict(N=0), "at least one sequence"), (dict(flags=2), "flags"), (dict(n=0), "num_outputs"),
    (dict(n=5), "num_outputs"), (dict(p_w=0), "null"), (dict(xs=56), "strides"), (dict(xs=68), "strides"),
    (dict(p_x=BASE + 8), "aligned"), (dict(widths=arr(ctypes.c_int64, 56)), "sum"),
    (dict(widths=arr(ctypes.c_int64, 60)), "multiples of 8"), (dict(outs=arr(P, 0)), "output 0"),
    (dict(outs=arr(P, BASE + 4)), "output 0"), (dict(p_cu=0), "null"), (dict(p_new=BASE + 64), "overlaps"),
    (dict(p_new=BASE), "overlaps")])
def test_conv(over, msg):
    rejects("gdn_conv", CONV, over, msg)


@pytest.mark.parametrize("over,msg", [
    (dict(T=0), "seq_len"), (dict(B=-1), "non-negative"), (dict(pool=-1), "pool_size"), (dict(pool=1 << 31), "pool_size"),
    (dict(p_in=0), "null"), (dict(p_pool=0), "null"), (dict(p_pool=BASE + 8), "aligned"), (dict(p_out=BASE + 2), "aligned"),
    (dict(xb=4), "strides")])
def test_conv_pool(over, msg):
    rejects("gdn_conv_pool", CONV_POOL, over, msg)


@pytest.mark.parametrize("over,msg", [
    (dict(N=0), "at least one"), (dict(T=-1), "non-negative"), (dict(H=3), "multiple"), (dict(H=0), "multiple"),
    (dict(G=0), "multiple"), (dict(Pd=32), "head_dim"), (dict(Ns=256), "state_dim"), (dict(p_x=0), "null"),
    (dict(p_A=0), "null"), (dict(p_cu=0), "null"), (dict(p_B=BASE + 8), "aligned"), (dict(p_new=BASE + 1024), "overlaps"),
    (dict(p_new=BASE), "overlaps"), (dict(T=1 << 31), "too large")])
def test_ssm(over, msg):
    rejects("gdn_ssm", SSM, over, msg)


@pytest.mark.parametrize("over,msg", [
    (dict(T=0), "seq_len"), (dict(B=-1), "non-negative"), (dict(flags=1), "flags"), (dict(pool=1 << 31), "pool_size"),
    (dict(p_in=0), "null"), (dict(p_pool=BASE + 4), "aligned"), (dict(p_in=BASE + 2), "aligned")])
def test_ssm_pool(over, msg):
    rejects("gdn_ssm_pool", SSM_POOL, over, msg)


@pytest.mark.parametrize("over,msg", [
    (dict(D=252), "multiple of 8"), (dict(D=16392), "up to 16384"), (dict(rows=-1), "non-negative"), (dict(flags=2), "flags"),
    (dict(group=64, p_scale=BASE), "group_size"), (dict(group=128), "scale"), (dict(p_gate=BASE), "both"),
    (dict(p_ro=0), "residual_out"), (dict(p_res=0), "residual_out"), (dict(p_x=0), "null"), (dict(p_x=BASE + 2), "aligned"),
    (dict(xs=248), "strides"), (dict(rs=260), "strides"), (dict(p_ro=BASE + 512), "overlaps"),
    (dict(p_ro=BASE, rs=264), "overlaps")])
def test_rms_norm(over, msg):
    rejects("gdn_rms_norm", NORM, over, msg)


def test_types():
    rejects("gdn_conv", CONV, dict(dt=2), "dtype", N.GDN_ERR_TYPE)
    rejects("gdn_ssm_pool", SSM_POOL, dict(sdt=2), "state_dtype", N.GDN_ERR_TYPE)
    rejects("gdn_rms_norm", NORM, dict(dt=-1), "dtype", N.GDN_ERR_TYPE)


def test_nothing_to_do():
    assert call("gdn_conv_pool", CONV_POOL, dict(B=0, p_x=0)) == N.GDN_OK
    assert call("gdn_ssm_pool", SSM_POOL, dict(B=0, p_x=0)) == N.GDN_OK
    assert call("gdn_rms_norm", NORM, dict(rows=0, p_x=0)) == N.GDN_OK


@pytest.mark.parametrize("with_ext", [True, False])
def test_python_entry_points_reject_cpu_tensors(with_ext, monkeypatch):
    from gdn_b200 import conv, norm, ssm
    if not with_ext:
        monkeypatch.setattr(N, "_ext", None)
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    cu, slots = torch.tensor([0, 4]), torch.zeros(4, dtype=torch.int32)
    f = z(2, dt=torch.float32)
    for fn, args in ((conv.run, (z(4, 64), z(64, 4), None, None, cu)),
                     (conv.run_pool, (z(4, 1, 64), z(64, 4), None, z(4, 3, 64), slots)),
                     (norm.run, (z(4, 64), z(64))), (norm.run_fp8, (z(4, 64), z(64))),
                     (ssm.run, (z(4, 2, 64), z(4, 1, 64), z(4, 1, 64), None, f, z(4, 2), f, f, cu)),
                     (ssm.run_pool, (z(4, 1, 2, 64), z(4, 1, 1, 64), z(4, 1, 1, 64), f, z(4, 1, 2), f, f,
                                     z(4, 2, 64, 64, dt=torch.float32), slots))):
        with pytest.raises(ValueError, match="CUDA"):
            fn(*args)


@pytest.mark.parametrize("fn,args,over", [
    ("gdn_conv", CONV, {}),  # (the output is x)
    ("gdn_conv", CONV, dict(outs=arr(P, BASE + 2 * 64 * 9))),
    ("gdn_conv", CONV, dict(xs=640, outs=arr(P, BASE + 2 * 128))),  # between the rows of x
    ("gdn_conv", CONV, dict(outs=arr(P, 1 << 24))),  # new_state
    ("gdn_conv", CONV, dict(outs=arr(P, 1 << 22, (1 << 22) + 640 - 16), widths=arr(ctypes.c_int64, 32, 32), n=2)),
    ("gdn_conv_pool", CONV_POOL, dict(p_pool=1 << 24)),  # (the output is x)
    ("gdn_conv_pool", CONV_POOL, dict(p_x=1 << 24)),  # (the output is the pool)
    ("gdn_conv_pool", CONV_POOL, dict(p_x=1 << 24, p_pool=1 << 26, p_w=BASE + 128)),
    ("gdn_ssm", SSM, {}),
    ("gdn_ssm", SSM, dict(p_y=BASE + 10 * 4 * 64 * 2 - 16)),
    ("gdn_ssm", SSM, dict(p_y=(1 << 26) + 1024)),
    ("gdn_ssm", SSM, dict(p_y=1 << 25, p_C=(1 << 25) - 16)),
    ("gdn_ssm_pool", SSM_POOL, dict(p_pool=1 << 24)),
    ("gdn_ssm_pool", SSM_POOL, dict(p_y=1 << 24, p_pool=1 << 24)),
    ("gdn_rms_norm", NORM, dict(p_out=BASE, xs=264)),
    ("gdn_rms_norm", NORM, dict(p_out=BASE + 512)),
    ("gdn_rms_norm", NORM, dict(p_out=BASE, p_scale=1 << 25)),
    ("gdn_rms_norm", NORM, dict(p_out=(1 << 23) + 512)),
    ("gdn_rms_norm", NORM, dict(p_x=1 << 24, p_ro=(1 << 24) + 512)),
    ("gdn_rms_norm", NORM, dict(p_res=0, p_ro=0, p_gate=1 << 24, p_out=(1 << 24) + 16))])
def test_outputs_that_overlap(fn, args, over):
    rejects(fn, args, over, "overlaps")


def test_sizes_past_any_tensor():
    rejects("gdn_ssm", SSM, dict(H=1 << 57, G=1), "65536")
    rejects("gdn_ssm_pool", SSM_POOL, dict(H=1 << 57, G=1), "65536")
    assert N.lib().gdn_ssm_workspace_bytes(*[ctypes.c_int64(v) for v in (1 << 62, 1, 64, 1, 64, 128)]) == 0
    assert N.lib().gdn_ssm_workspace_bytes(*[ctypes.c_int64(v) for v in (1 << 20, 1, 1 << 57, 1, 64, 128)]) == 0
