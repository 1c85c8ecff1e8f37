"""Overlaps that the norm and the scan refuse at the C ABI, before anything touches the GPU (CPU)."""
import ctypes

import pytest

from gdn_b200 import _native as N

P, I64 = ctypes.c_void_p, ctypes.c_int64
MB = 1 << 20
ROWS, D = 4, 256


def norm(x=1 * MB, w=2 * MB, res=None, gate=None, out=3 * MB, scale=None, group=0, res_out=None):
    rc = N.lib().gdn_rms_norm(P(x), I64(D), P(w), P(res), I64(D), P(gate), I64(D), ctypes.c_float(1e-6), P(out), P(scale),
                              I64(group), P(res_out), I64(ROWS), I64(D), 0, 0, P(0))
    return rc, N.lib().gdn_last_error().decode()


@pytest.mark.parametrize("kw", [
    dict(out=2 * MB),                                        # output over the weight
    dict(out=2 * MB - ROWS * D * 2 + 16),
    dict(res=4 * MB, res_out=2 * MB - 16),                   # residual_out over the weight
    dict(scale=2 * MB + D * 2 - 4),                          # scales over the weight
    dict(scale=2 * MB - 4 * ROWS + 4),
    dict(scale=1 * MB + 8),                                  # ... over x
    dict(res=4 * MB, res_out=5 * MB, scale=4 * MB + ROWS * D * 2 - 4),
    dict(gate=4 * MB, scale=4 * MB),
    dict(scale=3 * MB + ROWS * D - 4),                       # ... over the e4m3 output
    dict(scale=3 * MB - 4 * ROWS * (D // 128) + 4, group=128),
    dict(res=4 * MB, res_out=5 * MB, scale=5 * MB + 4)])
def test_norm(kw):
    rc, msg = norm(**kw)
    assert rc == N.GDN_ERR_VALUE and "overlaps" in msg


@pytest.mark.parametrize("ws", [1 * MB + 256, 6 * MB, 6 * MB + 2000 * 256 - 256, 8 * MB - 256])
def test_scan_workspace(ws):
    """A call in two launches: its pieces' states over x, the output, the new states."""
    T, n, H, G, Pd, Ns = 2000, 1, 2, 1, 64, 128
    L = N.lib()
    need = L.gdn_ssm_workspace_bytes(*map(I64, (T, n, H, G, Pd, Ns)))
    assert need > 0
    x, B, C, st, A, a, dtb, y, new, cu = (P(v) for v in (1 * MB, 3 * MB, 4 * MB, None, 90 * MB, 91 * MB, 92 * MB, 6 * MB, 8 * MB,
                                                        93 * MB))
    rc = L.gdn_ssm(x, B, C, st, A, a, dtb, P(None), cu, y, new, *map(I64, (T, n, H, G, Pd, Ns)), P(ws), ctypes.c_size_t(need),
                   P(0))
    assert rc == N.GDN_ERR_VALUE and "overlaps" in L.gdn_last_error().decode()
