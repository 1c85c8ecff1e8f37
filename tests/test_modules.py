"""The extension modules hold no C++ library of their own (CPU)."""
import shutil
import subprocess

import pytest

from gdn_b200 import _native as N

MODULES = ["_gdn_torch.so", "gdn_tvm_ffi.so"]


@pytest.mark.skipif(shutil.which("nm") is None, reason="needs binutils")
@pytest.mark.parametrize("name", MODULES)
def test_one_cxx_library(name):
    """std::locale's facets are looked up by objects of the C++ library: with two of them in a process, a number that is
    inserted into one's stream is formatted by the other's, and the process ends."""
    path = N.LIB_PATH.parent / name
    names = subprocess.run(["nm", "-D", "--defined-only", str(path)], capture_output=True, text=True, check=True).stdout
    assert "_ZNSt6localeC1Ev" not in names and "_ZNSt7num_put" not in names


@pytest.mark.gpu
def test_messages_with_numbers():
    """A refusal whose message holds a number, through the torch module."""
    import torch
    from gdn_b200 import conv
    assert N.torch_ext() is not None
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    with pytest.raises(ValueError, match="x must be a 2D tensor"):
        conv.run(z(1, 4, 64), z(64, 4), None, None, torch.tensor([0, 4], device="cuda"))
