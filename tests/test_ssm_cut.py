"""Which calls of the prompt scan are cut into pieces (and so take a workspace and two launches)."""
import pytest

from gdn_b200 import ssm


@pytest.mark.parametrize("T,n,H,G,P,cut", [
    (8192, 1, 64, 8, 64, True),       # few (sequence, head tile) pairs
    (65536, 4, 64, 8, 64, True),      # whole sequences fill the SMs, but one of twice the mean would run on alone
    (16384, 128, 32, 4, 64, True),    # many sequences, one of which may hold a large part of the tokens
    (65536, 1024, 16, 2, 64, True),
    (7648, 16, 32, 16, 128, False),   # only a sequence of seven times the mean would be cut
    (7648, 16, 64, 8, 64, False),
    (16384, 16, 64, 8, 64, False),
    (1024, 64, 64, 8, 64, False)])    # token by token
def test_calls_that_are_cut(T, n, H, G, P, cut):
    assert (ssm.workspace_bytes(T, n, H, G, P, 128) > 0) == cut
