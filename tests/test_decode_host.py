"""CPU-only: the host side of decode.py."""
import ctypes as C

import pytest
import torch

from pbs_attn_b200 import _cabi, decode


def test_a_wait_that_ran_out_names_the_calls_behind_it(monkeypatch):
    """Calls behind the one that gave up found its counters: their outputs are not to be trusted either."""
    monkeypatch.setattr(decode, "_WORKSPACES", {1: torch.zeros(1)})
    monkeypatch.setattr(_cabi, "load_host", lambda: None)
    word = C.c_int32(4)
    with pytest.raises(_cabi.PbsError, match="invalid, and so are those of the attention calls enqueued behind it"):
        decode._raise_fault(word)
    assert word.value == 0 and not decode._WORKSPACES


@pytest.mark.parametrize("t", [
    torch.arange(129.0, dtype=torch.bfloat16)[1:].view(1, 1, 1, 128),                                      # dense, but between the boundaries
    torch.arange(256.0, dtype=torch.bfloat16).as_strided((1, 2, 1, 128), (256, 128, 0, 1)),               # dense as its single token goes
    torch.arange(300.0, dtype=torch.bfloat16).as_strided((1, 2, 1, 128), (257, 128, 3, 1)),
    torch.arange(300.0, dtype=torch.bfloat16).as_strided((1, 1, 2, 128), (300, 7, 129, 1))])
def test_what_kernels_cannot_read_in_place_is_copied_to_where_they_can(t):
    from pbs_attn_b200.prefill import _readable
    got = _readable(t)
    assert torch.equal(got, t) and got.data_ptr() % 16 == 0 and got.stride(3) == 1 and got.stride(2) > 0
    assert not any(s * 2 % 16 for s in got.stride()[:3])
