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
