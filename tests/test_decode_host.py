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


def test_workspaces_of_one_kind_take_no_place_of_the_others(monkeypatch):
    """Eight of each kind are kept, those used last."""
    stream = [0]
    monkeypatch.setattr(decode, "_WORKSPACES", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: type("Stream", (), {"cuda_stream": stream[0]}))
    cpu = torch.device("cpu")

    def get(number, kind):
        stream[0] = number
        return decode._workspace(cpu, 5000, kind)

    held = {(i, kind): get(i, kind) for i in range(8) for kind in ("attention", "beams")}
    assert all((s[:_cabi.PAGED_COUNTER_BYTES] == 0).all() for s in held.values())
    for i, kind in held:
        assert get(i, kind) is held[i, kind]
    get(0, "attention")
    get(8, "attention")                                    # the ninth: that of stream 1 was used longest ago
    assert all(get(i, "beams") is held[i, "beams"] for i in range(8))
    assert all(get(i, "attention") is held[i, "attention"] for i in (0, 2, 3, 4, 5, 6, 7))
    assert get(1, "attention") is not held[1, "attention"] and len(decode._WORKSPACES) == 16
