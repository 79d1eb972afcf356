"""The choice among the continuations of beams, in one kernel; ``decode.paged_kv_reorder`` brings the caches behind it into order."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _cabi
from .decode import _workspace
from .prefill import _DTYPES

MAX_BEAMS, MAX_KEEP, MAX_BATCH, MAX_VOCAB = 32, 64, 1024, 1 << 30
_host = None
_addresses: tuple = ()


def beam_select(logits: torch.Tensor, scores: torch.Tensor, keep: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``keep`` best continuations of each batch entry's beams: (B * N, V) logits of bfloat16, float16 or float32, row b * N + i those of
    beam i of entry b, and (B, N) float32 ``scores`` of the beams -> scores (B, keep) float32, beams (B, keep) int32 and tokens (B, keep) int64.

    A continuation's score is its beam's plus the log-softmax of its logit.  Larger scores come first, of equal ones the lower beam, within a beam the
    larger logit, of equal ones the lower token.  ``keep`` defaults to 2 N, which leaves N continuations where each beam may end.  Beams of
    score -inf are not alive: their continuations, and tokens of logit -inf or NaN, have -inf and come where there is nothing else.
    N up to 32, ``keep`` up to 64, B up to 1024.  One kernel on the current stream, without synchronising."""
    global _host, _addresses
    if _host is None:
        lib = _cabi.load()
        _addresses = tuple(C.cast(f, C.c_void_p).value for f in (lib.pbs_beam_select, lib.pbs_beam_select_workspace))
        _host = _cabi.load_host() or False
    if _host:                                              # without Python in between (csrc/host_decode.cpp), where it can be
        done = _host.beam_select(*_addresses, logits, scores, keep)
        if done is not None:
            return done
    if not logits.is_cuda:
        raise RuntimeError("pbs_attn_b200 runs on CUDA devices only; there is no CPU path")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {logits.dtype}: need bfloat16, float16 or float32")
    if scores.dtype != torch.float32 or scores.device != logits.device:
        raise TypeError(f"scores must be a float32 tensor on {logits.device}")
    if scores.dim() != 2 or scores.stride(1) != 1 and scores.shape[1] > 1:
        raise ValueError("scores must be (B, N) with dense rows")
    B, N = scores.shape
    if logits.dim() != 2 or logits.shape[0] != B * N or logits.stride(1) != 1 and logits.shape[1] > 1:
        raise ValueError(f"logits must be (B * N, V) with dense rows, for {B} entries of {N} beams")
    keep = 2 * N if keep is None else int(keep)
    if N < 1 or keep < 1:
        raise ValueError(f"{N} beams, keep={keep}: at least one of each is needed")
    if B > MAX_BATCH or N > MAX_BEAMS or keep > MAX_KEEP or logits.shape[1] > MAX_VOCAB:
        raise _cabi.PbsError(f"beam selection: {B} entries of {N} beams of {logits.shape[1]} tokens, keep={keep}: up to {MAX_BATCH}, {MAX_BEAMS}, {MAX_VOCAB} and {MAX_KEEP}")
    out = tuple(torch.empty(B, keep, dtype=dt, device=logits.device) for dt in (torch.float32, torch.int32, torch.int64))
    if B == 0:
        return out
    a = _cabi.BeamSelect(_DTYPES[logits.dtype], B, N, logits.shape[1], keep, 0, logits.data_ptr(), logits.stride(0), scores.data_ptr(), scores.stride(0),
                         *(t.data_ptr() for t in out))
    lib = _cabi.load()
    with torch.cuda.device(logits.device):
        need = C.c_int64()
        _cabi.check(lib.pbs_beam_select_workspace(C.byref(a), C.byref(need)), "pbs_beam_select_workspace")
        space = _workspace(logits.device, need.value, "beams")
        _cabi.check(lib.pbs_beam_select(C.byref(a), C.c_void_p(space.data_ptr()), space.numel(),
                                        C.c_void_p(torch.cuda.current_stream(logits.device).cuda_stream)), "pbs_beam_select")
    return out
