"""Penalties for repeated tokens, biases and a grammar mask on the logits of a decoding step, in one kernel."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Union

import torch

from . import _cabi
from .prefill import _DTYPES

Penalty = Optional[Union[float, torch.Tensor]]
_host = _address = None


def process_logits(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, token_lens: Optional[torch.Tensor] = None,
                   prompt_lens: Optional[torch.Tensor] = None, repetition_penalty: Penalty = None, frequency_penalty: Penalty = None,
                   presence_penalty: Penalty = None, bias_ids: Optional[torch.Tensor] = None, bias_values: Optional[torch.Tensor] = None,
                   allowed: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(B, V) logits of bfloat16, float16 or float32 -> a new tensor (or ``out``, which may be ``logits``) after, in this order,

      * ``repetition_penalty`` r: x / r where x > 0, else x * r, for every token of the row's history;
      * ``frequency_penalty`` f and ``presence_penalty`` p: x - f * c, then x - p, for tokens that the history holds c > 0 times
        behind the prompt;
      * biases: ``bias_values`` (B, n) float32 added at ``bias_ids`` (B, n) (those of an id that is listed twice add up);
      * ``allowed`` (B or 1, ceil(V / 32)) int32: -inf where bit v % 32 of word v // 32 is 0.

    The history of row b is ``tokens[b, :token_lens[b]]``, the first ``prompt_lens[b]`` of it the prompt (without the lengths: the
    whole row, no prompt; lengths that the row does not have are taken as the nearest that it has).  ``tokens`` and ``bias_ids`` are
    int32 or int64; ids outside 0 .. V - 1 are skipped.  Penalties are numbers or (B,) float32 tensors.  All in 32 bits, rounded
    once.  Made for some hundreds of biases a row; thousands work, slowly.  Runs on the current stream without synchronising;
    tokens are counted anew in every call, so nothing has to be kept in step when rows move, leave or take back tokens."""
    global _host, _address
    if _host is None:
        _host, _address = _cabi.load_host() or False, C.cast(_cabi.load().pbs_process_logits, C.c_void_p).value
    if _host:                                              # without Python in between (csrc/host_decode.cpp), where it can be
        done = _host.process_logits(_address, logits, tokens, token_lens, prompt_lens, repetition_penalty, frequency_penalty, presence_penalty,
                                    bias_ids, bias_values, allowed, out)
        if done is not None:
            return done
    if not logits.is_cuda:
        raise RuntimeError("pbs_attn_b200 runs on CUDA devices only; there is no CPU path")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {logits.dtype}: need bfloat16, float16 or float32")
    if logits.dim() != 2 or logits.stride(1) != 1 and logits.shape[1] > 1:
        raise ValueError("logits must be (B, V) with dense rows")
    B, V = logits.shape
    if out is None:
        out = torch.empty(B, V, dtype=logits.dtype, device=logits.device)
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device or out.stride(1) != 1 and V > 1:
        raise ValueError("out must have the shape, dtype and device of logits, and dense rows")
    if logits.numel() == 0:
        return out

    def take(name, t, shape, dtypes):
        if t is None:
            return None
        if t.device != logits.device or t.dtype not in dtypes:
            raise TypeError(f"{name} must be {' or '.join(str(d)[6:] for d in dtypes)} on {logits.device}")
        if t.dim() != len(shape) or any(s is not None and t.shape[i] not in s for i, s in enumerate(shape)) or t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} has shape {tuple(t.shape)} and strides {t.stride()}: does not fit logits of {B} x {V}, or its rows are not dense")
        return t.data_ptr()

    a = _cabi.Logits(dtype=_DTYPES[logits.dtype], rows=B, vocab=V, logits=logits.data_ptr(), out=out.data_ptr(),
                     logits_stride=logits.stride(0), out_stride=out.stride(0))
    ints = (torch.int32, torch.int64)
    a.tokens = take("tokens", tokens, ((B,), None), ints)
    if tokens is not None:
        a.history, a.tokens_stride, a.token_bytes = tokens.shape[1], tokens.stride(0), tokens.element_size()
    a.token_lens = take("token_lens", token_lens, ((B,),), ints[:1])
    a.prompt_lens = take("prompt_lens", prompt_lens, ((B,),), ints[:1])
    for name, p, none in (("repetition", repetition_penalty, 1.0), ("frequency", frequency_penalty, 0.0), ("presence", presence_penalty, 0.0)):
        if isinstance(p, torch.Tensor):
            setattr(a, name, take(name + "_penalty", p, ((B,),), (torch.float32,)))
        p = none if p is None or isinstance(p, torch.Tensor) else float(p)
        if name == "repetition" and not p > 0:
            raise ValueError(f"repetition_penalty={p}: must be above 0")
        setattr(a, name + "_all", p)
    if tokens is None and any(p is not None for p in (repetition_penalty, frequency_penalty, presence_penalty)):
        raise ValueError("penalties need the tokens that they are for")
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("bias_ids and bias_values come together")
    a.bias_ids = take("bias_ids", bias_ids, ((B,), None), ints)
    if bias_ids is not None:
        a.bias_values = take("bias_values", bias_values, ((B,), (bias_ids.shape[1],)), (torch.float32,))
        a.biases, a.bias_id_bytes = bias_ids.shape[1], bias_ids.element_size()
        a.bias_ids_stride, a.bias_values_stride = bias_ids.stride(0), bias_values.stride(0)
    a.allowed = take("allowed", allowed, ((1, B), (-(-V // 32),)), ints[:1])
    if allowed is not None:
        a.allowed_stride = allowed.stride(0) if allowed.shape[0] > 1 else 0
    with torch.cuda.device(logits.device):
        _cabi.check(_cabi.load().pbs_process_logits(C.byref(a), C.c_void_p(torch.cuda.current_stream(logits.device).cuda_stream)), "pbs_process_logits")
    return out
