"""What follows a prompt: a paged cache of keys and values in 16 or 4 bits, and the attention of new tokens over it.

    cache = PagedKVCache(num_pages, page_size, kv_heads, head_dim, torch.bfloat16, "cuda", bits=4)     # one per layer
    q = paged_kv_append(cache, k, v, block_table, seq_lens, cos=cos, sin=sin, query_states=q)
    o = paged_attn_fwd(q, cache, block_table, seq_lens)

``block_table`` (B, pages) int32 names the pages of each sequence, ``seq_lens`` (B,) int32 counts its tokens, those of the call
among them: token i of the S new ones of sequence b is at position ``seq_lens[b] - S + i`` (with ``new_lens``, (B,) int32, the
first ``new_lens[b]`` rows are new tokens and the others padding).  Both live on the device and are read there, so a step can be
captured into a CUDA graph and replayed while they change.  The reference has no counterpart: it hands single tokens to the
model's own forward (pbs_attn/patch/huggingface.py:182-192).

A page number outside the pool, a sequence that is longer than its row of the table and a position behind the rotary tables
are found on the device: the tokens concerned are left out, and the next call on that device, or ``check_status``, raises.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _cabi
from .prefill import _ptr, _readable, _strides

_DTYPES = {torch.bfloat16: _cabi.BF16, torch.float16: _cabi.FP16}
_FAULTS = {1: "a page number in block_table is outside the pool", 2: "a sequence is longer than its row of block_table",
           3: "a position is behind the rotary tables"}
_TIMEOUT = 4

# One word a device that kernels report a fault in: pinned host memory, looked at without a copy, and never given back, since a kernel
# may still be on its way when the cache it works on is gone.
_STATUS: dict = {}
_ADDRESSES: list = []                   # of the library's functions, as the native calls take them


def _status_word(device: torch.device) -> C.c_int32:
    word = _STATUS.get(device.index)
    if word is None:
        with torch.cuda.device(device):
            ring = torch.zeros(1, dtype=torch.int32).pin_memory()
        word = C.c_int32.from_address(ring.data_ptr())
        word._keep = ring
        _STATUS[device.index] = word
    return word


def _raise_fault(word: C.c_int32):
    code, word.value = word.value, 0
    if code == _TIMEOUT:                                   # what the blocks meet at is out of step
        _WORKSPACES.clear()
        host = _cabi.load_host()
        if host is not None:
            host.paged_forget()
        raise _cabi.PbsError("paged attention: a bounded wait ran out in an earlier call on this device; its output is invalid, and "
                             "so are those of the attention calls enqueued behind it up to now")
    raise _cabi.PbsError(f"paged cache: {_FAULTS.get(code, code)} (in an earlier call on this device, which left the tokens concerned out)")


class PagedKVCache:
    """Pages of keys and values of one layer.

    ``k`` and ``v`` are (num_pages, kv_heads, page_size, head_dim) of ``dtype`` for 16 bits and (..., head_dim / 2) uint8 for 4
    (channel 2i in the low half of byte i); with 4 bits ``k_params`` and ``v_params``, (num_pages, kv_heads, page_size,
    head_dim / group_size, 2) of ``dtype``, hold step and minimum of each group of channels of a token: a code c stands for
    minimum + c * step.  ``page_size`` is a power of two from 16 to 1024, ``head_dim`` 64, 128 or 256, ``group_size`` 32 or 64.
    New pages hold whatever the memory held: no token is read that was not appended.
    """

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 device="cuda", bits: int = 16, group_size: int = 64):
        if bits not in (4, 16):
            raise ValueError(f"bits={bits}: a cache holds 16 or 4 bits a value")
        make = lambda *s, dt=dtype: torch.empty(num_pages, kv_heads, page_size, *s, dtype=dt, device=device)  # noqa: E731
        if bits == 16:
            self._set(make(head_dim), make(head_dim), None, None)
        else:
            if head_dim % group_size:
                raise ValueError(f"group_size={group_size} does not divide head_dim={head_dim}")
            self._set(*(make(head_dim // 2, dt=torch.uint8) for _ in "kv"), *(make(head_dim // group_size, 2) for _ in "kv"))

    @classmethod
    def from_tensors(cls, k, v, k_params=None, v_params=None) -> "PagedKVCache":
        """A cache over tensors that exist, of any strides that the kernels can read (a token's row dense, rows on 16-byte boundaries)."""
        self = object.__new__(cls)
        self._set(k, v, k_params, v_params)
        return self

    def _set(self, k, v, k_params, v_params):
        self.lib = _cabi.load()
        self.bits = 4 if k.dtype == torch.uint8 else 16
        pages, heads, page_size, row = k.shape
        if self.bits == 4 and (k_params is None or v_params is None):
            raise ValueError("pages of 4 bits need k_params and v_params")
        self.dtype = k.dtype if self.bits == 16 else k_params.dtype
        if self.dtype not in _DTYPES:
            raise TypeError(f"unsupported dtype {self.dtype}: need bfloat16 or float16")
        if not k.is_cuda:
            raise RuntimeError("pbs_attn_b200 runs on CUDA devices only; there is no CPU path")
        if v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
            raise ValueError("k and v pages must have one shape, dtype and device")
        self.head_dim = row * 16 // self.bits if self.bits == 16 else 2 * row
        self.group_size = 0
        if self.bits == 4:
            if (k_params.dim() != 5 or k_params.shape[:3] != k.shape[:3] or k_params.shape[4] != 2 or v_params.shape != k_params.shape
                    or v_params.dtype != k_params.dtype or self.head_dim % k_params.shape[3] or k_params.device != k.device
                    or v_params.device != k.device):
                raise ValueError("k_params and v_params must be (pages, heads, page_size, head_dim / group_size, 2)")
            self.group_size = self.head_dim // k_params.shape[3]
        elif k_params is not None or v_params is not None:
            raise ValueError("pages of 16 bits have no params")
        for t in (k, v):
            if t.stride(3) != 1:
                raise ValueError("a token's row must be dense")
        for t in (k_params, v_params) if self.bits == 4 else ():
            if t.stride(4) != 1 or t.stride(3) != 2 and t.shape[3] > 1:
                raise ValueError("a token's row of params must be dense")
        self.k, self.v, self.k_params, self.v_params = k, v, k_params, v_params
        self.num_pages, self.kv_heads, self.page_size, self.device = pages, heads, page_size, k.device
        three = lambda t: (C.c_int64 * 3)(*(t.stride()[:3] if t is not None else (0, 0, 0)))  # noqa: E731
        self._word = _status_word(self.device)
        self._c = _cabi.PagedCache(k.data_ptr(), v.data_ptr(), k_params.data_ptr() if self.bits == 4 else None,
                                   v_params.data_ptr() if self.bits == 4 else None, three(k), three(v), three(k_params), three(v_params),
                                   pages, page_size, heads, self.head_dim, _DTYPES[self.dtype], self.bits, self.group_size, 0,
                                   C.addressof(self._word))
        # what the sizes alone decide is refused here, not at the first call
        bytes_ = C.c_int64()
        probe = _cabi.PagedBatch(16, 1, 16, None, 1, 1, 1, 0)
        _cabi.check(self.lib.pbs_paged_attn_workspace(C.byref(self._c), C.byref(probe), heads, C.byref(bytes_)), "paged cache")
        # the common calls without Python (csrc/host_decode.cpp); None where that was not built
        self._host, self._native = _cabi.load_host(), None
        if self._host is not None:
            if not _ADDRESSES:
                _ADDRESSES.extend(C.cast(getattr(self.lib, "pbs_paged_" + f), C.c_void_p).value for f in ("append", "gather", "attn", "attn_workspace"))
            self._native = self._host.paged_attach(C.addressof(self._c), self.device.index, *_ADDRESSES)

    def check_status(self):
        """Synchronises and raises if a call on this device met a fault (see the module)."""
        torch.cuda.synchronize(self.device)
        if self._word.value:
            _raise_fault(self._word)


def _batch(cache: PagedKVCache, B: int, S: int, block_table, seq_lens, new_lens) -> _cabi.PagedBatch:
    if cache._word.value:
        _raise_fault(cache._word)
    for name, t, dims in (("block_table", block_table, 2), ("seq_lens", seq_lens, 1), ("new_lens", new_lens, 1)):
        if t is None and name == "new_lens":
            continue
        if t.dtype != torch.int32 or t.device != cache.device:
            raise TypeError(f"{name} must be an int32 tensor on {cache.device}")
        if t.dim() != dims or t.shape[0] != B or t.stride(-1) != 1 and t.shape[-1] > 1:
            raise ValueError(f"{name} must be {'(B, pages)' if dims == 2 else '(B,)'} for {B} sequences, its last dimension dense")
    return _cabi.PagedBatch(block_table.data_ptr(), block_table.stride(0), seq_lens.data_ptr(),
                            None if new_lens is None else new_lens.data_ptr(), block_table.shape[1], B, S, 0)


def _check_rows(cache: PagedKVCache, name: str, t: torch.Tensor, B: int, heads: Optional[int], S: int):
    if t.dtype != cache.dtype or t.device != cache.device:
        raise TypeError(f"{name} must be {cache.dtype} on {cache.device}, like the cache")
    if t.dim() != 4 or t.shape[0] != B or t.shape[2] != S or t.shape[3] != cache.head_dim or (t.shape[1] != heads if heads else t.shape[1] % cache.kv_heads or not t.shape[1]):
        raise ValueError(f"{name} has shape {tuple(t.shape)}: does not fit {B} sequences of {S} new tokens and the cache "
                         f"({cache.kv_heads} heads of {cache.head_dim})")


def _stream(device):
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _written(name: str, t: torch.Tensor, like: torch.Tensor):
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must have the shape, dtype and device of query_states")


def paged_kv_append(cache: PagedKVCache, key_states: torch.Tensor, value_states: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, new_lens: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                    sin: Optional[torch.Tensor] = None, query_states: Optional[torch.Tensor] = None,
                    query_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes the keys and values, (B, Hkv, S, D), of each sequence's new tokens into the cache, and returns the rotated queries.

    With ``cos`` and ``sin`` the keys are rotated on the way, x * cos + rotate_half(x) * sin in 32 bits and rounded once, and
    ``query_states`` (B, Hq, S, D), if given, into ``query_out`` (a new tensor by default; may be ``query_states``).  The tables
    are (positions, D), looked up by position, or (B or 1, S, D), one row per token as a model hands them over; of the cache's
    dtype.  Without them keys are taken as they are and None is returned.  Padding rows of ``query_out`` are 0.
    One kernel on the current stream, without synchronising."""
    if cache._native is not None:
        done = cache._host.paged_append(cache._native, key_states, value_states, block_table, seq_lens, new_lens, cos, sin, query_states, query_out)
        if done is not None:
            return None if done is True else done
    B, _, S, _ = key_states.shape
    _check_rows(cache, "key_states", key_states, B, cache.kv_heads, S)
    _check_rows(cache, "value_states", value_states, B, cache.kv_heads, S)
    batch = _batch(cache, B, S, block_table, seq_lens, new_lens)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if query_states is not None:
        if cos is None:
            raise ValueError("query_states are rotated: cos and sin are needed")
        _check_rows(cache, "query_states", query_states, B, None, S)
        if query_out is None:
            query_out = torch.empty_like(query_states)
        else:
            _written("query_out", query_out, query_states)
    elif query_out is not None:
        raise ValueError("query_out is for query_states, which are not given")
    rows, cs = 0, None
    if cos is not None:
        D = cache.head_dim
        if sin.shape != cos.shape or cos.shape[-1] != D or cos.dim() not in (2, 3) or cos.dim() == 3 and (cos.shape[1] != S or cos.shape[0] not in (1, B)):
            raise ValueError("cos / sin must be (positions, D) or (B or 1, S, D)")
        if cos.dtype != cache.dtype or sin.dtype != cache.dtype or cos.device != cache.device or sin.device != cache.device:
            raise TypeError(f"cos / sin must be {cache.dtype} on {cache.device}, like the cache")
        if not all(t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and not any(s * 2 % 16 for s in t.stride()[:-1]) for t in (cos, sin)) or sin.stride() != cos.stride():
            cos, sin = (t.clone(memory_format=torch.contiguous_format) for t in (cos, sin))
        if cos.dim() == 2:
            rows, cs = cos.shape[0], (C.c_int64 * 3)(0, cos.stride(0), 1)
        else:
            cs = (C.c_int64 * 3)(cos.stride(0) if cos.shape[0] > 1 else 0, cos.stride(1), 1)
        if rows == 0 and cos.dim() == 2:
            raise ValueError("cos / sin hold no position")
    if B * S == 0:
        return query_out
    k, v = _readable(key_states), _readable(value_states)
    q = None if query_states is None else _readable(query_states)
    qo = query_out if query_out is None else _readable(query_out)          # (a copy where the kernel cannot write to it)
    with torch.cuda.device(cache.device):
        _cabi.check(cache.lib.pbs_paged_append(C.byref(cache._c), C.byref(batch), _ptr(k), _strides(k), _ptr(v), _strides(v),
                                               0 if q is None else q.shape[1], _ptr(q), None if q is None else _strides(q), _ptr(qo),
                                               None if qo is None else _strides(qo), _ptr(cos), _ptr(sin), cs, rows, _stream(cache.device)),
                    "pbs_paged_append")
        if qo is not query_out:
            query_out.copy_(qo)
    return query_out


def paged_kv_gather(cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor, count: int,
                    new_lens: Optional[torch.Tensor] = None):
    """The last ``count`` tokens of each sequence (or the last ``new_lens[b]``, in the first rows) as the cache holds them: keys and values,
    (B, Hkv, count, D) of the cache's dtype, 0 where a sequence has no such token.  ``count`` = the longest sequence with ``new_lens`` =
    ``seq_lens`` reads everything."""
    if cache._native is not None:
        done = cache._host.paged_gather(cache._native, block_table, seq_lens, count, new_lens)
        if done is not None:
            return done
    B = seq_lens.shape[0]
    batch = _batch(cache, B, count, block_table, seq_lens, new_lens)
    # (B, S, H, D) memory: rows of one token lie together, as a projection's do
    k, v = (torch.empty(B, count, cache.kv_heads, cache.head_dim, dtype=cache.dtype, device=cache.device).transpose(1, 2) for _ in "kv")
    if k.numel() == 0:
        return k, v
    with torch.cuda.device(cache.device):
        _cabi.check(cache.lib.pbs_paged_gather(C.byref(cache._c), C.byref(batch), _ptr(k), _strides(k), _ptr(v), _strides(v),
                                               _stream(cache.device)), "pbs_paged_gather")
    return k, v


# Memory for partial results, one piece a stream: calls on a stream come after one another.
_WORKSPACES: dict = {}
_MAX_WORKSPACES = 8


def _workspace(device: torch.device, need: int) -> torch.Tensor:
    if torch.cuda.is_current_stream_capturing():           # a graph is replayed at times and on streams unknown here: it has its own
        space = torch.empty(need, dtype=torch.uint8, device=device)
        space[:_cabi.PAGED_COUNTER_BYTES].zero_()
        return space
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    space = _WORKSPACES.pop(key, None)                     # (back in behind the others: what was used longest ago goes first)
    if space is None or space.numel() < need:
        while len(_WORKSPACES) >= _MAX_WORKSPACES:
            _WORKSPACES.pop(next(iter(_WORKSPACES), None), None)
        space = torch.zeros(need, dtype=torch.uint8, device=device)
    _WORKSPACES[key] = space
    return space


def paged_attn_fwd(query_states: torch.Tensor, cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                   new_lens: Optional[torch.Tensor] = None, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the new tokens' queries, (B, Hq, S, D), over the cache, which holds their own keys already; query head h reads KV
    head h // (Hq // Hkv).  The result has the queries' shape, dtype and memory layout; rows that see no token (padding, or a sequence of
    length 0) are 0.  ``scale`` defaults to 1 / sqrt(D).  Made for one token a sequence or a few; any number works.
    One kernel on the current stream, without synchronising."""
    if cache._native is not None:
        done = cache._host.paged_attn(cache._native, query_states, block_table, seq_lens, new_lens, scale, out)
        if done is not None:
            return done
    B, Hq, S, D = query_states.shape
    _check_rows(cache, "query_states", query_states, B, None, S)
    batch = _batch(cache, B, S, block_table, seq_lens, new_lens)
    if out is None:
        out = torch.empty_like(query_states)
    else:
        _written("out", out, query_states)
    if query_states.numel() == 0:
        return out
    q, o = _readable(query_states), _readable(out)
    with torch.cuda.device(cache.device):
        need = C.c_int64()
        _cabi.check(cache.lib.pbs_paged_attn_workspace(C.byref(cache._c), C.byref(batch), Hq, C.byref(need)), "pbs_paged_attn_workspace")
        space = _workspace(cache.device, need.value)
        _cabi.check(cache.lib.pbs_paged_attn(C.byref(cache._c), C.byref(batch), Hq, _ptr(q), _strides(q), _ptr(o), _strides(o),
                                             1.0 / math.sqrt(D) if scale is None else float(scale), _ptr(space), space.numel(),
                                             _stream(cache.device)), "pbs_paged_attn")
        if o is not out:
            out.copy_(o)
    return out
