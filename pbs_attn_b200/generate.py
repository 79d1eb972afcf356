"""Generation on a patched model: the prompt through its prefill function, every further token through the paged cache.

    model = apply_patch_with_prefill(model, get_permuted_block_sparse_attn_fwd())
    tokens = generate(model, input_ids, max_new_tokens=64, bits=4, repetition_penalty=1.1)

A step is one replay of a CUDA graph: per layer the projections, ``paged_kv_append`` (which rotates), ``paged_attn_fwd`` and the MLP, then
``process_logits`` and the choice of the next token; lengths and histories live on the device, so nothing waits for the host.  The
reference patches prompts only and leaves single tokens to the model's own forward and cache (pbs_attn/patch/huggingface.py:182-192).
"""
from __future__ import annotations

import copy
from typing import Optional

import torch

from .decode import PagedKVCache, paged_attn_fwd, paged_kv_append
from .hf_patch import is_model_supported
from .logits import process_logits
from .prefill import apply_rope_


_STREAMS: dict = {}


def _capture_stream(device: torch.device):
    """One a device, as torch's own default is one of whichever device captured first: libraries keep workspaces by stream."""
    if device not in _STREAMS:
        _STREAMS[device] = torch.cuda.Stream(device)
    return _STREAMS[device]


class PagedModelCache:
    """A ``PagedKVCache`` for every layer of a model, with the block table and lengths that they share.

    Handed to the layers of a patched model as ``past_key_values``.  ``seq_lens`` counts the tokens of the current call in before
    the layers run; a call whose tokens are all that there are is the prompt and goes through the prefill function.  Any later call goes
    through ``paged_attn_fwd``, which is made for a few tokens: it reads the cache
    anew for every 32 rows of a KV head (tokens times queries; 16 rows of 256 channels)."""

    def __init__(self, model, batch: int, max_tokens: int, bits: int = 16, page_size: int = 64, group_size: int = 64):
        first = model.model.layers[0].self_attn
        weight = first.k_proj.weight
        self.head_dim = first.head_dim
        window = min((w for layer in model.model.layers if (w := getattr(layer.self_attn, "sliding_window", None))), default=max_tokens)
        if window < max_tokens:
            raise ValueError(f"a layer of the model sees a window of {window} tokens, and {max_tokens} are asked for: its steps would see them all")

        def tables(n):                                     # (of a copy: the module keeps what depends on the length, and the model's is its own)
            return copy.deepcopy(model.model.rotary_emb)(weight[:1, :1], torch.arange(n, device=weight.device)[None])

        cos, sin = tables(max_tokens)
        if not torch.equal(cos[:, :2], tables(2)[0][:, :max_tokens]):
            raise ValueError(f"the model's rotary tables change up to {max_tokens} tokens: keys that are cached rotated would not be the model's")
        self.cos, self.sin = (t[0].to(weight.dtype).contiguous() for t in (cos, sin))
        heads = weight.shape[0] // self.head_dim           # (of this rank's share, if the model is sharded by heads)
        per = -(-max_tokens // page_size)
        self.layers = [PagedKVCache(batch * per, page_size, heads, self.head_dim, weight.dtype, weight.device, bits, group_size)
                       for _ in model.model.layers]
        self.block_table = torch.arange(batch * per, dtype=torch.int32, device=weight.device).view(batch, per)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=weight.device)
        self.max_tokens, self.tokens = max_tokens, 0

    def add(self, tokens: int):
        """Counts the next call's tokens in."""
        if self.tokens + tokens > self.max_tokens:
            raise ValueError(f"the cache holds {self.max_tokens} tokens a sequence, {self.tokens + tokens} are asked for")
        self.tokens += tokens
        self.seq_lens += tokens

    def attend(self, attn, hidden_states: torch.Tensor, prefill_fn) -> torch.Tensor:
        """The attention layer ``attn`` on the call's tokens, up to the output projection."""
        B, S, _ = hidden_states.shape
        d, cache = self.head_dim, self.layers[attn.layer_idx]
        q, k, v = (p(hidden_states).view(B, S, -1, d).transpose(1, 2) for p in (attn.q_proj, attn.k_proj, attn.v_proj))
        if self.tokens == S and S > 1:
            cos, sin = self.cos[None, :S], self.sin[None, :S]
            q, k = apply_rope_(q, cos, sin), apply_rope_(k, cos, sin)
            paged_kv_append(cache, k, v, self.block_table, self.seq_lens)
            o = prefill_fn(q, k, v)
        else:
            q = paged_kv_append(cache, k, v, self.block_table, self.seq_lens, cos=self.cos, sin=self.sin, query_states=q)
            o = paged_attn_fwd(q, cache, self.block_table, self.seq_lens)
        return attn.o_proj(o.transpose(1, 2).reshape(B, S, -1))

    def check_status(self):
        self.layers[0].check_status()


def _run_layers(model, ids: torch.Tensor, cache: PagedModelCache) -> torch.Tensor:
    """Logits of the last of the call's tokens, (B, V)."""
    h = model.model.embed_tokens(ids)
    for layer in model.model.layers:
        h = layer(h, position_embeddings=None, past_key_values=cache, use_cache=True)
        h = h[0] if isinstance(h, tuple) else h
    return model.lm_head(model.model.norm(h[:, -1]))


@torch.no_grad()
def generate(model, input_ids: torch.Tensor, max_new_tokens: int, *, bits: int = 16, page_size: int = 64, group_size: int = 64,
             repetition_penalty=None, frequency_penalty=None, presence_penalty=None, bias_ids: Optional[torch.Tensor] = None,
             bias_values: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None, cuda_graph: bool = True,
             step_logits: Optional[list] = None, timings: Optional[dict] = None) -> torch.Tensor:
    """(B, S) prompts of one length -> (B, S + max_new_tokens): the token with the largest logit after penalties, biases and mask
    (the lowest of equals), step by step.

    ``model`` is a patched bfloat16 or float16 model with every layer patched (``apply_patch_with_prefill``).  ``bits``: what the cache
    holds keys and values in, 16 or 4.  The arguments after it are those of ``process_logits``; the history is the whole sequence, its
    prompt part the prompt.  ``cuda_graph=False`` runs every step eagerly; ``step_logits``, a list, receives each step's logits before
    the penalties (eager steps only); ``timings``, a dict, receives ``ms_per_token`` of the steps behind the second new token."""
    if not is_model_supported(model) or any("original_forward" not in layer.self_attn.__dict__ for layer in model.model.layers):
        raise ValueError("generate needs a model whose layers are all patched (apply_patch_with_prefill)")
    B, S = input_ids.shape
    if S < 1 or max_new_tokens < 1:
        raise ValueError("a prompt and at least one new token are needed")
    if step_logits is not None and cuda_graph:
        raise ValueError("step_logits are collected in eager steps (cuda_graph=False)")
    with torch.cuda.device(input_ids.device):              # (graphs, streams and events belong to the current one)
        cache = PagedModelCache(model, B, S + max_new_tokens, bits, page_size, group_size)
        history = torch.zeros(B, S + max_new_tokens, dtype=torch.long, device=input_ids.device)
        history[:, :S] = input_ids
        prompt_lens = torch.full((B,), S, dtype=torch.int32, device=input_ids.device)
        penalties = dict(repetition_penalty=repetition_penalty, frequency_penalty=frequency_penalty, presence_penalty=presence_penalty)
        if any(p is not None for p in penalties.values()):
            penalties.update(tokens=history, token_lens=cache.seq_lens, prompt_lens=prompt_lens)

        def choose(logits):
            if step_logits is not None:
                step_logits.append(logits.clone())
            logits = process_logits(logits, bias_ids=bias_ids, bias_values=bias_values, allowed=allowed, **penalties)
            token = logits.argmax(-1, keepdim=True)
            history.scatter_(1, cache.seq_lens.long()[:, None], token)      # behind the tokens that there are
            return token

        cache.add(S)
        token = choose(_run_layers(model, input_ids, cache))

        def step():
            token.copy_(choose(_run_layers(model, token, cache)))

        if max_new_tokens > 1:
            cache.add(1)
            step()                                             # (also brings up what a capture must not)
        if max_new_tokens > 2:
            if cuda_graph:
                torch.cuda.synchronize(input_ids.device)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=_capture_stream(input_ids.device)):
                    cache.seq_lens += 1
                    step()
                more = graph.replay
            else:
                def more():
                    cache.add(1)
                    step()
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            for _ in range(max_new_tokens - 2):
                more()
            end.record()
            if timings is not None:
                end.synchronize()
                timings["ms_per_token"] = start.elapsed_time(end) / (max_new_tokens - 2)
        cache.check_status()
        return history
