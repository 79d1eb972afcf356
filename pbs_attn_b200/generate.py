"""Generation on a patched model: the prompt through its prefill function, every further token through the paged cache.

    model = apply_patch_with_prefill(model, get_permuted_block_sparse_attn_fwd())
    tokens = generate(model, input_ids, max_new_tokens=64, bits=4, repetition_penalty=1.1)

A step is one replay of a CUDA graph: per layer the projections, ``paged_kv_append`` (which rotates), ``paged_attn_fwd`` and the MLP, then
``process_logits`` and the choice of the next token, or, with ``num_beams``, of the next tokens by ``beam_select`` and the reordering of the
caches by ``paged_kv_reorder``; lengths and histories live on the device, so nothing waits for the host.  The
reference patches prompts only and leaves single tokens to the model's own forward and cache (pbs_attn/patch/huggingface.py:182-192).
"""
from __future__ import annotations

import copy
import math
from typing import Optional, Sequence, Union

import torch

from .beam import MAX_BEAMS, MAX_KEEP, beam_select
from .decode import PagedKVCache, paged_attn_fwd, paged_kv_append, paged_kv_reorder
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
    anew for every 32 rows of a KV head (tokens times queries; 16 rows of 256 channels).

    With ``beams`` each sequence becomes that many rows by ``fork``, once the ``prompt`` tokens are in: its full pages are shared, and for what
    comes after them each row has pages of its own."""

    def __init__(self, model, batch: int, max_tokens: int, bits: int = 16, page_size: int = 64, group_size: int = 64, block_size: int = 16,
                 beams: int = 1, prompt: int = 0):
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
        shared = prompt // page_size
        pages = batch * (per + (beams - 1) * (per - shared))
        self.layers = [PagedKVCache(pages, page_size, heads, self.head_dim, weight.dtype, weight.device, bits, group_size, block_size)
                       for _ in model.model.layers]
        self.block_table = torch.arange(batch * per, dtype=torch.int32, device=weight.device).view(batch, per)
        self._beams, self._shared = beams, shared
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=weight.device)
        self.max_tokens, self.tokens = max_tokens, 0

    def add(self, tokens: int):
        """Counts the next call's tokens in."""
        if self.tokens + tokens > self.max_tokens:
            raise ValueError(f"the cache holds {self.max_tokens} tokens a sequence, {self.tokens + tokens} are asked for")
        self.tokens += tokens
        self.seq_lens += tokens

    def fork(self):
        """The prompt's sequences become groups of rows, of which the first alone holds the page under way: the others have to go on from it
        (``paged_kv_reorder``) before they are written to."""
        batch, per = self.block_table.shape
        table = self.block_table[:, None].repeat(1, self._beams, 1)
        table[:, 1:, self._shared:] = torch.arange(batch * per, batch * per + table[:, 1:, self._shared:].numel(), dtype=torch.int32,
                                                   device=table.device).view(batch, self._beams - 1, -1)
        self.block_table = table.flatten(0, 1)
        self.seq_lens = self.seq_lens.repeat_interleave(self._beams)

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


class _Beams:
    """The running beams of each sequence, those that have ended, and a step's choice among their continuations."""

    def __init__(self, input_ids: torch.Tensor, steps: int, beams: int, ends: Sequence[int], length_penalty: float):
        B, S = input_ids.shape
        device = input_ids.device
        self.N, self.S, self.power = beams, S, float(length_penalty)
        self.keep = beams * (1 + len(ends))                # (so many that N go on where each beam may end in every way)
        self.ends = torch.tensor(ends, device=device) if ends else None
        self.pad = ends[0] if ends else 0
        self.history = torch.zeros(B * beams, S + steps, dtype=torch.long, device=device)
        self.history[:, :S] = input_ids.repeat_interleave(beams, 0)
        self.rows = torch.arange(B, device=device)[:, None] * beams
        self.scores = torch.full((B, beams), float("-inf"), device=device)
        self.scores[:, 0] = 0.0                            # (all rows are the prompt still)
        # (in 64 bits: 32 do not hold large powers of a length)
        self.done_scores = torch.full((B, beams), float("-inf"), dtype=torch.double, device=device)
        self.done_tokens = torch.full((B, beams, steps), self.pad, dtype=torch.long, device=device)

    def choose(self, logits: torch.Tensor, cache: PagedModelCache) -> torch.Tensor:
        """(B * N, V) -> the next token of every row, (B * N, 1), with histories and caches in the order of the new rows."""
        scores, beams, tokens = beam_select(logits, self.scores, self.keep)
        written = self.history[:, self.S:]
        if self.ends is not None:
            ended = (tokens[..., None] == self.ends).any(-1)
            count = cache.seq_lens[0] - (self.S - 1)       # tokens written, this one among them
            # of the N best alone: one that comes after them is not a beam
            final = torch.where(ended[:, :self.N], scores[:, :self.N].double() / count.double() ** self.power, float("-inf"))
            texts = written[self.rows + beams[:, :self.N]]                            # (B, N, steps)
            texts = texts.scatter(2, (count - 1).long().expand(*texts.shape[:2], 1), tokens[:, :self.N, None])
            after = torch.arange(texts.shape[2], device=texts.device) >= count
            self._enter(final, texts.masked_fill(after, self.pad))
            first = ended.to(torch.uint8).argsort(dim=1, stable=True)[:, :self.N]      # the best that go on
            scores, beams, tokens = (x.gather(1, first) for x in (scores, beams, tokens))
        self.scores.copy_(scores)
        written.copy_(written[(self.rows + beams).flatten()])
        tokens = tokens.reshape(-1, 1)
        self.history.scatter_(1, cache.seq_lens.long()[:, None], tokens)              # behind the tokens that there are
        paged_kv_reorder(cache.layers, cache.block_table, cache.seq_lens, beams)
        return tokens

    def _enter(self, scores, texts):
        scores, texts = torch.cat([self.done_scores, scores], 1), torch.cat([self.done_tokens, texts], 1)
        scores, at = scores.topk(self.N)
        self.done_scores.copy_(scores)
        self.done_tokens.copy_(texts.gather(1, at[..., None].expand(-1, -1, texts.shape[2])))

    def best(self, input_ids: torch.Tensor) -> torch.Tensor:
        """The best of each sequence, those that have not ended among them: (B, S + steps)."""
        steps = self.done_tokens.shape[2]
        self._enter(self.scores.double() / steps ** self.power, self.history[:, self.S:].unflatten(0, (-1, self.N)))
        return torch.cat([input_ids, self.done_tokens[:, 0]], 1)


def _for_beams(x, beams: int, batch: int):
    """What is given by the sequence, by the row."""
    return x.repeat_interleave(beams, 0) if isinstance(x, torch.Tensor) and x.dim() and x.shape[0] == batch else x


@torch.no_grad()
def generate(model, input_ids: torch.Tensor, max_new_tokens: int, *, bits: int = 16, page_size: int = 64, group_size: int = 64,
             repetition_penalty=None, frequency_penalty=None, presence_penalty=None, bias_ids: Optional[torch.Tensor] = None,
             bias_values: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None, cuda_graph: bool = True,
             step_logits: Optional[list] = None, timings: Optional[dict] = None, block_size: int = 16, num_beams: int = 1,
             length_penalty: float = 1.0, eos_token_id: Optional[Union[int, Sequence[int]]] = None) -> torch.Tensor:
    """(B, S) prompts of one length -> (B, S + max_new_tokens): the token with the largest logit after penalties, biases and mask
    (the lowest of equals), step by step.

    ``model`` is a patched bfloat16 or float16 model with every layer patched (``apply_patch_with_prefill``).  ``bits``: what the cache
    holds keys and values in, 16, 8 (a scale for ``block_size`` tokens of a head) or 4 (a step and minimum for ``group_size`` channels of a
    token).  The arguments after them are those of ``process_logits``; the history is the whole sequence, its
    prompt part the prompt.  ``cuda_graph=False`` runs every step eagerly; ``step_logits``, a list, receives each step's logits before
    the penalties (eager steps only); ``timings``, a dict, receives ``ms_per_token`` of the steps behind the second new token.

    With ``num_beams`` N > 1 the N best continuations of each sequence go on instead: by the sum of their tokens' log-probabilities after penalties,
    biases and mask.  One of the N best that ends in ``eos_token_id`` (one or a few) leaves them, with its sum divided by its number of new tokens
    to the power of ``length_penalty`` (a power that 64 bits hold).  After ``max_new_tokens`` steps the best of those that ended and of those that run is returned, filled up with the
    (first) end token.  What is given by the sequence holds for its beams; ``step_logits`` has a row for each."""
    if not is_model_supported(model) or any("original_forward" not in layer.self_attn.__dict__ for layer in model.model.layers):
        raise ValueError("generate needs a model whose layers are all patched (apply_patch_with_prefill)")
    B, S = input_ids.shape
    if S < 1 or max_new_tokens < 1:
        raise ValueError("a prompt and at least one new token are needed")
    if step_logits is not None and cuda_graph:
        raise ValueError("step_logits are collected in eager steps (cuda_graph=False)")
    ends = () if eos_token_id is None else (eos_token_id,) if isinstance(eos_token_id, int) else tuple(eos_token_id)
    if num_beams < 1 or num_beams > MAX_BEAMS or num_beams * (1 + len(ends)) > MAX_KEEP:
        raise ValueError(f"num_beams={num_beams} with {len(ends)} end tokens: at most {MAX_BEAMS}, and {MAX_KEEP} continuations a step")
    if ends and num_beams == 1:
        raise ValueError("eos_token_id is for beams (num_beams > 1): a greedy sequence goes on for max_new_tokens")
    if num_beams > 1 and not (math.isfinite(length_penalty) and abs(length_penalty) * math.log(max_new_tokens) < 600):
        raise ValueError(f"length_penalty={length_penalty}: {max_new_tokens} to the power of it is beyond 64 bits")
    with torch.cuda.device(input_ids.device):              # (graphs, streams and events belong to the current one)
        cache = PagedModelCache(model, B, S + max_new_tokens, bits, page_size, group_size, block_size, num_beams, S)
        beams = _Beams(input_ids, max_new_tokens, num_beams, ends, length_penalty) if num_beams > 1 else None
        if beams is None:
            history = torch.zeros(B, S + max_new_tokens, dtype=torch.long, device=input_ids.device)
            history[:, :S] = input_ids
        else:
            history = beams.history
            repetition_penalty, frequency_penalty, presence_penalty, bias_ids, bias_values, allowed = (
                _for_beams(x, num_beams, B) for x in (repetition_penalty, frequency_penalty, presence_penalty, bias_ids, bias_values, allowed))
        prompt_lens = torch.full((history.shape[0],), S, dtype=torch.int32, device=input_ids.device)
        penalties = dict(repetition_penalty=repetition_penalty, frequency_penalty=frequency_penalty, presence_penalty=presence_penalty)
        penalised = any(p is not None for p in penalties.values())

        def choose(logits):
            if step_logits is not None:
                step_logits.append(logits.clone())
            if penalised:
                penalties.update(tokens=history, token_lens=cache.seq_lens, prompt_lens=prompt_lens)
            logits = process_logits(logits, bias_ids=bias_ids, bias_values=bias_values, allowed=allowed, **penalties)
            if beams is not None:
                return beams.choose(logits, cache)
            token = logits.argmax(-1, keepdim=True)
            history.scatter_(1, cache.seq_lens.long()[:, None], token)      # behind the tokens that there are
            return token

        cache.add(S)
        logits = _run_layers(model, input_ids, cache)
        if beams is not None:
            cache.fork()
            logits = logits.repeat_interleave(num_beams, 0)
        token = choose(logits)

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
        return history if beams is None else beams.best(input_ids)
