"""Measured workloads of generation with beams over a cache of 8 bits: writing and reading the cache, attention over it, the choice of
beams, and the reordering of the caches behind it.

A case is a dict of plain values; `op` says which:
  append   new keys and values into a paged cache of 8 bits, rotated on the way if `rope` (the queries too); then the tokens of all
           blocks that were touched are read back as the values that they stand for, the older ones among them
  attn     attention of the last `new` tokens of every sequence over a paged cache of 8 bits
  select   the best `keep` continuations of each batch entry's beams
  reorder  rows of a batch go on from other rows of their group of beams: tables and the page under way, in all layers

  batch, q_heads, kv_heads, head_dim, dtype, page (tokens a page), block (tokens that share a scale; 0 for pages of 16 bits)
  tokens   longest sequence, the new tokens among them;  shortest: the shortest (lengths are drawn between the two)
  new      new tokens a sequence;  ragged: True for 1 to `new` of them instead
  beams, vocab, keep;  first: True for a first step, where only one beam of each group is alive;  layers
"""
import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_LEAST = 2.0 ** -120                                       # least scale of a block


def _append(name, batch, new, tokens, q_heads=32, kv_heads=8, head_dim=128, dtype="bf16", page=64, block=16, rope=True, ragged=False):
    return {"name": name, "op": "append", "batch": batch, "new": new, "tokens": tokens, "shortest": max(new, tokens // 4),
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "page": page, "block": block,
            "rope": rope, "ragged": ragged}


def _attn(name, batch, tokens, new=1, shortest=None, q_heads=32, kv_heads=8, head_dim=128, dtype="bf16", page=64, block=16):
    return {"name": name, "op": "attn", "batch": batch, "new": new, "tokens": tokens, "shortest": shortest or tokens,
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "page": page, "block": block}


def _select(name, batch, beams, vocab, dtype="bf16", keep=None, first=False):
    return {"name": name, "op": "select", "batch": batch, "beams": beams, "vocab": vocab, "dtype": dtype, "keep": keep or 2 * beams,
            "first": first}


def _reorder(name, batch, beams, tokens, layers, kv_heads=8, head_dim=128, dtype="bf16", page=64, block=16):
    return {"name": name, "op": "reorder", "batch": batch, "beams": beams, "tokens": tokens, "shortest": max(1, tokens // 2),
            "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "page": page, "block": block}


def listed():
    return [
        # one chat's next token: launches and host work are all there is
        _append("append8_one", 1, 1, 4096),
        # a server's step with drafted tokens, up to four a sequence, narrow heads, coarse blocks, fp16
        _append("append8_64_drafts", 64, 4, 4000, head_dim=64, dtype="fp16", page=32, block=32, ragged=True),
        # a prompt's keys and values after its prefill, rotated already, of odd length
        _append("append8_prompt_8k", 1, 8191, 8191, rope=False),
        # the token after a short chat turn
        _attn("attn8_one_187", 1, 187),
        # the token after the longest prompt
        _attn("attn8_one_128k", 1, 131072),
        # a server's step with sequences of all lengths, 28 query heads on 4 KV heads, fp16
        _attn("attn8_32_ragged", 32, 8000, shortest=100, q_heads=28, kv_heads=4, dtype="fp16", page=32, block=32),
        # drafted tokens, small pages
        _attn("attn8_16x5", 16, 8192, new=5, shortest=2000, page=16),
        # a full server
        _attn("attn8_64_16k", 64, 16384, shortest=12000, block=64),
        # four beams of one answer
        _select("select_4", 1, 4, 128256),
        # a server's beams over a large vocabulary
        _select("select_64x8", 64, 8, 152064, dtype="fp32"),
        # four beams' caches of 8 bits (the tokens of the page under way are read back)
        _reorder("reorder_4", 1, 4, 1000, 32),
        # a server's beams, pages of 16 bits
        _reorder("reorder_8x4_16bit", 8, 4, 4000, 32, block=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "select", "reorder"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        return {"op": op, "batch": _log_int(rng, 1, 512 // beams), "beams": beams, "vocab": _log_int(rng, 1000, 152064),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "keep": rng.choice([beams, 2 * beams]), "first": rng.random() < 0.15}
    q_heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (32, 8, 128), (28, 4, 128), (4, 1, 128), (8, 8, 64), (32, 8, 64),
                                              (16, 2, 256)])
    page = rng.choice([16, 32, 64, 128])
    case = {"op": op, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "page": page,
            "block": rng.choice([b for b in (16, 32, 64) if b <= page])}
    if op == "reorder":
        beams, tokens = rng.choice([2, 3, 4, 5, 8]), _log_int(rng, 1, 16384)
        layers = rng.choice([1, 4, 28, 32])
        row = page * kv_heads * head_dim * layers           # values of a row's page under way, at most the largest listed case's
        batch = _log_int(rng, 1, max(1, min(64, 32 * 64 * 8 * 128 * 32 // (row * beams))))
        return case | {"batch": batch, "beams": beams, "tokens": tokens, "shortest": max(1, tokens // 2), "layers": layers,
                       "block": rng.choice([0, case["block"]])}
    if op == "append":
        if rng.random() < 0.5:                              # a step of a server
            batch, new = _log_int(rng, 1, 256), rng.choice([1, 1, rng.randint(2, 8)])
            tokens = _log_int(rng, 16, 4096)
        else:                                               # prompts
            batch = rng.choice([1, 1, 2, 4])
            new = tokens = _log_int(rng, 16, 16384 // batch)
        tokens = max(tokens, new)
        return case | {"batch": batch, "new": new, "tokens": tokens, "shortest": max(new, tokens // 3),
                       "rope": rng.random() < 0.7, "ragged": rng.random() < 0.3}
    batch = _log_int(rng, 1, 128)
    most = (1 << 30) // (kv_heads * head_dim * batch)       # tokens of one sequence, at the largest listed case's bytes in all
    tokens = _log_int(rng, 1, min(131072, most))
    new = min(tokens, rng.choice([1, 1, 1, rng.randint(2, 8)]))
    return case | {"batch": batch, "new": new, "tokens": tokens, "shortest": max(new, _log_int(rng, 1, tokens))}


def _lengths(case, seed):
    """Lengths of the sequences with their new tokens: the longest is as long as said."""
    g = torch.Generator().manual_seed(seed + 17)
    lens = torch.randint(case["shortest"], case["tokens"] + 1, (case["batch"],), generator=g)
    lens[0] = case["tokens"]
    return lens.int(), g


def _rope_tables(n, d, dtype):
    inv = 1.0 / (5e5 ** (torch.arange(0, d, 2, dtype=torch.float32, device="cuda") / d))
    ang = torch.arange(n, dtype=torch.float32, device="cuda")[:, None] * inv
    ang = torch.cat([ang, ang], -1)
    return ang.cos().to(dtype), ang.sin().to(dtype)


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    dt = _DTYPE[case["dtype"]]
    B = case["batch"]
    if case["op"] == "select":
        N = case["beams"]
        # running beams: sums of log-probabilities, best first; in a first step the prompt's own beam and nothing else
        scores = (-torch.rand(B, N, generator=g, device="cuda") * 20).sort(-1, descending=True).values
        if case["first"]:
            scores[:, 0], scores[:, 1:] = 0.0, -math.inf
        return {"case": case, "logits": (rand(B * N, case["vocab"]) * 3).to(dt), "scores": scores, "keep": case["keep"]}
    H, D, ps, bs = case["kv_heads"], case["head_dim"], case["page"], case["block"]
    lens, g_cpu = _lengths(case, seed)
    per = -(-case["tokens"] // ps)
    state = {"case": case, "lens": lens.cuda()}
    if case["op"] == "reorder":
        N, L = case["beams"], case["layers"]
        # a row's own page of what it writes now, and as many of the full ones that rows share
        pages = 2 * B * N
        order = torch.randperm(pages, generator=g, device="cuda").int()
        full = order[B * N + torch.randint(0, B * N, (B * N, per), generator=g, device="cuda")]
        j = torch.arange(per, device="cuda")
        state["lens"] = state["lens"].repeat_interleave(N)
        state["table"] = torch.where(j == (state["lens"] // ps)[:, None], order[:B * N, None], full).contiguous()
        # the better half goes on, the others go on from one of it
        half = (N + 1) // 2
        pick = torch.randint(0, half, (B, N), generator=g, device="cuda")
        i = torch.arange(N, device="cuda")
        state["beams"] = torch.where(i < half, i, pick).int()
        if bs:
            state["held"] = {n: (rand(L, pages, H, ps, D) * 40).clamp_(-127, 127).to(torch.int8) for n in "kv"}
            state["held"] |= {n + "_params": (2.5 + 2 * torch.rand(L, pages, H, ps // bs, generator=g, device="cuda")) / 127 for n in "kv"}
            # the rows of all layers, whose pages lie behind one another, and how far they have come in the pages under way (which they keep)
            at = torch.arange(L, device="cuda", dtype=torch.int32)[:, None, None] * pages
            state["all_rows"] = (state["table"] + at).flatten(0, 1), state["lens"].repeat(L), (state["lens"] % ps).repeat(L)
        else:
            state["held"] = {n: rand(L, pages, H, ps, D).to(dt) for n in "kv"}
        if own:
            from pbs_attn_b200.decode import PagedKVCache
            state["caches"] = [PagedKVCache.from_tensors(**{n: x[i] for n, x in state["held"].items()}, dtype=dt) for i in range(L)]
            state["all"] = PagedKVCache.from_tensors(**{n: x.flatten(0, 1) for n, x in state["held"].items()}, dtype=dt)
        return state
    pages = B * per + 3
    # the pages of a server that has run for a while lie in no order
    state["table"] = torch.randperm(pages, generator=g, device="cuda")[:B * per].view(B, per).int()
    shared = rand(D)
    shared /= shared.norm()
    held = {n: torch.empty(pages, H, ps, D, dtype=torch.int8, device="cuda") for n in "kv"}
    held |= {n + "_params": torch.empty(pages, H, ps // bs, device="cuda") for n in "kv"}
    for name in "kv":
        for p in range(0, pages, 4096):                     # (bounds the memory that the filling takes)
            x = rand(min(4096, pages - p), H, ps, D)
            if name == "k":                                 # a few keys that all queries look for
                x += 3.0 * shared * (torch.rand(*x.shape[:3], 1, generator=g, device="cuda") < 0.02)
            scale = x.unflatten(2, (-1, bs)).abs().amax((3, 4)) / 127
            if case["op"] == "append":                      # blocks under way have seen a part of their tokens
                scale *= 0.8 + 0.2 * torch.rand(scale.shape, generator=g, device="cuda")
            held[name][p:p + 4096] = (x / scale.repeat_interleave(bs, 2)[..., None]).round().clamp(-127, 127).to(torch.int8)
            held[name + "_params"][p:p + 4096] = scale
    state["held"] = held
    # (B, S, heads, D) memory seen as (B, heads, S, D), which is what a projection hands over
    x = lambda h: rand(B, case["new"], h, D).to(dt).transpose(1, 2)  # noqa: E731
    state["q"] = (x(case["q_heads"]).float() + shared).to(dt)
    if case["op"] == "append":
        state["new_lens"] = torch.randint(1, case["new"] + 1, (B,), generator=g_cpu).int().cuda() if case["ragged"] else None
        state["k_new"], state["v_new"] = x(H), x(H)
        state["cos"], state["sin"] = _rope_tables(case["tokens"], D, dt) if case["rope"] else (None, None)
    if own:
        from pbs_attn_b200.decode import PagedKVCache
        state["cache"] = PagedKVCache.from_tensors(**held, dtype=dt)
    return state


def run(state):
    case = state["case"]
    if case["op"] == "select":
        if not own:
            return _plain_select(state["logits"], state["scores"], state["keep"])
        from pbs_attn_b200.beam import beam_select
        return beam_select(state["logits"], state["scores"], state["keep"])
    if case["op"] == "reorder":
        if not own:
            return _plain_reorder(state)
        from pbs_attn_b200.decode import paged_kv_gather, paged_kv_reorder
        paged_kv_reorder(state["caches"], state["table"], state["lens"], state["beams"])
        out = {"table": state["table"]}
        if not case["block"]:
            return out | state["held"]
        table, lens, new = state["all_rows"]
        out["k"], out["v"] = paged_kv_gather(state["all"], table, lens, case["page"], new_lens=new)
        return out
    if case["op"] == "append":
        if not own:
            return _plain_append(state)
        from pbs_attn_b200.decode import paged_kv_append, paged_kv_gather
        q = paged_kv_append(state["cache"], state["k_new"], state["v_new"], state["table"], state["lens"], new_lens=state["new_lens"],
                            cos=state["cos"], sin=state["sin"], query_states=state["q"] if case["rope"] else None)
        k, v = paged_kv_gather(state["cache"], state["table"], state["lens"], _touched(case))
        return {"q": q, "k": k, "v": v}
    if own:
        from pbs_attn_b200.decode import paged_attn_fwd
        return paged_attn_fwd(state["q"], state["cache"], state["table"], state["lens"])
    return _plain_attn(state)


def _touched(case):
    """Tokens of the blocks that new ones came into, at most."""
    return min(case["tokens"], case["new"] + case["block"] - 1)


# ------------------------------------------------------------------------------------------------ the plain forms, in 32 bits
def _values(held, name, page, slot, block):
    """Values of the tokens in these slots of pages, (..., H, D), in 32 bits."""
    return held[name][page, :, slot].float() * held[name + "_params"][page, :, slot // block][..., None]


def _plain_append(state):
    case, held, dt = state["case"], state["held"], _DTYPE[state["case"]["dtype"]]
    B, S, ps, bs = case["batch"], case["new"], case["page"], case["block"]
    lens = state["lens"].long()
    new = state["new_lens"].long() if state["new_lens"] is not None else torch.full((B,), S, device="cuda")
    start = lens - new
    q, k, v = state["q"], state["k_new"].float(), state["v_new"].float()
    if case["rope"]:
        pos = (start[:, None] + torch.arange(S, device="cuda")).clamp(0, case["tokens"] - 1)
        cos, sin = state["cos"][pos].float()[:, None], state["sin"][pos].float()[:, None]
        there = torch.arange(S, device="cuda") < new[:, None]
        q = torch.where(there[:, None, :, None], _rotate(q.float(), cos, sin), 0.0).to(dt)
        k = _rotate(k, cos, sin)
    else:
        q = None
    # a window of whole blocks over what is written
    n = (S + bs - 2) // bs + 1
    pos = (start // bs * bs)[:, None] + torch.arange(n * bs, device="cuda")            # (B, W)
    fresh, kept = (pos >= start[:, None]) & (pos < lens[:, None]), pos < start[:, None]
    at = state["table"].long().gather(1, (pos // ps).clamp(max=state["table"].shape[1] - 1))
    row = (pos - start[:, None]).clamp(0, S - 1)
    back = []
    for name, x in (("k", k), ("v", v)):
        params = held[name + "_params"]
        x = x.transpose(1, 2).gather(1, row[..., None, None].expand(-1, -1, *x.shape[1::2])) * fresh[..., None, None]       # (B, W, H, D)
        amax = x.abs().amax(-1).unflatten(1, (n, bs)).amax(2)                          # (B, n, H)
        older = kept.unflatten(1, (n, bs))[:, :, :1]                                   # blocks that hold tokens already
        first, page = (pos % ps // bs)[:, ::bs], at[:, ::bs]
        old = params[page, :, first]
        scale = (amax * (1 / 127)).clamp(min=_LEAST)
        scale = torch.where(older, torch.maximum(scale, old), scale)
        wide = lambda s: s.repeat_interleave(bs, 1)[..., None]  # noqa: E731
        codes = torch.where(kept[..., None, None], (held[name][at, :, pos % ps].float() * wide(old / scale)), x * wide(1 / scale)).round()
        some = fresh | kept & fresh.unflatten(1, (n, bs)).any(2).repeat_interleave(bs, 1)
        held[name][at[some], :, (pos % ps)[some]] = codes[some].to(torch.int8)
        hit = fresh.unflatten(1, (n, bs)).any(2)
        params[page[hit], :, first[hit]] = scale[hit]
        p = lens[:, None] - _touched(case) + torch.arange(_touched(case), device="cuda")
        got = _values(held, name, state["table"].long().gather(1, p.clamp(min=0) // ps), p.clamp(min=0) % ps, bs)
        back.append((got * (p >= 0)[..., None, None]).to(dt).transpose(1, 2))
    return {"q": q, "k": back[0], "v": back[1]}


def _plain_attn(state):
    case, held = state["case"], state["held"]
    H, D, S, bs = case["kv_heads"], case["head_dim"], case["new"], case["block"]

    def seen(name):                                                        # (B, H, T, D) in 32 bits
        at = state["table"].long()
        x = held[name][at].float().unflatten(3, (-1, bs)) * held[name + "_params"][at][..., None, None]
        return x.flatten(3, 4).transpose(2, 1).flatten(2, 3)

    q = state["q"].float().unflatten(1, (H, -1))                           # (B, H, group, S, D)
    scores = (q.flatten(2, 3) / math.sqrt(D)) @ seen("k").transpose(-1, -2)
    scores = scores.unflatten(2, (-1, S))                                  # (B, H, group, S, T)
    last = state["lens"][:, None] - S + torch.arange(S, device="cuda")     # (B, S)
    hidden = torch.arange(scores.shape[-1], device="cuda") > last[..., None]
    scores = scores.masked_fill_(hidden[:, None, None], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp_()
    p = p / p.sum(-1, keepdim=True)
    return (p.flatten(2, 3) @ seen("v")).unflatten(2, (-1, S)).flatten(1, 2).to(_DTYPE[case["dtype"]])


def _plain_select(logits, scores, keep):
    B, N = scores.shape
    # in 64 bits: candidates of different beams may lie next to one another
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    x = x - top - (x - top).exp().sum(-1, keepdim=True).log()
    x = (x.view(B, N, -1) + scores.double()[..., None]).flatten(1)
    # the lowest places of those that are equal to the last that is kept, and all that are larger
    best, place = x.topk(keep)
    last, large = best[:, -1:], x.numel()
    order = torch.arange(x.shape[1], device="cuda")
    equal = torch.where(x == last, order, large).topk(min(keep, x.shape[1]), largest=False).values
    place = torch.cat([torch.where(best > last, place, large), equal], 1).sort(1).values
    value = torch.where(place < large, x.gather(1, place.clamp(max=x.shape[1] - 1)), -math.inf)
    value, at = value.sort(dim=1, descending=True, stable=True)
    place = place.gather(1, at)[:, :keep]
    V = logits.shape[1]
    return value[:, :keep].float(), (place // V).int(), place % V


def _plain_reorder(state):
    case, held, table = state["case"], state["held"], state["table"]
    B, N, ps, bs = case["batch"], case["beams"], case["page"], case["block"]
    parent = (torch.arange(B, device="cuda")[:, None] * N + state["beams"]).flatten()
    fill, under = state["lens"] % ps, state["lens"] // ps
    column = under.clamp(max=table.shape[1] - 1).long()[:, None]
    to, by = table.long().gather(1, column)[:, 0], table.long()[parent].gather(1, column)[:, 0]
    slot = torch.arange(ps, device="cuda")
    for name in held:
        there = slot < fill[:, None] if held[name].dim() == 5 else slot[::bs] < fill[:, None]
        there = there[:, None, :, None] if held[name].dim() == 5 else there[:, None]
        held[name][:, to] = torch.where(there, held[name][:, by], held[name][:, to])
    full = torch.arange(table.shape[1], device="cuda") < under[:, None]
    table.copy_(torch.where(full, table[parent], table))
    if not bs:
        return {"table": table} | held
    at, lens, new = state["all_rows"]
    p = (lens // ps * ps)[:, None] + slot
    page = at.long().gather(1, (p // ps).clamp(max=at.shape[1] - 1))
    there = (slot < new[:, None])[..., None, None]
    flat = {n: x.flatten(0, 1) for n, x in held.items()}
    back = [torch.where(there, _values(flat, n, page, slot.expand_as(page), bs), 0.0).to(_DTYPE[case["dtype"]]).transpose(1, 2) for n in "kv"]
    return {"table": table, "k": back[0], "v": back[1]}


def work(case):
    B = case["batch"]
    if case["op"] == "select":
        size, n = 4 if case["dtype"] == "fp32" else 2, B * case["beams"]
        return {"bytes": n * (size * case["vocab"] + 4) + 16 * B * case["keep"], "flops": 4.0 * n * case["vocab"]}
    H, D = case["kv_heads"], case["head_dim"]
    row = D + 4 / case["block"] if case["block"] else 2 * D                # bytes of one token's key (or value) of one head
    if case["op"] == "reorder":
        moved = B * (case["beams"] // 2) * case["page"] / 2                # tokens that are copied, and all that are read back
        back = B * case["beams"] * case["page"] * (row + 2 * D) / 2 if case["block"] else 0
        return {"bytes": case["layers"] * 2 * H * (2 * row * moved + back) + 8 * B * case["beams"] * (case["tokens"] / case["page"] + 2), "flops": 0}
    S = case["new"]
    if case["op"] == "append":
        new = S * (0.5 if case["ragged"] else 1.0) * B
        q = 2 * case["q_heads"] if case["rope"] else 0
        # read once, written once; what is in the blocks is then read and written back as values
        return {"bytes": new * (2 * D * (q + 2 * H) + 2 * H * row + (4 * D if case["rope"] else 0)) + B * _touched(case) * 2 * H * (row + 2 * D),
                "flops": new * D * (3 * (case["q_heads"] + H) * bool(case["rope"]) + 8 * H)}
    tokens = B * (case["tokens"] + case["shortest"]) / 2
    return {"bytes": 2 * H * row * tokens + 4 * B * case["q_heads"] * S * D, "flops": 4.0 * tokens * S * case["q_heads"] * D}


# ------------------------------------------------------------------ the definitions in 64 bits, one sequence, block or row at a time
def _exact_attn(case, seed):
    s = prepare(case, seed)
    D, S, H, bs = case["head_dim"], case["new"], case["kv_heads"], case["block"]
    out = []
    for b, n in enumerate(s["lens"].tolist()):
        t = torch.arange(n, device="cuda")
        page, slot = s["table"][b].long()[t // case["page"]], t % case["page"]
        k, v = (torch.einsum("thd,th->htd", s["held"][x][page, :, slot].double(), s["held"][x + "_params"][page, :, slot // bs].double()) for x in "kv")
        rows = []
        for i in range(S):
            q = s["q"][b, :, i].double().view(H, -1, D)
            e = n - S + i + 1
            p = torch.softmax(torch.einsum("hgd,htd->hgt", q, k[:, :e]) / D ** 0.5, -1)
            rows.append(torch.einsum("hgt,htd->hgd", p, v[:, :e]).flatten(0, 1))
        out.append(torch.stack(rows, 1))
    return torch.stack(out)


def _exact_append(case, seed):
    if case["new"] * case["batch"] > 40000:
        return None
    s = prepare(case, seed)
    D, B, S, ps, bs = case["head_dim"], case["batch"], case["new"], case["page"], case["block"]
    new = (s["new_lens"] if case["ragged"] else torch.full((B,), S)).tolist()
    count = _touched(case)
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda") if case["rope"] else None
    back = {n: torch.zeros(B, case["kv_heads"], count, D, dtype=torch.float64, device="cuda") for n in "kv"}
    for b, n in enumerate(s["lens"].tolist()):
        p = torch.arange(n - new[b], n, device="cuda")

        def turned(x):
            x = x[b, :, :new[b]].double()
            if not case["rope"]:
                return x
            c, z = s["cos"][p].double(), s["sin"][p].double()
            u, w = x.chunk(2, -1)
            cu, cw = c.chunk(2, -1)
            zu, zw = z.chunk(2, -1)
            return torch.cat([u * cu - w * zu, w * cw + u * zw], -1)

        if case["rope"]:
            q[b, :, :new[b]] = turned(s["q"])
        pages = s["table"][b].long()
        for name, x in (("k", turned(s["k_new"])), ("v", s["v_new"][b, :, :new[b]].double())):
            for block in range(max(0, n - count) // bs, (n - 1) // bs + 1):
                t0, t1 = block * bs, min(n, block * bs + bs)               # its tokens
                codes = s["held"][name][pages[t0 // ps], :, t0 % ps:t0 % ps + t1 - t0].double()
                scale = s["held"][name + "_params"][pages[t0 // ps], :, t0 % ps // bs].double()[:, None, None]
                w = max(t0, n - new[b])                                    # first new one
                if w < t1:
                    rows = x[:, w - (n - new[b]):t1 - (n - new[b])]
                    most = torch.clamp(rows.abs().amax((1, 2), keepdim=True) / 127, min=_LEAST)
                    if w > t0:
                        most = torch.maximum(most, scale)
                    codes = torch.cat([torch.round(codes[:, :w - t0] * scale / most), torch.round(rows / most)], 1)
                    scale = most
                r0 = max(t0, n - count)
                back[name][b, :, r0 - (n - count):t1 - (n - count)] = (codes * scale)[:, r0 - t0:]
    return {"q": q, **back}


def _exact_select(case, seed):
    s = prepare(case, seed)
    values = []
    for b in range(case["batch"]):
        rows = torch.log_softmax(s["logits"].view(case["batch"], case["beams"], -1)[b].double(), -1) + s["scores"][b].double()[:, None]
        values.append(rows.flatten().sort(descending=True).values[:case["keep"]])
    return [torch.stack(values), None, None]


def _exact_reorder(case, seed):
    s = prepare(case, seed)
    ps, bs, N, L = case["page"], case["block"], case["beams"], case["layers"]
    table, old = s["table"].long(), {n: x.clone() for n, x in s["held"].items()}
    back = {n: torch.zeros(L, table.shape[0], case["kv_heads"], ps, case["head_dim"], dtype=torch.float64, device="cuda") for n in "kv"} if bs else None
    for r, n in enumerate(s["lens"].tolist()):
        if n % ps == 0:
            continue
        src = table[r // N * N + int(s["beams"][r // N, r % N]), n // ps]
        for x in "kv":
            if bs:
                scale = old[x + "_params"][:, src].double().repeat_interleave(bs, -1)[..., None]
                back[x][:, r, :, :n % ps] = (old[x][:, src].double() * scale)[:, :, :n % ps]
            else:
                s["held"][x][:, table[r, n // ps], :, :n % ps] = old[x][:, src, :, :n % ps]
    return {"table": None, **({x: back[x].flatten(0, 1) for x in "kv"} if bs else {x: s["held"][x].double() for x in "kv"})}


def exact(case, seed):
    return {"attn": _exact_attn, "append": _exact_append, "select": _exact_select, "reorder": _exact_reorder}[case["op"]](case, seed)
