"""Measured workloads of the operators that follow a prompt: paged cache, attention over it, logits.

A case is a dict of plain values; `op` says which:
  append   new keys and values into a paged cache, rotated on the way if `rope` (the queries too).  With 16-bit pages the
           pages are the result; with 4-bit pages the new tokens are read back as the values that they stand for
  attn     attention of the last `new` tokens of every sequence over a paged cache
  logits   penalties for repeated tokens, biases and a grammar mask

  batch, q_heads, kv_heads, head_dim, dtype, page (tokens a page), bits (of the cache: 4 or 16), group (channels that share
  a step and a minimum in 4 bits)
  tokens   longest sequence, the new tokens among them;  shortest: the shortest (lengths are drawn between the two)
  new      new tokens a sequence;  ragged: True for 1 to `new` of them instead
  vocab, history (longest), prompt (share of the history that is the prompt), banned (share of tokens that the grammar forbids)
"""
import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _append(name, batch, new, tokens, q_heads=32, kv_heads=8, head_dim=128, dtype="bf16", page=64, bits=4, group=64,
            rope=True, ragged=False):
    return {"name": name, "op": "append", "batch": batch, "new": new, "tokens": tokens, "shortest": max(new, tokens // 4),
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "page": page, "bits": bits,
            "group": group, "rope": rope, "ragged": ragged}


def _attn(name, batch, tokens, new=1, shortest=None, q_heads=32, kv_heads=8, head_dim=128, dtype="bf16", page=64, bits=4,
          group=64):
    return {"name": name, "op": "attn", "batch": batch, "new": new, "tokens": tokens, "shortest": shortest or tokens,
            "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "page": page, "bits": bits,
            "group": group, "ragged": False}


def _logits(name, batch, vocab, history, dtype="bf16", prompt=0.5, banned=0.5, biases=100):
    return {"name": name, "op": "logits", "batch": batch, "vocab": vocab, "history": history, "dtype": dtype,
            "prompt": prompt, "banned": banned, "biases": biases}


def listed():
    return [
        # one chat's next token: launches and host work are all there is
        _append("append_one", 1, 1, 4096),
        # a server's step, 64 sequences, pages of 16 bits
        _append("append_64_16bit", 64, 1, 4096, bits=16, page=16),
        # a prompt's keys and values after its prefill, rotated already, of odd length
        _append("append_prompt_8k", 1, 8191, 8191, rope=False),
        # drafted tokens, up to five a sequence, narrow heads and groups, fp16
        _append("append_drafts_fp16", 16, 5, 2000, head_dim=64, dtype="fp16", group=32, ragged=True),
        # the token after a short chat turn
        _attn("attn_one_187", 1, 187),
        # the token after a document, 28 query heads on 4 KV heads
        _attn("attn_one_32k", 1, 32768, q_heads=28, kv_heads=4),
        # the token after the longest prompt
        _attn("attn_one_128k", 1, 131072),
        # a server's step with sequences of all lengths, fp16, fine groups, small pages
        _attn("attn_32_ragged", 32, 8000, shortest=100, dtype="fp16", page=16, group=32),
        # drafted tokens over pages of 16 bits
        _attn("attn_8x5_16bit", 8, 8192, new=5, shortest=2000, bits=16),
        # a full server
        _attn("attn_64_16k", 64, 16384, shortest=12000),
        # one chat's logits
        _logits("logits_one", 1, 128256, 2000),
        # a server's logits with long histories
        _logits("logits_64", 64, 152064, 8192, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "logits"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "logits":
        batch = _log_int(rng, 1, 128)
        return {"op": op, "batch": batch, "vocab": _log_int(rng, 1000, 160000), "history": _log_int(rng, 1, 16384),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "prompt": round(rng.random(), 2),
                "banned": round(rng.choice([0.0, rng.random(), 0.99]), 2), "biases": rng.choice([0, _log_int(rng, 1, 300)])}
    q_heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (32, 8, 128), (28, 4, 128), (4, 1, 128), (8, 8, 64), (32, 8, 64),
                                              (16, 2, 256)])
    case = {"op": op, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
            "page": rng.choice([16, 32, 64, 128]), "bits": rng.choice([4, 4, 16]), "group": rng.choice([32, 64])}
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
    tokens = _log_int(rng, 1, min(131072, most // (4 if case["bits"] == 16 else 1)))
    new = min(tokens, rng.choice([1, 1, 1, rng.randint(2, 8)]))
    return case | {"batch": batch, "new": new, "tokens": tokens, "shortest": max(new, _log_int(rng, 1, tokens)), "ragged": False}


def _lengths(case, seed):
    """Lengths of the sequences with their new tokens, and the numbers of new tokens: the longest sequence is as long as said."""
    g = torch.Generator().manual_seed(seed + 17)
    lens = torch.randint(case["shortest"], case["tokens"] + 1, (case["batch"],), generator=g)
    lens[0] = case["tokens"]
    new = torch.full((case["batch"],), case["new"])
    if case["ragged"]:
        new = torch.randint(1, case["new"] + 1, (case["batch"],), generator=g)
    return lens.int(), new.int()


def _rope_tables(n, d, dtype):
    inv = 1.0 / (5e5 ** (torch.arange(0, d, 2, dtype=torch.float32, device="cuda") / d))
    ang = torch.arange(n, dtype=torch.float32, device="cuda")[:, None] * inv
    ang = torch.cat([ang, ang], -1)
    return ang.cos().to(dtype), ang.sin().to(dtype)


def _quantise(x, group, dtype):
    """(..., D) in 32 bits -> codes (..., D / group, group) and params (..., D / group, 2) of `dtype`."""
    x = x.unflatten(-1, (-1, group))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    params = torch.cat([(high * 0.5 - low * 0.5) * (2 / 15), low], -1).to(dtype)
    step, low = params.float().split(1, -1)
    codes = ((x - low) * torch.where(step > 0, 1 / step, 0.0)).round().clamp(0, 15)
    return codes.to(torch.uint8), params


def _pack(codes):
    c = codes.flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _values(packed, params):
    """The values that packed codes stand for, in 32 bits."""
    c = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float()
    step, low = params.float().split(1, -1)
    return (c.unflatten(-1, (step.shape[-2], -1)) * step + low).flatten(-2)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPE[case["dtype"]]
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    B = case["batch"]
    if case["op"] == "logits":
        V, L = case["vocab"], case["history"]
        # a history has few distinct tokens and many repeats, as text does
        zipf = torch.rand(B, L, generator=g, device="cuda").pow(4)
        words = torch.randint(0, V, (B, max(1, L // 2)), generator=g, device="cuda")
        tokens = words.gather(1, (zipf * words.shape[1]).long().clamp(max=words.shape[1] - 1))
        lens = torch.randint(0, L + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        lens[0] = L
        bits = (torch.rand(B, -(-V // 32) * 32, generator=g, device="cuda") >= case["banned"]).view(B, -1, 32).long()
        words = (bits << torch.arange(32, device="cuda")).sum(-1)
        allowed = torch.where(words >= 1 << 31, words - (1 << 32), words).int()
        n = min(case["biases"], V)
        at = torch.rand(B, V, generator=g, device="cuda").topk(n, dim=1).indices if n else None
        f = lambda lo, hi: torch.rand(B, generator=g, device="cuda") * (hi - lo) + lo  # noqa: E731
        return {"case": case, "logits": (rand(B, V) * 3).to(dt), "tokens": tokens, "token_lens": lens,
                "prompt_lens": (lens * case["prompt"]).int(), "repetition_penalty": f(1.0, 1.5), "frequency_penalty": f(0.0, 1.0),
                "presence_penalty": f(0.0, 1.0), "bias_ids": at, "bias_values": rand(B, n) * 4 if n else None, "allowed": allowed}
    H, D, ps, G = case["kv_heads"], case["head_dim"], case["page"], case["group"]
    lens, new = _lengths(case, seed)
    per = -(-case["tokens"] // ps)
    pages = B * per + 3
    # the pages of a server that has run for a while lie in no order
    table = torch.randperm(pages, generator=g, device="cuda")[:B * per].view(B, per).int()
    state = {"case": case, "table": table, "lens": lens.cuda(), "new_lens": new.cuda() if case["ragged"] else None}
    shared = rand(D)
    shared /= shared.norm()
    held = {}
    for name in ("k", "v"):
        if case["bits"] == 16:
            held[name] = torch.empty(pages, H, ps, D, dtype=dt, device="cuda")
        else:
            held[name] = torch.empty(pages, H, ps, D // 2, dtype=torch.uint8, device="cuda")
            held[name + "_params"] = torch.empty(pages, H, ps, D // G, 2, dtype=dt, device="cuda")
        for p in range(0, pages, 4096):                     # (bounds the memory that the filling takes)
            x = rand(min(4096, pages - p), H, ps, D)
            if name == "k":                                 # a few keys that all queries look for
                x += 3.0 * shared * (torch.rand(*x.shape[:3], 1, generator=g, device="cuda") < 0.02)
            if case["bits"] == 16:
                held[name][p:p + 4096] = x.to(dt)
            else:
                codes, params = _quantise(x, G, dt)
                held[name][p:p + 4096], held[name + "_params"][p:p + 4096] = _pack(codes), params
    state["held"] = held
    # (B, S, heads, D) memory seen as (B, heads, S, D), which is what a projection hands over
    x = lambda h: rand(B, case["new"], h, D).to(dt).transpose(1, 2)  # noqa: E731
    state["q"] = (x(case["q_heads"]).float() + shared).to(dt)
    if case["op"] == "append":
        state["k_new"], state["v_new"] = x(H), x(H)
        state["cos"], state["sin"] = _rope_tables(case["tokens"], D, dt) if case["rope"] else (None, None)
    if own:
        from pbs_attn_b200.decode import PagedKVCache
        state["cache"] = PagedKVCache.from_tensors(**held)
    return state


def run(state):
    case = state["case"]
    if case["op"] == "logits":
        args = {k: v for k, v in state.items() if k != "case"}
        if own:
            from pbs_attn_b200.logits import process_logits
            return process_logits(**args)
        return _plain_logits(**args)
    if case["op"] == "append":
        if not own:
            return _plain_append(state)
        from pbs_attn_b200.decode import paged_kv_append, paged_kv_gather
        cache = state["cache"]
        q = paged_kv_append(cache, state["k_new"], state["v_new"], state["table"], state["lens"], new_lens=state["new_lens"],
                            cos=state["cos"], sin=state["sin"], query_states=state["q"] if case["rope"] else None)
        if case["bits"] == 16:
            return {"q": q, "k": cache.k, "v": cache.v}
        k, v = paged_kv_gather(cache, state["table"], state["lens"], case["new"], new_lens=state["new_lens"])
        return {"q": q, "k": k, "v": v}
    if own:
        from pbs_attn_b200.decode import paged_attn_fwd
        return paged_attn_fwd(state["q"], state["cache"], state["table"], state["lens"])
    return _plain_attn(state)


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin


def _plain_append(state):
    case, held, dt = state["case"], state["held"], _DTYPE[state["case"]["dtype"]]
    B, S, ps = case["batch"], case["new"], case["page"]
    new = state["new_lens"] if state["new_lens"] is not None else torch.full((B,), S, device="cuda")
    i = torch.arange(S, device="cuda")
    fresh = i < new[:, None]                                               # (B, S)
    pos = ((state["lens"] - new)[:, None] + i).clamp(0, case["tokens"] - 1)
    q, k, v = state["q"], state["k_new"].float(), state["v_new"].float()
    if case["rope"]:
        cos, sin = state["cos"][pos].float()[:, None], state["sin"][pos].float()[:, None]
        q, k = _rotate(q.float(), cos, sin), _rotate(k, cos, sin)
        q = torch.where(fresh[:, None, :, None], q, 0.0).to(dt)
    else:
        q = None
    page, slot = state["table"].long().gather(1, pos // ps), pos % ps      # (B, S)
    page, slot = page[fresh], slot[fresh]
    back = []
    for name, x in (("k", k), ("v", v)):
        rows = x.transpose(1, 2)[fresh]                                    # (n, H, D)
        if case["bits"] == 16:
            held[name][page, :, slot] = rows.to(dt)
            back.append(held[name])
            continue
        codes, params = _quantise(rows, case["group"], dt)
        held[name][page, :, slot], held[name + "_params"][page, :, slot] = _pack(codes), params
        got = torch.zeros(B, S, *rows.shape[1:], dtype=dt, device="cuda")
        got[fresh] = _values(held[name][page, :, slot], held[name + "_params"][page, :, slot]).to(dt)
        back.append(got.transpose(1, 2))
    return {"q": q, "k": back[0], "v": back[1]}


def _plain_attn(state):
    case, held = state["case"], state["held"]
    B, H, D, S = case["batch"], case["kv_heads"], case["head_dim"], case["new"]

    def seen(name):                                                        # (B, H, T, D) in 32 bits
        at = state["table"].long()
        x = held[name][at].float() if case["bits"] == 16 else _values(held[name][at], held[name + "_params"][at])
        return x.transpose(2, 1).flatten(2, 3)

    q = state["q"].float().unflatten(1, (H, -1))                           # (B, H, group, S, D)
    scores = (q.flatten(2, 3) / math.sqrt(D)) @ seen("k").transpose(-1, -2)
    scores = scores.unflatten(2, (-1, S))                                  # (B, H, group, S, T)
    last = state["lens"][:, None] - S + torch.arange(S, device="cuda")     # (B, S)
    hidden = torch.arange(scores.shape[-1], device="cuda") > last[..., None]
    scores = scores.masked_fill_(hidden[:, None, None], -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp_()
    p = p / p.sum(-1, keepdim=True)
    return (p.flatten(2, 3) @ seen("v")).unflatten(2, (-1, S)).flatten(1, 2).to(_DTYPE[case["dtype"]])


def _plain_logits(logits, tokens, token_lens, prompt_lens, repetition_penalty, frequency_penalty, presence_penalty, bias_ids,
                  bias_values, allowed):
    B, V = logits.shape
    x = logits.float()
    at = torch.arange(tokens.shape[1], device="cuda")
    there = at < token_lens[:, None]
    written = there & (at >= prompt_lens[:, None])
    count = lambda m: torch.zeros(B, V, device="cuda").scatter_add_(1, tokens, m.float())  # noqa: E731
    r, made = repetition_penalty[:, None], count(written)
    x = torch.where(count(there) > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - frequency_penalty[:, None] * made
    x = x - presence_penalty[:, None] * (made > 0)
    if bias_ids is not None:
        x = x.scatter_add_(1, bias_ids, bias_values)
    may = (allowed[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    return x.masked_fill_(may.flatten(1)[:, :V] == 0, -math.inf).to(logits.dtype)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    B = case["batch"]
    if case["op"] == "logits":
        V = case["vocab"]
        return {"bytes": B * (2 * size * V + V / 8 + 8 * case["history"] * 0.5 + 12 * case["biases"]), "flops": 4.0 * B * V}
    H, D, S = case["kv_heads"], case["head_dim"], case["new"]
    row = 2 * D if case["bits"] == 16 else D // 2 + 4 * (D // case["group"])     # bytes of one token's key (or value) of one head
    if case["op"] == "append":
        new = S * (0.5 if case["ragged"] else 1.0) * B
        q = 2 * case["q_heads"] if case["rope"] else 0
        # read once, written once; 4 bits are then read and written back as values
        return {"bytes": new * (2 * D * (q + 2 * H) + 2 * H * row + (4 * D if case["rope"] else 0)
                                + (2 * H * (row + 2 * D) if case["bits"] == 4 else 0)),
                "flops": new * D * (3 * (case["q_heads"] + H) * bool(case["rope"]) + 8 * H)}
    tokens = B * (case["tokens"] + case["shortest"]) / 2
    return {"bytes": 2 * H * row * tokens + 4 * B * case["q_heads"] * S * D, "flops": 4.0 * tokens * S * case["q_heads"] * D}


# ------------------------------------------------------------------ the definitions in 64 bits, one sequence or row at a time
def _exact_rows(held, name, case, pages, count):
    """The first `count` tokens of a sequence as (H, count, D) in 64 bits."""
    if case["bits"] == 16:
        x = held[name][pages].double()
    else:
        packed, params = held[name][pages].int(), held[name + "_params"][pages].double()
        x = torch.empty(*packed.shape[:-1], case["head_dim"], dtype=torch.float64, device="cuda")
        x[..., 0::2], x[..., 1::2] = packed % 16, packed // 16
        x = (x.view(*params.shape[:-1], -1) * params[..., :1] + params[..., 1:]).flatten(-2)
    return x.permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, case["head_dim"])[:, :count]


def _exact_attn(case, seed):
    s = prepare(case, seed)
    D, S, H = case["head_dim"], case["new"], case["kv_heads"]
    out = []
    for b, n in enumerate(s["lens"].tolist()):
        k, v = (_exact_rows(s["held"], name, case, s["table"][b, :-(-n // case["page"])].long(), n) for name in ("k", "v"))
        rows = []
        for i in range(S):
            q = s["q"][b, :, i].double().view(H, -1, D)
            e = n - S + i + 1
            p = torch.softmax(torch.einsum("hgd,htd->hgt", q, k[:, :e]) / D ** 0.5, -1)
            rows.append(torch.einsum("hgt,htd->hgd", p, v[:, :e]).flatten(0, 1))
        out.append(torch.stack(rows, 1))
    return torch.stack(out)


def _exact_append(case, seed):
    s = prepare(case, seed)
    dt, D, G, B, S = _DTYPE[case["dtype"]], case["head_dim"], case["group"], case["batch"], case["new"]
    new = (s["new_lens"] if case["ragged"] else torch.full((B,), S)).tolist()
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda") if case["rope"] else None
    back = {n: torch.zeros(s["k_new"].shape, dtype=torch.float64, device="cuda") for n in ("k", "v")}
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
        for name, x in (("k", turned(s["k_new"])), ("v", s["v_new"][b, :, :new[b]].double())):
            if case["bits"] == 16:
                s["held"][name][s["table"][b].long()[p // case["page"]], :, p % case["page"]] = x.transpose(0, 1).to(dt)
                continue
            y = x.reshape(*x.shape[:-1], D // G, G)
            low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
            step, low = ((high - low) / 15).to(dt).double(), low.to(dt).double()
            back[name][b, :, :new[b]] = (torch.clamp(torch.round((y - low) / step), 0, 15) * step + low).flatten(-2)
    if case["bits"] == 16:
        back = {n: s["held"][n].double() for n in ("k", "v")}
    return {"q": q, **back}


def _exact_logits(case, seed):
    s = prepare(case, seed)
    V, out = case["vocab"], []
    for b in range(case["batch"]):
        n, m = int(s["token_lens"][b]), int(s["prompt_lens"][b])
        x = s["logits"][b].double()
        seen = torch.unique(s["tokens"][b, :n])
        r = float(s["repetition_penalty"][b])
        x[seen] = torch.where(x[seen] > 0, x[seen] / r, x[seen] * r)
        made, times = torch.unique(s["tokens"][b, m:n], return_counts=True)
        x[made] -= float(s["frequency_penalty"][b]) * times + float(s["presence_penalty"][b])
        if s["bias_ids"] is not None:
            x[s["bias_ids"][b]] += s["bias_values"][b].double()
        v = torch.arange(V, device="cuda")
        x[(s["allowed"][b][v // 32].long() >> (v % 32)) % 2 == 0] = -math.inf
        out.append(x)
    return torch.stack(out)


def exact(case, seed):
    return {"attn": _exact_attn, "append": _exact_append, "logits": _exact_logits}[case["op"]](case, seed)
