"""Generation with beams and caches of 8 bits: against the model itself, and against a plain beam search on the steps' own logits."""
import math

import pytest
import torch

from paged_ref import ints, assert_within
from paged_ref8 import attention8, make_cache8, values8
from test_gpu_generate import _model, _patched

pytestmark = pytest.mark.gpu


def _plain_search(steps, B, N, new, ends, power):
    """Beam search on recorded logits, a list of (B * N, V): the best texts, and each step's running texts before it, by the row."""
    best, before = [], [[] for _ in range(new)]
    for b in range(B):
        running, done = [([], 0.0 if i == 0 else -math.inf) for i in range(N)], []
        for t in range(new):
            before[t] += [text for text, _ in running]
            rows = torch.log_softmax(steps[t][b * N:(b + 1) * N].double(), -1)
            rows = rows + torch.tensor([s for _, s in running], dtype=torch.float64, device="cuda")[:, None]
            value, at = rows.flatten().sort(descending=True, stable=True)
            V, following = rows.shape[1], []
            for rank in range(N * (1 + len(ends))):
                i, v = divmod(int(at[rank]), V)
                text, score = running[i][0] + [v], float(value[rank])
                if v in ends:
                    if rank < N:
                        done.append((text, score / (t + 1) ** power))
                elif len(following) < N:
                    following.append((text, score))
            running = following
        done += [(text, score / new ** power) for text, score in running]
        text = max(done, key=lambda x: x[1])[0]
        best.append(text + [ends[0] if ends else 0] * (new - len(text)))
    return best, before


@pytest.mark.parametrize("kind,batch,prompt,N", [("llama", 1, 200, 4), ("llama", 3, 65, 3), ("qwen2", 2, 64, 5), ("qwen2", 2, 1, 2)])
@pytest.mark.parametrize("ends,power", [((), 1.0), ((5, 250), 0.6)])
def test_steps_follow_the_model_on_every_beam(kind, batch, prompt, N, ends, power):
    """With a cache of 16 bits each row's logits are those of the model on the row's text (the bound is that of greedy steps), and the
    result is that of a plain search on these logits."""
    from pbs_attn_b200.generate import generate
    from pbs_attn_b200.hf_patch import remove_patch
    model, new = _model(kind), 24
    ids = torch.randint(0, 300, (batch, prompt), device="cuda")
    bias = {}
    if ends:                                               # (so that some end)
        bias = dict(bias_ids=torch.tensor([list(ends)] * batch, device="cuda"), bias_values=torch.full((batch, 2), 1.0, device="cuda"))
    steps = []
    out = generate(_patched(model), ids, new, bits=16, page_size=16, cuda_graph=False, step_logits=steps, num_beams=N, length_penalty=power, eos_token_id=ends or None, **bias)
    assert out.shape == (batch, prompt + new) and torch.equal(out[:, :prompt], ids) and len(steps) == new
    biased = [s.clone() for s in steps]
    for s in biased if ends else ():
        s[:, list(ends)] = (s[:, list(ends)].float() + 1.0).to(s.dtype)
    best, before = _plain_search(biased, batch, N, new, ends, power)
    assert out[:, prompt:].tolist() == best
    remove_patch(model)
    for t in (1, 2, 9, 17, new - 1):
        rows = torch.tensor(before[t], device="cuda")
        with torch.no_grad():
            want = model(torch.cat([ids.repeat_interleave(N, 0), rows], 1)).logits[:, -1].float()
        bound = 5 * (32 ** 0.5) * 2.0 ** -8 * want.abs().amax(-1, keepdim=True)
        assert ((steps[t].float() - want).abs() <= bound).all()


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("N", [1, 4])
def test_graph_and_eager_choose_the_same(bits, N):
    from pbs_attn_b200.generate import generate
    model = _patched(_model())
    ids = torch.randint(0, 300, (2, 150), device="cuda")
    kw = dict(bits=bits, group_size=32, block_size=32, repetition_penalty=1.3, frequency_penalty=torch.tensor([0.1, 0.3], device="cuda"), presence_penalty=0.2, num_beams=N)
    if N > 1:
        kw.update(eos_token_id=7, length_penalty=2.0)
    a, b = generate(model, ids, 40, **kw), generate(model, ids, 40, cuda_graph=False, **kw)
    assert torch.equal(a, b)


def test_masks_reach_every_beam():
    from pbs_attn_b200.generate import generate
    model = _patched(_model())
    ids = torch.randint(0, 300, (2, 80), device="cuda")
    allowed = torch.zeros(2, 10, dtype=torch.int32, device="cuda")
    allowed[0, 3], allowed[1, 4] = 0b1111 << 4, 0b1111 << 4
    out = generate(model, ids, 12, bits=8, allowed=allowed, num_beams=3)[:, 80:]
    assert ((out[0] >= 100) & (out[0] < 104)).all() and ((out[1] >= 132) & (out[1] < 136)).all()
    out = generate(model, ids, 12, bits=8, allowed=allowed[:1], num_beams=3)[:, 80:]
    assert ((out >= 100) & (out < 104)).all()


def test_whole_numbers_as_length_penalties():
    from pbs_attn_b200.generate import generate
    model = _patched(_model())
    ids = torch.randint(0, 300, (1, 40), device="cuda")
    kw = dict(num_beams=3, eos_token_id=list(range(0, 60, 6)))
    for power in (-1, 0, 2):
        assert torch.equal(generate(model, ids, 8, length_penalty=power, **kw), generate(model, ids, 8, length_penalty=float(power), **kw))


def test_refusals():
    from pbs_attn_b200.generate import generate
    model = _patched(_model())
    ids = torch.zeros(1, 4, dtype=torch.long, device="cuda")
    for kw in (dict(num_beams=0), dict(num_beams=33), dict(num_beams=32, eos_token_id=(1, 2)), dict(eos_token_id=3)):
        with pytest.raises(ValueError, match="beams"):
            generate(model, ids, 3, **kw)
    with pytest.raises(ValueError, match="block_size"):
        generate(model, ids, 3, bits=8, block_size=24)


def test_call_after_call_keeps_no_memory():
    from pbs_attn_b200.generate import generate
    model = _patched(_model())
    ids = torch.randint(0, 300, (2, 150), device="cuda")
    held = []
    for _ in range(4):
        generate(model, ids, 6, bits=8, num_beams=4, eos_token_id=3)
        held.append(torch.cuda.memory_allocated())
    assert held[3] <= held[0]


@pytest.mark.parametrize("block", [16, 32])
def test_append_attend_select_and_reorder_together(block):
    """Steps of two groups of four beams over a cache of 8 bits: attention against the formula on what the cache stands for, which in turn is
    each row's own history, in spite of the pages that rows share.  A value is off by half a step when it is written and by half a step, of then and
    so no larger than now, each time that its block's scale grows: at most with each token that comes into the block behind it.  The reciprocals and
    ratios that codes up to 127 are multiplied by are rounded, up to 2^-23 together, which moves the border between two codes by up to 2^-16 of a step.
    (The values are of size 1, steps 0.03: that many of them tell one token's 128 values from another's.)"""
    from pbs_attn_b200.beam import beam_select
    from pbs_attn_b200.decode import paged_attn_fwd, paged_kv_append, paged_kv_reorder
    B, N, H, D, ps, prompt, new = 2, 4, 2, 64, 32, 37, 70
    R, per = B * N, -(-(prompt + new) // ps)
    g = torch.Generator(device="cuda").manual_seed(block)
    caches = [make_cache8(R * per, ps, H, D, torch.bfloat16, block) for _ in range(2)]
    table = torch.arange(R * per, dtype=torch.int32, device="cuda").view(R, per)
    x = torch.randn(B, 2, prompt, H, D, generator=g, device="cuda").bfloat16()          # a group's prompt is its first row's
    texts = [list(x[r // N].transpose(0, 1)) for r in range(R)]
    first = table[::N].contiguous()
    lens = torch.full((B,), prompt, dtype=torch.int32, device="cuda")
    for c in caches:
        paged_kv_append(c, x[:, 0].transpose(1, 2), x[:, 1].transpose(1, 2), first, lens)
    lens = lens.repeat_interleave(N)
    scores = torch.full((B, N), -math.inf, device="cuda")
    scores[:, 0] = 0
    V = 50
    for step in range(new):
        logits = torch.randn(R, V, generator=g, device="cuda") * 2
        scores, beams, _ = beam_select(logits, scores, N)
        assert scores.isfinite().all()
        paged_kv_reorder(caches, table, lens, beams)
        parents = (torch.arange(B, device="cuda")[:, None] * N + beams).flatten().tolist()
        texts = [list(texts[p]) for p in parents]
        lens += 1
        x = torch.randn(R, 2, 1, H, D, generator=g, device="cuda").bfloat16()
        q = torch.randn(R, 1, 2 * H, D, generator=g, device="cuda").bfloat16().transpose(1, 2)
        for r in range(R):
            texts[r].append(x[r, :, 0])
        for c in caches:
            paged_kv_append(c, x[:, 0].transpose(1, 2), x[:, 1].transpose(1, 2), table, lens)
        n = lens.tolist()
        got = [paged_attn_fwd(q, c, table, lens) for c in caches]
        assert torch.equal(got[0], got[1])
        if step % 7 == 0 or step > new - 3:
            assert_within(got[0], *attention8(q, caches[0], table, n))
            for r in range(R):
                own = torch.stack(texts[r]).double()                                    # (tokens, 2, H, D)
                for i, (codes, scales) in enumerate(((caches[1].k, caches[1].k_params), (caches[1].v, caches[1].v_params))):
                    value, _ = values8(caches[1], codes, scales, table, r, n[r])
                    t = torch.arange(n[r], device="cuda")
                    scale = scales[table[r].long()[t // ps], :, t % ps // block].double().t()[..., None]
                    off = (value - own[:, i].transpose(0, 1)).abs() / scale / ((0.5 + 2.0 ** -16) * (block - t % block)[:, None])
                    assert off.max() <= 1, (step, r, i, float(off.max()), (off > 1).nonzero()[:5].tolist())
    caches[0].check_status()


@pytest.mark.parametrize("captured", [False, True])
def test_calls_that_follow_one_another_see_what_the_one_before_wrote(captured):
    """Kernels are put on the SMs while the one before ends: append, attend, read back, reorder and select on one stream, many times over without a
    pause, give what they give with a pause after each."""
    from pbs_attn_b200.beam import beam_select
    from pbs_attn_b200.decode import PagedKVCache, paged_attn_fwd, paged_kv_append, paged_kv_gather, paged_kv_reorder
    B, N, H, D, V = 2, 4, 2, 128, 4000
    g = torch.Generator(device="cuda").manual_seed(21)
    rows = torch.randn(3, B * N, H, 1, D, generator=g, device="cuda").bfloat16()
    out = torch.randn(H * D, V, generator=g, device="cuda").bfloat16() / 4
    results = []
    for pause in (True, False):
        cache = PagedKVCache(B * N * 4, 64, H, D, torch.bfloat16, "cuda", bits=8, block_size=16)
        for t in (cache.k, cache.v, cache.k_params, cache.v_params):
            t.zero_()
        table = torch.arange(B * N * 4, dtype=torch.int32, device="cuda").view(B * N, 4)
        lens, scores = torch.zeros(B * N, dtype=torch.int32, device="cuda"), torch.zeros(B, N, device="cuda")
        last, back = torch.zeros(B * N, H, 1, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(B * N, H, 1, D, dtype=torch.bfloat16, device="cuda")

        def step():
            wait = torch.cuda.synchronize if pause else lambda: None
            lens.add_(1)
            k, v, q = rows[0] + last, rows[1] - last, rows[2] + last
            wait()
            paged_kv_append(cache, k, v, table, lens)
            wait()
            o = paged_attn_fwd(q, cache, table, lens)
            wait()
            got, _ = paged_kv_gather(cache, table, lens, 1)
            wait()
            back.add_(got)
            s, beams, tokens = beam_select(o.reshape(B * N, H * D) @ out, scores, N)
            wait()
            paged_kv_reorder(cache, table, lens, beams)
            wait()
            scores.copy_(s - s[:, :1])
            last.copy_(((tokens % 13).view(-1, 1, 1, 1) / 13 + o).bfloat16())

        step()
        if captured and not pause:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        for _ in range(150):
            graph.replay() if captured and not pause else step()
        torch.cuda.synchronize()
        cache.check_status()
        results.append([x.clone() for x in (back, last, scores, table, lens, cache.k, cache.v, cache.k_params)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("power", [30.0, 60.0, -30.0])
def test_length_penalties_whose_powers_32_bits_do_not_hold(power):
    """24 tokens to the power of 30 are more than 2^128: texts are told apart all the same."""
    from pbs_attn_b200.generate import generate
    model, new, ends = _model(), 24, tuple(range(0, 60, 6))
    ids = torch.randint(0, 300, (3, 40), device="cuda")
    steps = []
    out = generate(_patched(model), ids, new, cuda_graph=False, step_logits=steps, num_beams=4, length_penalty=power, eos_token_id=ends)
    assert out[:, 40:].tolist() == _plain_search(steps, 3, 4, new, ends, power)[0]
    assert torch.equal(out, generate(model, ids, new, num_beams=4, length_penalty=power, eos_token_id=ends))


def test_length_penalties_that_are_no_numbers_to_count_with():
    from pbs_attn_b200.generate import generate
    model = _patched(_model())
    ids = torch.zeros(1, 4, dtype=torch.long, device="cuda")
    for power in (math.inf, -math.inf, math.nan, 1e4, -1e4):
        with pytest.raises(ValueError, match="length_penalty"):
            generate(model, ids, 3, num_beams=2, length_penalty=power)
