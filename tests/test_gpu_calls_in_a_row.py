"""Calls on one stream without a pause between them, which kernels are put on the SMs early for, give what they give one at a time."""
import pytest
import torch

from paged_ref import ints, rope_tables

pytestmark = pytest.mark.gpu


def _steps(bits, long, prompt, pause, how, rounds=40):
    """Rounds of append (rotated, with queries), attend, read back, choose and reorder, each on what the one before left."""
    from pbs_attn_b200.beam import beam_select
    from pbs_attn_b200.decode import PagedKVCache, paged_attn_fwd, paged_kv_append, paged_kv_gather, paged_kv_reorder
    B, N, H, D, V, ps = 2, 4, 2, 128, 4000, 64
    R, S = B * N, prompt or 1
    past = 1500 if long else 0
    per = (past + rounds * S) // ps + 2
    g = torch.Generator(device="cuda").manual_seed(bits)
    draw = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    caches = [PagedKVCache(R * per, ps, H, D, torch.bfloat16, "cuda", bits=bits, block_size=32) for _ in range(2)]
    for c in caches:
        for t in (c.k, c.v, c.k_params, c.v_params):
            if t is not None:
                t.zero_()
    table = torch.arange(R * per, dtype=torch.int32, device="cuda").view(R, per)
    lens, scores = torch.full((R,), past, dtype=torch.int32, device="cuda"), torch.zeros(B, N, device="cuda")
    cos, sin = rope_tables(per * ps, D, torch.bfloat16)
    if past:
        k = draw(1, H, past, D).expand(R, H, past, D)
        for c in caches:
            paged_kv_append(c, k, k, table, lens)
    rows, q0, out = draw(2, R, H, S, D), draw(R, 4 * H, S, D), draw(4 * H * D, V) / 4
    last, back = torch.zeros(R, H, S, D, dtype=torch.bfloat16, device="cuda"), torch.zeros(R, H, S, D, device="cuda")
    chosen = torch.zeros(B, N, dtype=torch.long, device="cuda")
    wait = torch.cuda.synchronize if pause else lambda: None

    def step():
        lens.add_(S)
        wait()
        o = 0
        for c in caches:
            k, v, q = rows[0] + last, rows[1] - last, q0 + last.repeat(1, 4, 1, 1)
            wait()
            q = paged_kv_append(c, k, v, table, lens, cos=cos, sin=sin, query_states=q)
            wait()
            x = paged_attn_fwd(q, c, table, lens)
            wait()
            x = paged_attn_fwd(x, c, table, lens)          # (two without a torch kernel in between)
            wait()
            got, values = paged_kv_gather(c, table, lens, S)
            wait()
            back.add_(got.float() - values.float())
            o = o + x
        wait()
        s, beams, tokens = beam_select(o[:, :, -1].reshape(R, 4 * H * D) @ out, scores, N)
        wait()
        paged_kv_reorder(caches, table, lens, beams)
        wait()
        scores.copy_(s - s[:, :1])
        chosen.copy_(tokens)
        last.copy_((tokens % 13).view(R, 1, 1, 1) / 13 + o[:, :H])

    step()
    if how == "captured":
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            # (what comes first waits for two streams, as behind a model's own branches)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                chosen.add_(0)
            torch.cuda.current_stream().wait_stream(side)
            step()
    for _ in range(rounds - 1):
        graph.replay() if how == "captured" else step()
    torch.cuda.synchronize()
    caches[0].check_status()
    return [x.clone() for x in (back, last, scores, chosen, table, lens)] + [t.clone() for c in caches for t in (c.k, c.v)]


@pytest.mark.parametrize("bits", [4, 8, 16])
@pytest.mark.parametrize("long,prompt", [(False, 0), (True, 0), (False, 40), (True, 5)])
def test_they_see_what_the_one_before_wrote(bits, long, prompt):
    """Short sequences and long ones, whose attention is launched for its CTAs to wait for one another, single tokens and prompts, whose queries may be
    a launch of their own; eager, captured, and on a stream beside another that does the same."""
    want = _steps(bits, long, prompt, True, "eager", 12)
    for how in ("eager", "captured"):
        assert all(torch.equal(a, b) for a, b in zip(_steps(bits, long, prompt, False, how, 12), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(_steps(bits, long, prompt, False, "eager", 12), want))
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_streams_that_call_at_the_same_time(bits):
    """Two streams with caches of their own, their calls enqueued in turn."""
    from pbs_attn_b200.beam import beam_select
    from pbs_attn_b200.decode import PagedKVCache, paged_attn_fwd, paged_kv_append
    g = torch.Generator(device="cuda").manual_seed(1)
    draw = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    table, lens = torch.arange(64, dtype=torch.int32, device="cuda").view(2, 32), ints(2000, 1700)
    k, q, logits, scores = draw(2, 2, 2000, 128), draw(2, 8, 1, 128), draw(8, 50000), torch.zeros(2, 4, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    caches = [PagedKVCache(64, 64, 2, 128, torch.bfloat16, "cuda", bits=bits, block_size=16) for _ in streams]
    results = [[] for _ in streams]
    torch.cuda.synchronize()
    for i in range(20):
        for s, c, r in zip(streams, caches, results):
            with torch.cuda.stream(s):
                paged_kv_append(c, k, k, table, lens, new_lens=lens)
                o = paged_attn_fwd(q, c, table, lens)
                r.append((o, *beam_select(logits, scores)))
    torch.cuda.synchronize()
    for r in results:
        for x in r:
            assert all(torch.equal(a, b) for a, b in zip(x, results[0][0]))
    caches[0].check_status()
