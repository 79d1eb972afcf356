"""Pools of more than 4 GiB and logits of more than 2^31: the same bits as with the same tokens near the beginning."""
import pytest
import torch

from paged_ref import ints, rope_tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 8, 16])
def test_pages_beyond_four_gibibytes(bits):
    from pbs_attn_b200.decode import PagedKVCache, paged_attn_fwd, paged_kv_append, paged_kv_gather, paged_kv_reorder
    H, D, ps, n = 4, 256, 64, 300
    page = H * ps * D * bits // 8
    far = 5 * 2 ** 30 // page
    g = torch.Generator(device="cuda").manual_seed(bits)
    draw = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    k, v = draw(2, H, n, D), draw(2, H, n, D)
    steps = draw(3, 2, H, 3, D)
    q = draw(2, 4 * H, 3, D)
    cos, sin = rope_tables(400, D, torch.bfloat16)
    gib = 2 ** 30 // page
    tables = [[[0, 1, 2, 3, 4, 5], [6, 7, 8, 9, 10, 11]],
              [[far - 1, 2 * gib, 2 * gib - 1, 4 * gib, 4 * gib - 1, 4 * gib + 3], [far - 2, 0, gib, 3 * gib + 1, far - 5, 4 * gib + 1]]]
    results = []
    for pages, table in ((12, tables[0]), (far, tables[1])):
        cache = PagedKVCache(pages, ps, H, D, torch.bfloat16, "cuda", bits=bits, block_size=32)
        table = torch.tensor(table, dtype=torch.int32, device="cuda")
        lens = ints(n, n)
        paged_kv_append(cache, k, v, table, lens)
        out = []
        for i in range(3):
            lens = lens + 3
            turned = paged_kv_append(cache, steps[i], steps[i - 1], table, lens, cos=cos, sin=sin, query_states=q)
            out.append(paged_attn_fwd(turned, cache, table, lens))
            names = table.clone()
            paged_kv_reorder(cache, table, lens, ints(1, 0)[None] if i == 1 else ints(1, 1)[None])
            out += [x.clone() for x in paged_kv_gather(cache, table, lens, 309)]
            assert torch.equal(table[0, :4], names[1, :4]) and torch.equal(table[:, 4:], names[:, 4:])
            if i != 1:                                     # (the rows share their full pages from here on, and go on apart)
                assert all(torch.equal(x[0], x[1]) for x in out[-2:])
        cache.check_status()
        results.append(out)
        del cache
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_logits_far_apart(dtype):
    from pbs_attn_b200.beam import beam_select
    V, stride, rows = 3001, 2 ** 27 + 5, 20
    g = torch.Generator(device="cuda").manual_seed(1)
    logits, scores = torch.randn(rows, V, generator=g, device="cuda").to(dtype), torch.rand(5, 4, generator=g, device="cuda")
    memory = torch.empty(rows * stride, dtype=dtype, device="cuda")
    view = memory.view(rows, stride)[:, :V]
    view.copy_(logits)
    want, got = beam_select(logits, scores), beam_select(view, scores)
    assert all(torch.equal(a, b) for a, b in zip(want[1:], got[1:]))
    # (rows begin elsewhere between boundaries: sums are added in another order)
    assert (want[0] - got[0]).abs().max() <= 1e-4
