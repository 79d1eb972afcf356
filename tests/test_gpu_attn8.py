"""Attention of new tokens over a paged cache of 8 bits, against the formula in 64 bits on the values that the cache stands for."""
import math

import pytest
import torch

from paged_ref import assert_within, ints, make_table, pages_for
from paged_ref8 import attention8, make_cache8

pytestmark = pytest.mark.gpu


def _case(lens, Hq=8, Hkv=2, S=1, D=128, dtype=torch.bfloat16, block=16, ps=64, seed=0, token_major=False, spread=1.0, spare=0):
    """A cache with `lens` tokens, and queries: some keys are what the queries look for, some tokens are large."""
    from pbs_attn_b200.decode import paged_kv_append
    cache = make_cache8(pages_for(lens, ps), ps, Hkv, D, dtype, block, token_major)
    table = make_table(cache, lens, seed, spare)
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = max(max(lens), 1)
    x = lambda h, s: torch.randn(len(lens), s, h, D, generator=g, device="cuda").transpose(1, 2)  # noqa: E731
    shared = torch.randn(D, generator=g, device="cuda")
    shared /= shared.norm()
    k, v, q = x(Hkv, n), x(Hkv, n), x(Hq, S)
    k += 4 * spread * shared * (torch.rand(len(lens), 1, n, 1, generator=g, device="cuda") < 0.05)
    v *= torch.where(torch.rand(len(lens), Hkv, n, 1, generator=g, device="cuda") < 0.05, 8.0, 1.0)
    q = (q + 2 * spread * shared).to(dtype)
    if max(lens):
        paged_kv_append(cache, k.to(dtype), v.to(dtype), table, ints(*lens), new_lens=ints(*lens))
    return q, cache, table


def _run(q, cache, table, lens, new=None, **kw):
    from pbs_attn_b200.decode import paged_attn_fwd
    got = paged_attn_fwd(q, cache, table, ints(*lens), new_lens=None if new is None else ints(*new), **kw)
    cache.check_status()
    assert got.shape == q.shape and got.dtype == q.dtype
    assert_within(got, *attention8(q, cache, table, lens, new, kw.get("scale")))
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,S", [(4, 4, 1), (7, 1, 1), (8, 1, 1), (16, 2, 2), (28, 4, 5), (12, 1, 3), (20, 1, 1), (14, 2, 4)])
def test_types_and_heads(dtype, D, Hq, Hkv, S):
    lens = [300, 5, 77]
    _run(*_case(lens, Hq, Hkv, S, D, dtype, block=(16, 32, 64)[Hq % 3]), lens)


@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 1000, 2049, 5000])
def test_lengths(block, n):
    _run(*_case([n], block=block, seed=n), [n])


@pytest.mark.parametrize("ps,block", [(16, 16), (32, 16), (32, 32), (64, 32), (128, 64), (1024, 16), (1024, 64)])
@pytest.mark.parametrize("token_major", [False, True])
def test_pages(ps, block, token_major):
    lens = [1, ps - 1, ps, ps + 1, 3 * ps + 5]
    _run(*_case(lens, block=block, ps=ps, token_major=token_major, spare=2), lens)


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("S,new", [(4, [4, 1, 0, 3, 2]), (9, None), (33, [33, 1, 20, 0, 7]), (40, None)])
def test_new_tokens_that_differ_in_number_and_rows_that_see_nothing(block, S, new):
    lens = [200, 0, 33, 3, 1]
    _run(*_case(lens, 14, 2, S, block=block), lens, new)


def test_many_sequences_of_all_lengths():
    lens = [int(x) for x in torch.randint(0, 700, (150,), generator=torch.Generator().manual_seed(1))]
    lens[7], lens[80] = 6000, 0
    for dtype in (torch.bfloat16, torch.float16):
        _run(*_case(lens, 8, 2, 1, dtype=dtype, ps=16), lens)


def test_one_long_sequence():
    _run(*_case([70001], 8, 1, 1, spread=1.5), [70001])
    _run(*_case([70001], 8, 1, 1, dtype=torch.float16, block=64), [70001])


@pytest.mark.parametrize("scale", [0.0, 1e-6, 1.0, 30.0, -0.1])
def test_scales(scale):
    lens = [400]
    _run(*_case(lens), lens, scale=scale)


def test_layouts_of_queries_and_result():
    from pbs_attn_b200.decode import paged_attn_fwd
    lens = [70, 200]
    q, cache, table = _case(lens, S=3)
    want = _run(q, cache, table, lens)
    assert want.stride() == q.stride()
    assert torch.equal(_run(q.contiguous(), cache, table, lens), want)
    odd = torch.zeros(*q.shape[:3], 129, dtype=q.dtype, device="cuda")[..., 1:]
    odd.copy_(q)
    assert torch.equal(_run(odd, cache, table, lens), want)
    out = torch.zeros(2, 11, 3, 128, dtype=q.dtype, device="cuda")
    part = out[:, 2:10]
    assert paged_attn_fwd(q, cache, table, ints(*lens), out=part) is part and torch.equal(part, want)
    assert (out[:, :2] == 0).all() and (out[:, 10:] == 0).all()
    same = q.clone(memory_format=torch.preserve_format)
    assert paged_attn_fwd(same, cache, table, ints(*lens), out=same) is same and torch.equal(same, want)
    _run(q[:, :1].expand(2, 8, 3, 128), cache, table, lens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_and_values_of_very_different_sizes(dtype):
    """Maxima that rise from tile to tile, queries and values far from 1, steps that differ from block to block by up to 2^18."""
    from pbs_attn_b200.decode import paged_kv_append
    n, D, ps = 900, 128, 16
    big = 2.0 ** 9 if dtype == torch.float16 else 2.0 ** 30
    for q_size, k_size, v_size in ((1, 1, 1), (1 / big, big, 1 / big), (big, 1 / big, big), (1, 1, 2.0 ** -12)):
        g = torch.Generator(device="cuda").manual_seed(3)
        cache = make_cache8(60, ps, 1, D, dtype, 16)
        x = lambda s: torch.randn(1, 1, s, D, generator=g, device="cuda")  # noqa: E731
        k = x(n) * torch.linspace(0.1, 6, n, device="cuda")[:, None] * k_size
        v = x(n) * 2.0 ** (torch.arange(n, device="cuda") // 16 % 10 * 2 - 12)[:, None] * v_size
        q = (torch.randn(1, 8, 1, D, generator=g, device="cuda") * q_size).to(dtype)
        table = torch.arange(60, dtype=torch.int32, device="cuda")[None]
        paged_kv_append(cache, k.to(dtype), v.to(dtype), table, ints(n))
        _run(q, cache, table, [n])


def test_blocks_of_zeros_and_values_near_the_ends_of_bf16():
    from pbs_attn_b200.decode import paged_kv_append
    D, ps, n = 64, 16, 200
    table = torch.arange(13, dtype=torch.int32, device="cuda")[None]
    for size in (0.0, 2.0 ** -80, 2.0 ** 100):
        g = torch.Generator(device="cuda").manual_seed(8)
        cache = make_cache8(13, ps, 1, D, torch.bfloat16, 16)
        x = torch.randn(2, 1, 1, n, D, generator=g, device="cuda")
        v = x[1] * size
        v[:, :, 32:64] = 0
        q = torch.randn(1, 4, 1, D, generator=g, device="cuda").bfloat16()
        paged_kv_append(cache, x[0].bfloat16(), v.bfloat16(), table, ints(n))
        _run(q, cache, table, [n])
        # keys that are all 0: every token weighs the same
        cache = make_cache8(13, ps, 1, D, torch.bfloat16, 16)
        paged_kv_append(cache, x[0].bfloat16() * 0, v.bfloat16(), table, ints(n))
        _run(q, cache, table, [n])


@pytest.mark.parametrize("q_size,k_size", [(2.0 ** 120, 2.0 ** -115), (1.99 * 2.0 ** 127, 2.0 ** -116), (2.0 ** -110, 2.0 ** 118), (2.0 ** 60, 2.0 ** -60)])
def test_queries_and_keys_at_the_ends_of_bf16(q_size, k_size):
    from pbs_attn_b200.decode import paged_kv_append
    g = torch.Generator(device="cuda").manual_seed(9)
    n, D, ps = 300, 64, 16
    cache = make_cache8(20, ps, 1, D, torch.bfloat16, 16)
    x = torch.randn(2, 1, 1, n, D, generator=g, device="cuda").clamp(-4, 4)
    q = (torch.rand(1, 4, 1, D, generator=g, device="cuda", dtype=torch.float64) * 2 - 1) * q_size
    table = torch.arange(20, dtype=torch.int32, device="cuda")[None]
    paged_kv_append(cache, (x[0].double() * k_size).bfloat16(), x[1].bfloat16(), table, ints(n))
    _run(q.bfloat16(), cache, table, [n], scale=0.25 / (q_size * k_size))


def test_what_a_row_does_not_see_does_not_reach_it():
    """Blocks behind a row's last token that are not finite, stale pages among them; a block that a row sees makes it NaN."""
    from pbs_attn_b200.decode import paged_attn_fwd, paged_kv_append
    lens = [100]
    q, cache, table = _case(lens, S=30, block=16, ps=16)
    want = _run(q, cache, table, lens)
    k = torch.full((1, 2, 4, 128), math.nan, dtype=torch.bfloat16, device="cuda")
    cache.k_params[table[0, 6].long()] = math.nan             # tokens 96 .. 99, seen by the last four rows
    cache.v_params[table[0, 6].long()] = math.inf
    got = paged_attn_fwd(q, cache, table, ints(*lens))
    assert got[:, :, 26:].isnan().all()
    assert torch.equal(got[:, :, :26], want[:, :, :26])
    # and before the row's own end in its block
    lens2 = [96]
    again = paged_attn_fwd(q[:, :, :26], cache, table, ints(*lens2))
    assert not again.isnan().any()
    assert_within(again, *attention8(q[:, :, :26], cache, table, lens2))
    paged_kv_append(cache, k, k, table, ints(100))
    assert paged_attn_fwd(q, cache, table, ints(100))[:, :, 26:].isnan().all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_queries_that_are_not_finite(bad):
    """Their rows are NaN, and no others."""
    from pbs_attn_b200.decode import paged_attn_fwd
    lens = [90, 33]
    q, cache, table = _case(lens, S=2)
    want = paged_attn_fwd(q, cache, table, ints(*lens))
    q = q.clone()
    q[1, 3, 1, 77] = bad
    got = paged_attn_fwd(q, cache, table, ints(*lens))
    assert got[1, 3, 1].isnan().all()
    got[1, 3, 1] = want[1, 3, 1]
    assert torch.equal(got, want)


def test_queries_of_very_different_sizes():
    """One channel far above the others, mantissas next to the largest that two bytes hold, and rows of zeros."""
    from pbs_attn_b200.decode import paged_attn_fwd
    lens = [200]
    for dtype in (torch.bfloat16, torch.float16):
        q, cache, table = _case(lens, Hq=8, Hkv=1, dtype=dtype)
        q = q.clone()
        for i, x in enumerate((255 / 128, 127 / 64, 1.0, 1.9921264, 1.99999, 2.0 ** -10)):
            q[0, i, 0, 5 * i] = 8 * x
        q[0, 6] = 0
        q[0, 7, 0, 1:] = 0
        _run(q, cache, table, lens)
        assert paged_attn_fwd(q, cache, table, ints(*lens))[0, 6].isfinite().all()


def test_pages_that_are_not_there():
    from pbs_attn_b200 import _cabi
    from pbs_attn_b200.decode import paged_attn_fwd
    lens = [100]
    q, cache, table = _case(lens, ps=16)
    bad = table.clone()
    bad[0, 2] = 99
    got = paged_attn_fwd(q, cache, bad, ints(*lens))
    with pytest.raises(_cabi.PbsError, match="outside the pool"):
        cache.check_status()
    want = torch.cat([table[:, :2], table[:, 3:]], 1)         # (attention does not ask where a token is)
    assert_within(got, *attention8(q, cache, want, [84]))


def test_lengths_beyond_a_short_table_split_nothing():
    """Sequences of a table of two units are not split, so no CTA waits for another, whatever the lengths say."""
    from pbs_attn_b200 import _cabi
    from pbs_attn_b200.decode import paged_attn_fwd
    q, cache, table = _case([256, 100], ps=64)
    assert table.shape[1] == 4
    lib = _cabi.load()
    try:
        lib.pbs_debug_set_attn_wait(5_000_000, 1)          # 5 ms, and one would not arrive
        got = paged_attn_fwd(q, cache, table, ints(300, 100))
        torch.cuda.synchronize()
    finally:
        lib.pbs_debug_set_attn_wait(0, 0)
    with pytest.raises(_cabi.PbsError, match="longer than its row"):
        cache.check_status()
    assert_within(got, *attention8(q, cache, table, [256, 100]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_negative_scales_of_a_pool_that_was_filled_elsewhere(dtype):
    from pbs_attn_b200.decode import paged_kv_append, paged_kv_gather
    lens = [333, 40]
    q, cache, table = _case(lens, dtype=dtype, ps=32)
    want = paged_kv_gather(cache, table, ints(*lens), 333)
    for codes, scales in ((cache.k, cache.k_params), (cache.v, cache.v_params)):
        scales[:, :, ::2] *= -1
        codes[:, :, :16] *= -1
    assert all(torch.equal(a, b) for a, b in zip(want, paged_kv_gather(cache, table, ints(*lens), 333)))
    _run(q, cache, table, lens)
    # larger tokens behind the others of a block whose scale is negative
    lens, new = [335, 42], 100 * torch.ones(2, 2, 2, 128, dtype=dtype, device="cuda")
    before = want[0][1, :, -8:].double()                    # tokens 32 .. 39
    paged_kv_append(cache, new, new, table, ints(*lens))
    got = paged_kv_gather(cache, table, ints(*lens), 10)[0][1].double()
    step = cache.k_params[table[1, 1].long(), :, 0].double()
    assert (step > 0).all() and ((got[:, :8] - before).abs() <= step[:, None, None] * 0.51 + before.abs() * 2.0 ** -7).all()
    assert ((got[:, 8:] - 100).abs() <= step[:, None, None] * 0.51 + 100 * 2.0 ** -8).all()
    _run(q, cache, table, lens)


def test_same_bits_through_python_and_again(monkeypatch):
    from pbs_attn_b200.decode import paged_attn_fwd, paged_kv_append, paged_kv_gather
    lens = [3000, 17]
    q, cache, table = _case(lens, S=2)
    n = ints(*lens)
    k, v = q[:, :2].clone(), q[:, 2:4].clone()
    native = cache._native
    assert native is not None
    results = []
    for handle in (native, None, native):
        monkeypatch.setattr(cache, "_native", handle)
        paged_kv_append(cache, k, v, table, n)
        results.append([paged_attn_fwd(q, cache, table, n), *paged_kv_gather(cache, table, n, 50), cache.k.clone(), cache.v_params.clone()])
    for other in results[1:]:
        assert all(torch.equal(a.nan_to_num(7), b.nan_to_num(7)) for a, b in zip(results[0], other))


def test_captured_and_replayed_beside_other_streams():
    from pbs_attn_b200.decode import paged_attn_fwd
    lens = [5000, 700]
    q, cache, table = _case(lens)
    q2, cache2, table2 = _case(lens, seed=5)
    n = ints(*lens)
    want, want2 = paged_attn_fwd(q, cache, table, n), paged_attn_fwd(q2, cache2, table2, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attn_fwd(q, cache, table, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            got2 = paged_attn_fwd(q2, cache2, table2, n)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(got2, want2)
        out.zero_()
    cache.check_status()


def test_written_rows_attended_rows_and_rows_behind_them():
    """Append and attention together, token by token, each step against the formula on what the cache stands for."""
    from pbs_attn_b200.decode import paged_kv_append
    lens = [29, 64]
    q, cache, table = _case(lens, ps=32, block=16, spare=2)
    g = torch.Generator(device="cuda").manual_seed(11)
    free = [p for p in range(cache.num_pages) if p not in table[0, :1].tolist() + table[1, :2].tolist()]
    table[0, 1], table[1, 2] = free[0], free[1]
    for step in range(12):
        lens = [n + 1 for n in lens]
        x = torch.randn(3, 2, 2, 1, 128, generator=g, device="cuda").mul(1 + step / 3).bfloat16()
        paged_kv_append(cache, x[0], x[1], table, ints(*lens))
        _run(q, cache, table, lens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [2, 11, 200, 3000])
def test_channels_in_which_the_token_that_weighs_most_is_zero(dtype, n):
    """What is left there is small, beside sums of codes plus 128, up to 255 of a weight times its scale.  These run over up to eight tiles of up to two
    products of 17 terms, each of which is cut below 2^-23 of the largest, and what they are less is summed up the same: 2 * 16 * 17 * 255 * 2^-23 of the
    weighted scale at most, below 2^-5, beside the other bounds.  (Half a step of it is what a value lost when it was written.)"""
    from pbs_attn_b200.decode import paged_attn_fwd, paged_kv_append
    D, ps = 128, 64
    pages = -(-n // ps)
    for at in (0, n // 2, n - 1):
        g = torch.Generator(device="cuda").manual_seed(n + at)
        cache = make_cache8(pages, ps, 1, D, dtype, 64)
        k, v, q = (torch.randn(1, 1, s, D, generator=g, device="cuda") for s in (n, n, 1))
        k[0, 0, at] = 12 * q[0, 0, 0] / q.norm() * D ** 0.5 / q.norm() * D ** 0.5
        v[0, 0, at, :D // 2] = 0
        table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
        paged_kv_append(cache, k.to(dtype), v.to(dtype), table, ints(n))
        q = q.expand(1, 8, 1, D).to(dtype)
        got = paged_attn_fwd(q, cache, table, ints(n))
        cache.check_status()
        want, bound = attention8(q, cache, table, [n])
        scale = cache.v_params.abs().max().double()
        assert_within(got, want, bound + scale * 2.0 ** -5)
        assert (want[..., :D // 2].abs() < 1e-2 * want[..., D // 2:].abs().max()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,Hq,Hkv,S", [(128, 8, 2, 1), (128, 20, 1, 1), (64, 16, 2, 2), (256, 8, 1, 1)])
def test_a_results_own_rounding_is_the_largest_of_its_errors(dtype, D, Hq, Hkv, S):
    """Over a whole result what the kernel adds to rounding it once to its type stays below half of that rounding: sqrt(1 + 1 / 4) of it together."""
    from pbs_attn_b200.decode import paged_attn_fwd
    lens = [40, 300, 1200, 3000]
    for spread in (0.0, 1.0):
        q, cache, table = _case(lens, Hq, Hkv, S, D, dtype, spread=spread, seed=3)
        want, _ = attention8(q, cache, table, lens)
        got = paged_attn_fwd(q, cache, table, ints(*lens))
        off, own = (got.double() - want).norm(), (want.to(dtype).double() - want).norm()
        assert off <= math.sqrt(1.25) * own, (float(off / want.norm()), float(own / want.norm()))
