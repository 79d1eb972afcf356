"""Attention of new tokens over a paged cache of 16 or 4 bits, against the formula in 64 bits on the values that the cache stands for."""
import math

import pytest
import torch

from paged_ref import assert_within, attention, ints, make_cache, make_table, pages_for

pytestmark = pytest.mark.gpu


def _case(lens, Hq=8, Hkv=2, S=1, D=128, dtype=torch.bfloat16, bits=4, group=64, ps=16, seed=0, token_major=False, spread=1.0, spare=0):
    """A cache with `lens` tokens, and queries: some keys are what the queries look for, some tokens are large."""
    from pbs_attn_b200.decode import paged_kv_append
    cache = make_cache(pages_for(lens, ps), ps, Hkv, D, dtype, bits, group, token_major)
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
    assert_within(got, *attention(q, cache, table, lens, new, kw.get("scale")))
    return got


FORMATS = [(16, 0), (4, 32), (4, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits,group", FORMATS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,S", [(4, 4, 1), (7, 1, 1), (8, 1, 1), (16, 2, 2), (28, 4, 5), (12, 1, 3)])
def test_types_and_heads(dtype, bits, group, D, Hq, Hkv, S):
    lens = [300, 5, 77]
    _run(*_case(lens, Hq, Hkv, S, D, dtype, bits, group), lens)


@pytest.mark.parametrize("bits,group", FORMATS)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 1000, 2049, 5000])
def test_lengths(bits, group, n):
    _run(*_case([n], bits=bits, group=group, ps=32, seed=n), [n])


@pytest.mark.parametrize("bits,group", FORMATS)
@pytest.mark.parametrize("ps", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("token_major", [False, True])
def test_pages(bits, group, ps, token_major):
    lens = [1, ps - 1, ps, ps + 1, 3 * ps + 5]
    _run(*_case(lens, bits=bits, group=group, ps=ps, token_major=token_major, S=1, spare=2), lens)


@pytest.mark.parametrize("bits,group", FORMATS)
@pytest.mark.parametrize("S,new", [(4, [4, 1, 0, 3, 2]), (9, None), (33, [33, 1, 20, 0, 7]), (40, None)])
def test_new_tokens_that_differ_in_number_and_rows_that_see_nothing(bits, group, S, new):
    lens = [200, 0, 33, 3, 1]
    _run(*_case(lens, 14, 2, S, bits=bits, group=group), lens, new)


def test_many_sequences_of_all_lengths():
    lens = [int(x) for x in torch.randint(0, 700, (150,), generator=torch.Generator().manual_seed(1))]
    lens[7], lens[80] = 6000, 0
    _run(*_case(lens, 8, 2, 1), lens)


def test_one_long_sequence():
    lens = [70001]
    for bits, group in FORMATS:
        _run(*_case(lens, 8, 1, 1, bits=bits, group=group, ps=64, spread=1.5), lens)


def test_batches_at_the_edges_of_what_the_threads_look_up_at_once():
    for B in (31, 32, 33, 255, 256, 257, 600):
        lens = [(37 * b) % 90 for b in range(B)]
        _run(*_case(lens, 2, 1, 1, 64, seed=B), lens)


@pytest.mark.parametrize("bits,group", FORMATS)
def test_layouts_of_queries_and_result(bits, group):
    from pbs_attn_b200.decode import paged_attn_fwd
    lens = [70, 200]
    q, cache, table = _case(lens, S=3, bits=bits, group=group)
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
    odd.zero_()
    assert paged_attn_fwd(q, cache, table, ints(*lens), out=odd) is odd and torch.equal(odd, want)
    same = q.clone(memory_format=torch.preserve_format)
    assert paged_attn_fwd(same, cache, table, ints(*lens), out=same) is same and torch.equal(same, want)
    one = q[:, :1].expand(2, 8, 3, 128)
    _run(one, cache, table, lens)


@pytest.mark.parametrize("bits,group", FORMATS)
@pytest.mark.parametrize("scale", [0.0, 1e-6, 1.0, 30.0, -0.1])
def test_scales(bits, group, scale):
    lens = [400]
    _run(*_case(lens, bits=bits, group=group), lens, scale=scale)


@pytest.mark.parametrize("bits,group", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_and_values_of_very_different_sizes(bits, group, dtype):
    """Maxima that rise from tile to tile, queries and values far from 1."""
    from pbs_attn_b200.decode import paged_kv_append
    n, D, ps = 900, 128, 16
    big = 2.0 ** 9 if dtype == torch.float16 else 2.0 ** 30
    g = torch.Generator(device="cuda").manual_seed(3)
    for q_size, k_size, v_size in ((1, 1, 1), (1 / big, big, 1 / big), (big, 1 / big, big), (1, 1, 2.0 ** -12)):
        cache = make_cache(60, ps, 1, D, dtype, bits, group)
        table = make_table(cache, [n])
        k, v = (torch.randn(1, 1, n, D, generator=g, device="cuda") for _ in "kv")
        q = torch.randn(1, 4, 1, D, generator=g, device="cuda")
        rise = torch.linspace(-3, 3, n, device="cuda")[:, None]
        k += rise * q[0, 0, 0] / q[0, 0, 0].norm() * 4
        v *= torch.linspace(-10, 0, n, device="cuda").exp2()[:, None]
        paged_kv_append(cache, (k * k_size).to(dtype), (v * v_size).to(dtype), table, ints(n))
        _run((q * q_size).to(dtype), cache, table, [n])
        order = torch.arange(n - 1, -1, -1, device="cuda")              # and falling ones
        paged_kv_append(cache, (k[:, :, order] * k_size).to(dtype), (v[:, :, order] * v_size).to(dtype), table, ints(n))
        _run((q * q_size).to(dtype), cache, table, [n])


@pytest.mark.parametrize("bits,group", FORMATS)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see_does_not_reach_it(bits, group, value):
    """NaN and infinities in the keys and values of later tokens; behind the sequence's end the pages hold NaN anyway."""
    from pbs_attn_b200.decode import paged_attn_fwd, paged_kv_append
    n, S, D = 50, 5, 128
    q, cache, table = _case([n], S=S, bits=bits, group=group)
    want = paged_attn_fwd(q, cache, table, ints(n))
    for at in (n - 1, n - 3):
        bad = torch.full((1, 2, 1, D), value, dtype=q.dtype, device="cuda")
        paged_kv_append(cache, bad, bad, table, ints(at + 1))
        got = paged_attn_fwd(q, cache, table, ints(n))
        cache.check_status()
        first = at - (n - S)                                # first row that sees it
        assert torch.equal(got[:, :, :first], want[:, :, :first])
        assert not got[:, :, first:].isfinite().any()


def test_values_that_are_not_finite_are_seen():
    """A value of infinity in 16 bits reaches its channel of the rows that see it, and no other."""
    from pbs_attn_b200.decode import paged_attn_fwd
    n, S = 40, 3
    for dtype in (torch.bfloat16, torch.float16):
        q, cache, table = _case([n], S=S, bits=16, group=0, dtype=dtype)
        want = paged_attn_fwd(q, cache, table, ints(n))
        p = n - 2
        cache.v[int(table[0, p // 16]), 1, p % 16, 9] = math.inf
        got = paged_attn_fwd(q, cache, table, ints(n))
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[:, 4:, 1:, 9] = True
        assert (got[hit] == math.inf).all() and torch.equal(got[~hit], want[~hit])


def test_queries_that_are_not_finite_keep_to_their_rows():
    from pbs_attn_b200.decode import paged_attn_fwd
    for bits, group in FORMATS:
        q, cache, table = _case([300], bits=bits, group=group)
        want = paged_attn_fwd(q, cache, table, ints(300))
        for value in (math.nan, math.inf):
            bad = q.clone(memory_format=torch.preserve_format)
            bad[0, 5, 0, 17] = value
            got = paged_attn_fwd(bad, cache, table, ints(300))
            rows = torch.arange(8, device="cuda") != 5
            assert torch.equal(got[:, rows], want[:, rows]) and not got[:, 5].isfinite().any()


def test_same_bits_every_time_and_on_streams():
    from pbs_attn_b200.decode import paged_attn_fwd
    lens = [9000, 1, 400, 3333]
    q, cache, table = _case(lens, 8, 2, 2)
    t = ints(*lens)
    want = paged_attn_fwd(q, cache, table, t)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                got = paged_attn_fwd(q, cache, table, t)
                got.record_stream(s)
                same = torch.equal(got, want)
            assert same
    cache.check_status()


def test_captured_steps_follow_the_lengths():
    """One graph of append and attention, replayed while the lengths on the device go on."""
    from pbs_attn_b200.decode import paged_attn_fwd, paged_kv_append
    D, ps, B = 128, 16, 2
    cache = make_cache(40, ps, 2, D, torch.bfloat16, 4, 64)
    table = make_table(cache, [100, 100])
    lens, x = ints(1, 60), torch.zeros(B, 2, 1, D, dtype=torch.bfloat16, device="cuda")
    q = torch.randn(B, 8, 1, D, device="cuda").to(torch.bfloat16)
    g0 = torch.Generator(device="cuda").manual_seed(0)
    past = torch.randn(B, 2, 59, D, generator=g0, device="cuda").to(torch.bfloat16)
    paged_kv_append(cache, past, past, table, ints(0, 59), new_lens=ints(0, 59))
    paged_attn_fwd(q, cache, table, lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged_kv_append(cache, x, x, table, lens)
        out = paged_attn_fwd(q, cache, table, lens)
    for step in range(5):
        x.copy_(torch.randn(B, 2, 1, D, generator=g0, device="cuda"))
        g.replay()
        n = lens.tolist()
        assert_within(out, *attention(q, cache, table, n))
        lens += 1
    cache.check_status()
    torch.cuda.synchronize()
    del g


def test_long_offsets():
    """Pages behind 2^31 bytes of the pool."""
    from pbs_attn_b200.decode import paged_kv_append
    ps, H, D, n = 64, 8, 128, 150
    for bits, pages in ((4, 74000), (16, 34000)):
        cache = make_cache(pages, ps, H, D, torch.bfloat16, bits, 64)
        table = torch.tensor([[pages - 1, pages - 4000, 3]], dtype=torch.int32, device="cuda")
        g = torch.Generator(device="cuda").manual_seed(3)
        k, v = (torch.randn(1, H, n, D, generator=g, device="cuda").to(torch.bfloat16) for _ in "kv")
        paged_kv_append(cache, k, v, table, ints(n))
        _run(torch.randn(1, 16, 1, D, generator=g, device="cuda").to(torch.bfloat16), cache, table, [n])
        del cache


@pytest.mark.parametrize("bits,group", FORMATS)
def test_faults_leave_tokens_out_and_are_raised_later(bits, group):
    from pbs_attn_b200 import _cabi
    from pbs_attn_b200.decode import paged_attn_fwd
    q, cache, table = _case([40], bits=bits, group=group)
    short = paged_attn_fwd(q, cache, table[:, :2], ints(32))
    got = paged_attn_fwd(q, cache, table[:, :2], ints(40))               # 40 tokens, a table for 32
    with pytest.raises(_cabi.PbsError, match="longer than its row"):
        cache.check_status()
    assert torch.equal(got, short)
    hole = table.clone()
    hole[0, 2] = cache.num_pages
    got = paged_attn_fwd(q, cache, hole, ints(40))                       # tokens 32 .. 39 have no page
    torch.cuda.synchronize()
    with pytest.raises(_cabi.PbsError, match="outside the pool"):
        paged_attn_fwd(q, cache, table, ints(40))
    assert torch.equal(got, short)


def test_refusals():
    from pbs_attn_b200 import _cabi
    from pbs_attn_b200.decode import paged_attn_fwd
    q, cache, table = _case([40], Hq=8, Hkv=2)
    n = ints(40)
    for error, args, kw in (
            (TypeError, (q.half(), cache, table, n), {}), (TypeError, (q.cpu(), cache, table, n), {}),
            (ValueError, (q[:, :7], cache, table, n), {}), (ValueError, (q[..., :64], cache, table, n), {}),
            (ValueError, (q, cache, table, ints(40, 40)), {}), (TypeError, (q, cache, table.long(), n), {}),
            (ValueError, (q, cache, table, n), {"out": q[:, :4]}), (ValueError, (q, cache, table, n), {"out": q.half()}),
            (TypeError, (q, cache, table, n), {"new_lens": n.long()}),
            (_cabi.PbsError, (q, cache, table, n), {"out": q[:, :1].expand(1, 8, 1, 128)})):
        with pytest.raises(error):
            paged_attn_fwd(*args, **kw)
    assert paged_attn_fwd(q[:0], cache, table[:0], n[:0]).shape == (0, 8, 1, 128)
    cache.check_status()


def test_calls_that_overlap_on_streams():
    """Calls whose blocks wait for one another, under way on several streams at a time."""
    from pbs_attn_b200.decode import paged_attn_fwd
    cases = []
    for i, lens in enumerate(([20000], [5000, 300], [60000], [100, 9000, 40])):
        q, cache, table = _case(lens, 8, 2, 1, seed=i, ps=64)
        t = ints(*lens)
        cases.append((torch.cuda.Stream(), q, cache, table, t, paged_attn_fwd(q, cache, table, t)))
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(30):
        for i, (s, q, cache, table, t, _) in enumerate(cases):
            with torch.cuda.stream(s):
                got[i].append(paged_attn_fwd(q, cache, table, t))
    torch.cuda.synchronize()
    for g, c in zip(got, cases):
        c[2].check_status()
        assert all(torch.equal(x, c[5]) for x in g)


def test_a_wait_that_runs_out_is_reported():
    from pbs_attn_b200 import _cabi
    from pbs_attn_b200.decode import paged_attn_fwd
    q, cache, table = _case([5000], 8, 2, 1)
    want = paged_attn_fwd(q, cache, table, ints(5000))
    torch.cuda.synchronize()
    lib = _cabi.load()
    try:
        lib.pbs_debug_set_attn_wait(5_000_000, 1)              # 5 ms; the first block does not arrive
        paged_attn_fwd(q, cache, table, ints(5000))
        torch.cuda.synchronize()
    finally:
        lib.pbs_debug_set_attn_wait(0, 0)
    with pytest.raises(_cabi.PbsError, match="bounded wait"):
        paged_attn_fwd(q, cache, table, ints(5000))
    assert torch.equal(paged_attn_fwd(q, cache, table, ints(5000)), want)
    cache.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64])
def test_flat_attention_over_many_tokens_keeps_its_precision(dtype, group):
    """All tokens weigh about the same, and what they leave is the root of their number: errors that grow with the number would show.

    Rounding a result to its type is 0.42 unit of relative error in the mean square; in fp16 the weights' rounding, the same of 2^-11, acts
    on code - 8, about 3.3 steps of a range of 15 that covers 4.6 deviations (64 channels) of a value.  A quarter on top."""
    from pbs_attn_b200.decode import paged_attn_fwd, paged_kv_append
    B, H, n, D, ps = 16, 8, 20000, 128, 64
    cache = make_cache(B * -(-n // ps) + 2, ps, H, D, dtype, 4, group)
    lens = [n] * B
    table = make_table(cache, lens)
    g = torch.Generator(device="cuda").manual_seed(1)
    for b in range(B):
        k, v = (torch.randn(1, H, n, D, generator=g, device="cuda").to(dtype) for _ in "kv")
        paged_kv_append(cache, k, v, table[b:b + 1], ints(n))
    q = (torch.randn(B, 8, 1, D, generator=g, device="cuda") * 0.2).to(dtype)
    got = paged_attn_fwd(q, cache, table, ints(*lens)).double()
    want = torch.cat([attention(q[b:b + 1], cache, table[b:b + 1], [n])[0] for b in range(B)])
    rounding = 0.42 * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11)
    weights = 0.42 * 2.0 ** -11 * 3.3 * 4.6 / 15 if dtype == torch.float16 else 0.0
    assert (got - want).norm() / want.norm() <= 1.25 * (rounding ** 2 + weights ** 2) ** 0.5


def test_the_largest_batch():
    lens = [(7 * b) % 40 for b in range(4096)]
    lens[4000] = 3000
    q, cache, table = _case(lens, 2, 1, 1, 64)
    from pbs_attn_b200.decode import paged_attn_fwd
    got = paged_attn_fwd(q, cache, table, ints(*lens))
    cache.check_status()
    for b in (0, 1, 17, 2000, 4000, 4095):
        assert_within(got[b:b + 1], *attention(q[b:b + 1], cache, table[b:b + 1], [lens[b]]))


@pytest.mark.parametrize("bits,group", FORMATS)
def test_values_of_others_leave_a_row_its_bits(bits, group):
    """Other sequences' values, far larger ones among them, and other queries do not reach a row, lengths and sizes being the same."""
    from pbs_attn_b200.decode import paged_attn_fwd, paged_kv_append
    lens, D = [3000, 500, 70], 128
    q, cache, table = _case(lens, S=2, bits=bits, group=group)
    want = paged_attn_fwd(q, cache, table, ints(*lens))
    other = torch.randn(1, 2, 500, D, device="cuda").to(q.dtype) * 2.0 ** 20
    paged_kv_append(cache, other, other, table[1:2], ints(500))
    bad = q.clone(memory_format=torch.preserve_format)
    bad[1] *= 100
    bad[0, 3] *= 50
    got = paged_attn_fwd(bad, cache, table, ints(*lens))
    cache.check_status()
    rows = torch.arange(8, device="cuda") != 3
    assert torch.equal(got[0, rows], want[0, rows]) and torch.equal(got[2], want[2]) and not torch.equal(got[1], want[1])
