"""A paged cache of 8 bits with a scale for each block of tokens and head: writing, reading back and refusals."""
import math

import pytest
import torch

from paged_ref import assert_within, ints, make_table, pages_for, rope_tables
from paged_ref8 import append8, make_cache8, rotate, values8

pytestmark = pytest.mark.gpu


def _data(lens, S, heads, D, dtype, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = lambda h: (size * torch.randn(len(lens), S, h, D, generator=g, device="cuda")).to(dtype).transpose(1, 2)  # noqa: E731
    return x(heads), x(heads), x(2 * heads)


def _copies(cache):
    return {n: getattr(cache, n).clone() for n in ("k", "v", "k_params", "v_params")}


def _same(cache, want):
    """Every code and scale of the pool, those that nothing was to change among them."""
    for n, x in want.items():
        got = getattr(cache, n)
        assert torch.equal(got.isnan(), x.isnan()), n
        # (a block that a NaN has spoilt has no codes to speak of)
        bad = x.isnan() if x.dtype == torch.float32 else want[n + "_params"].isnan().repeat_interleave(cache.block_size, -1)[..., None]
        assert torch.equal(got.masked_fill(bad, 0), x.masked_fill(bad, 0)), n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("rope", [None, "positions", "rows"])
def test_append_and_gather(dtype, D, block, rope):
    from pbs_attn_b200.decode import paged_kv_append, paged_kv_gather
    H, S, ps = 3, 70, 64
    lens, new = [70, 200, 1, 0, 83, 66], [70, 37, 1, 0, 70, 2]
    cache = make_cache8(pages_for(lens, ps), ps, H, D, dtype, block, token_major=D == 64)
    table = make_table(cache, lens, seed=D + block)
    # what the sequences hold already
    before = [n - m for n, m in zip(lens, new)]
    k0, v0, _ = _data(lens, max(before), H, D, dtype, 1)
    paged_kv_append(cache, k0, v0, table, ints(*before), new_lens=ints(*before))
    want = _copies(cache)
    k, v, q = _data(lens, S, H, D, dtype, 2, 1.3)
    kw, kf = {}, k.float()
    if rope:
        cos, sin = rope_tables(300, D, dtype)
        pos = torch.stack([(n - m + torch.arange(S, device="cuda")).clamp(0, 299) for n, m in zip(lens, new)])
        c, s = cos[pos], sin[pos]                                              # (B, S, D)
        kf = rotate(kf, c.float()[:, None], s.float()[:, None])
        kw = dict(query_states=q, **(dict(cos=cos, sin=sin) if rope == "positions" else dict(cos=c, sin=s)))
    got_q = paged_kv_append(cache, k, v, table, ints(*lens), new_lens=ints(*new), **kw)
    append8(cache, want["k"], want["k_params"], kf, table, lens, new)
    append8(cache, want["v"], want["v_params"], v.float(), table, lens, new)
    _same(cache, want)
    if rope:
        qf = rotate(q.float(), c.float()[:, None], s.float()[:, None]).to(dtype)
        there = torch.arange(S, device="cuda") < ints(*new)[:, None]
        assert torch.equal(got_q, torch.where(there[:, None, :, None], qf, 0))
    else:
        assert got_q is None
    back = paged_kv_gather(cache, table, ints(*lens), 90)
    for got, codes, scales in zip(back, (cache.k, cache.v), (cache.k_params, cache.v_params)):
        assert got.shape == (len(lens), H, 90, D) and got.dtype == dtype
        for b, n in enumerate(lens):
            x = values8(cache, codes, scales, table, b, n)[0][:, max(0, n - 90):]
            assert torch.equal(got[b, :, 90 - x.shape[1]:], x.float().to(dtype)) and (got[b, :, :90 - x.shape[1]] == 0).all()
    # half a step of the scale, and of the type
    for got, x, codes, scales in zip(back, (kf, v.float()), (cache.k, cache.v), (cache.k_params, cache.v_params)):
        for b, (n, m) in enumerate(zip(lens, new)):
            if m:
                room = values8(cache, codes, scales, table, b, n)[1].max()
                assert ((got[b, :, 90 - m:].double() - x[b, :, :m].double()).abs() <= room / 254 * (1 + 2.0 ** -20) + room * 2.0 ** -8).all()
    cache.check_status()


@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_token_by_token(block, D):
    """Scales that grow with the tokens, blocks and pages that begin, drafts of several tokens and some that are taken back."""
    from pbs_attn_b200.decode import paged_kv_append
    H, ps, B = 2, 64, 3
    cache = make_cache8(12, ps, H, D, torch.bfloat16, block)
    table = torch.randperm(12, generator=torch.Generator().manual_seed(3)).int().view(B, 4).cuda()
    want = _copies(cache)
    lens = [0, 30, 61]
    k, v, _ = _data(lens, 61, H, D, torch.bfloat16, 4)
    calls = [(lens, lens, k, v)]
    for i in range(90):
        S = 1 if i % 3 else 4
        new = [S, S, min(S, 1 + i % 4)]
        lens = [n + m for n, m in zip(lens, new)]
        k, v, _ = _data(lens, S, H, D, torch.bfloat16, 100 + i, 1.0 + i % 7 / 4)
        calls.append((lens, new, k, v))
        if i % 9 == 3:                                     # the last tokens were wrong
            lens = [n - m for n, m in zip(lens, new)]
    for lens, new, k, v in calls:
        paged_kv_append(cache, k, v, table, ints(*lens), new_lens=ints(*new))
        append8(cache, want["k"], want["k_params"], k.float(), table, lens, new)
        append8(cache, want["v"], want["v_params"], v.float(), table, lens, new)
    _same(cache, want)
    cache.check_status()


def test_a_tokens_error_stays_below_a_step():
    """Each growth of the scale rounds anew, by half of a step of then: over a block whose scale doubles these come to less than a step."""
    from pbs_attn_b200.decode import paged_kv_append, paged_kv_gather
    cache = make_cache8(1, 16, 1, 64, torch.float16, 16)
    x = torch.randn(16, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)) * 2.0 ** torch.arange(-8, 8, device="cuda")[:, None]
    x = x.half()
    for n in range(1, 17):
        row = x[n - 1].view(1, 1, 1, 64)
        paged_kv_append(cache, row, row, ints(0)[None], ints(n))
    k, _ = paged_kv_gather(cache, ints(0)[None], ints(16), 16)
    step = cache.k_params[0, 0, 0].double()
    # (the steps before are no more than the last; of the eleven bits of fp16 half a unit comes on top)
    assert ((k[0, 0].double() - x.double()).abs() <= step * 1.5 + x.double().abs() * 2.0 ** -11).all()


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_is_not_finite_spoils_its_block_and_head_alone(D, bad):
    from pbs_attn_b200.decode import paged_kv_append, paged_kv_gather
    cache = make_cache8(4, 32, 2, D, torch.bfloat16, 16)
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    k, v, _ = _data([70], 70, 2, D, torch.bfloat16, 6)
    k, v = k.clone(), v.clone()
    k[0, 1, 20, D - 3] = bad
    v[0, 0, 69, 0] = bad
    paged_kv_append(cache, k, v, table, ints(70))
    gk, gv = paged_kv_gather(cache, table, ints(70), 70)
    nan = torch.zeros_like(gk, dtype=torch.bool)
    nan[0, 1, 16:32] = True
    assert torch.equal(gk.isnan(), nan)
    nan.zero_()[0, 0, 64:70] = True
    assert torch.equal(gv.isnan(), nan)
    # it stays so with tokens that come after, and goes with the block
    paged_kv_append(cache, k[:, :, :1], v[:, :, :1], table, ints(71))
    gk, gv = paged_kv_gather(cache, table, ints(71), 7)
    assert gv[0, 0].isnan().all() and not gv[0, 1].isnan().any() and not gk.isnan().any()
    paged_kv_append(cache, k[:, :, :6], v[:, :, :6], table, ints(70))
    assert not paged_kv_gather(cache, table, ints(70), 6)[1].isnan().any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [0.0, 2.0 ** -133, 2.0 ** -121, 2.0 ** -24, 65504.0, 3e38])
def test_sizes_of_values(dtype, size):
    from pbs_attn_b200.decode import paged_kv_append, paged_kv_gather
    if dtype == torch.float16 and (size > 65504 or 0 < size < 2.0 ** -24):
        size = 1.0
    cache = make_cache8(1, 16, 1, 128, dtype, 16)
    want = _copies(cache)
    x = (torch.linspace(-1, 1, 16 * 128, device="cuda", dtype=torch.float64) * size).to(dtype).view(1, 1, 16, 128)
    for a, b in ((0, 9), (9, 16)):
        paged_kv_append(cache, x[:, :, a:b], x[:, :, a:b], ints(0)[None], ints(b))
        append8(cache, want["k"], want["k_params"], x[:, :, a:b].float(), ints(0)[None], [b], [b - a])
        append8(cache, want["v"], want["v_params"], x[:, :, a:b].float(), ints(0)[None], [b], [b - a])
    _same(cache, want)
    k, v = paged_kv_gather(cache, ints(0)[None], ints(16), 16)
    assert k.isfinite().all() and torch.equal(k, v)


def test_rotated_keys_beyond_fp16_stay_finite():
    from pbs_attn_b200.decode import paged_kv_append, paged_kv_gather
    cache = make_cache8(1, 16, 1, 64, torch.float16, 16)
    k = torch.full((1, 1, 2, 64), 65504.0, dtype=torch.float16, device="cuda")
    cos = torch.full((2, 64), 0.75, dtype=torch.float16, device="cuda")
    paged_kv_append(cache, k, k, ints(0)[None], ints(2), cos=cos, sin=cos)
    got = paged_kv_gather(cache, ints(0)[None], ints(2), 2)[0]
    assert (got[..., 32:] == 65504).all() and (got[..., :32] == 0).all()


def test_strides_batches_and_many_heads():
    from pbs_attn_b200.decode import paged_kv_append
    B, H, S, D, ps = 40, 5, 3, 128, 16
    lens = [3 + 7 * b % 60 for b in range(B)]
    for token_major in (False, True):
        cache = make_cache8(pages_for(lens, ps), ps, H, D, torch.bfloat16, 16, token_major)
        table = make_table(cache, lens, 1)
        before = [n - S for n in lens]
        k0, v0, _ = _data(lens, max(before), H, D, torch.bfloat16, 7)
        paged_kv_append(cache, k0.contiguous(), v0, table, ints(*before), new_lens=ints(*before))
        want = _copies(cache)
        k, v, _ = _data(lens, S, H, D, torch.bfloat16, 8)
        odd = torch.zeros(B, H, S, D + 1, dtype=torch.bfloat16, device="cuda")[..., 1:]
        odd.copy_(k)
        one = v[:, :1].expand(B, H, S, D)                  # (heads that share their memory)
        paged_kv_append(cache, odd, one, table, ints(*lens))
        append8(cache, want["k"], want["k_params"], k.float(), table, lens, [S] * B)
        append8(cache, want["v"], want["v_params"], one.float(), table, lens, [S] * B)
        _same(cache, want)


def test_faults_leave_tokens_out_and_raise():
    from pbs_attn_b200 import _cabi
    from pbs_attn_b200.decode import paged_kv_append, paged_kv_gather
    cache = make_cache8(3, 16, 2, 64, torch.bfloat16, 16)
    k, v, _ = _data([40], 40, 2, 64, torch.bfloat16, 9)
    before = _copies(cache)
    paged_kv_append(cache, k, v, ints(1, 7, -2)[None], ints(40))             # pages 7 and -2 are not there
    with pytest.raises(_cabi.PbsError, match="outside the pool"):
        cache.check_status()
    for n in before:                                       # page 1 alone was written
        for p in (0, 2):
            assert torch.equal(getattr(cache, n)[p].nan_to_num(7), before[n][p].nan_to_num(7))
    assert not cache.k_params[1].isnan().any()
    paged_kv_append(cache, k, v, ints(0)[None], ints(40))                    # a row of the table that ends
    with pytest.raises(_cabi.PbsError, match="longer than its row"):
        cache.check_status()
    cos, sin = rope_tables(20, 64, torch.bfloat16)
    cache = make_cache8(3, 16, 2, 64, torch.bfloat16, 16)
    want = _copies(cache)
    paged_kv_append(cache, k, v, ints(0, 1, 2)[None], ints(40), cos=cos, sin=sin)
    with pytest.raises(_cabi.PbsError, match="behind the rotary tables"):
        cache.check_status()
    append8(cache, want["v"], want["v_params"], v[:, :, :20].float(), ints(0, 1, 2)[None], [20], [20])
    append8(cache, want["k"], want["k_params"], rotate(k[:, :, :20].float(), cos.float(), sin.float()), ints(0, 1, 2)[None], [20], [20])
    _same(cache, want)
    with pytest.raises(_cabi.PbsError, match="outside the pool"):
        got = paged_kv_gather(cache, ints(0, 9)[None], ints(20), 20)
        assert (got[0][:, :, 16:] == 0).all() and not got[0][:, :, :16].isnan().any()
        cache.check_status()


def test_captured_with_lengths_that_change():
    from pbs_attn_b200.decode import paged_kv_append
    cache = make_cache8(8, 16, 2, 128, torch.bfloat16, 16)
    table, lens = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4), ints(14, 20)
    k0, v0, _ = _data([14, 20], 20, 2, 128, torch.bfloat16, 10)
    paged_kv_append(cache, k0, v0, table, lens, new_lens=lens)
    want = _copies(cache)
    k, v, _ = _data([1, 1], 1, 2, 128, torch.bfloat16, 11)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens += 1
        k.mul_(1.5)
        paged_kv_append(cache, k, v, table, lens)
    for i in range(6):
        now = (k.float() * 1.5).to(torch.bfloat16)
        graph.replay()
        k_now = k.clone()
        assert torch.equal(k_now, now)
        append8(cache, want["k"], want["k_params"], k_now.float(), table, [15 + i, 21 + i], [1, 1])
        append8(cache, want["v"], want["v_params"], v.float(), table, [15 + i, 21 + i], [1, 1])
    _same(cache, want)


def test_the_constructor():
    from pbs_attn_b200 import _cabi
    from pbs_attn_b200.decode import PagedKVCache
    cache = PagedKVCache(3, 64, 2, 128, torch.float16, "cuda", bits=8, block_size=32)
    assert cache.k.dtype == torch.int8 and cache.k.shape == (3, 2, 64, 128) and cache.k_params.shape == (3, 2, 2) and cache.dtype == torch.float16
    assert cache.bits == 8 and cache.block_size == 32
    for kw in (dict(block_size=None), dict(block_size=24), dict(block_size=0), dict(block_size=128)):
        with pytest.raises(ValueError):
            PagedKVCache(3, 64, 2, 128, bits=8, **kw)
    for kw in (dict(block_size=8), dict(block_size=128, page_size=256), dict(block_size=32, head_dim=96)):
        with pytest.raises(_cabi.PbsError):
            PagedKVCache(**{**dict(num_pages=2, page_size=64, kv_heads=2, head_dim=64, bits=8), **kw})
    k, s = torch.zeros(2, 2, 32, 64, dtype=torch.int8, device="cuda"), torch.zeros(2, 2, 2, device="cuda")
    bf = torch.bfloat16
    for error, args, dt in ((ValueError, (k, k), bf), (ValueError, (k, k, s, s), None), (TypeError, (k, k, s, s), torch.float32), (TypeError, (k, k, s.half(), s.half()), bf),
                            (ValueError, (k, k, s[:, :, :, None], s[:, :, :, None]), bf), (ValueError, (k, k, s[:1], s[:1]), bf), (ValueError, (k, k, s, s[:, :, :1]), bf),
                            (TypeError, (k.half(), k.half()), bf)):
        with pytest.raises(error):
            PagedKVCache.from_tensors(*args, dtype=dt)


def test_gather_within_the_rounding_of_the_type():
    """A code times its scale in 32 bits, rounded once more: at most half a unit of either."""
    from pbs_attn_b200.decode import paged_kv_append, paged_kv_gather
    cache = make_cache8(2, 16, 2, 128, torch.bfloat16, 16)
    k, v, _ = _data([20], 20, 2, 128, torch.bfloat16, 12)
    paged_kv_append(cache, k, v, ints(1, 0)[None], ints(20))
    got = paged_kv_gather(cache, ints(1, 0)[None], ints(20), 20)[0][0]
    want = values8(cache, cache.k, cache.k_params, ints(1, 0)[None], 0, 20)[0]
    assert_within(got, want, want.abs() * (2.0 ** -8 + 2.0 ** -23) + 2.0 ** -134)


def _guarded(pages, page_size, heads, dim, dtype, block, seed):
    """A cache of codes and scales that are all different, and finite, inside of memory that is none of its own on every side."""
    from pbs_attn_b200.decode import PagedKVCache
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = [torch.randint(-127, 128, (pages + 2, heads + 2, page_size + 2, dim + 32), generator=g, device="cuda", dtype=torch.int8) for _ in "kv"]
    scales = [torch.rand(pages + 2, heads + 2, page_size // block + 2, generator=g, device="cuda") / 8 for _ in "kv"]
    inside = lambda memory: ([t[1:-1, 1:-1, 1:-1, 16:-16] for t in memory[:2]] + [t[1:-1, 1:-1, 1:-1] for t in memory[2:]])  # noqa: E731
    return PagedKVCache.from_tensors(*inside(codes + scales), dtype=dtype), codes + scales, inside


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ps,block", [(16, 16), (64, 16), (64, 32), (64, 64), (128, 64)])
@pytest.mark.parametrize("S", [1, 4, 5, 16, 17, 70])
def test_nothing_beside_a_calls_tokens_changes(dtype, D, ps, block, S):
    """Codes and scales of every page, block and head, and of the memory around them, are known and compared, those that no call comes to among them."""
    from pbs_attn_b200.decode import paged_kv_append
    H = 3
    starts = [0, 1, block - 1, block, ps - 1, ps, 2 * ps + 3]
    new = [S, 0, S, max(1, S // 2), S, 1, S]
    lens = [a + m for a, m in zip(starts, new)]
    cache, memory, inside = _guarded(pages_for(lens, ps), ps, H, D, dtype, block, S + D)
    want = [t.clone() for t in memory]
    wk, wv, wks, wvs = inside(want)
    table = make_table(cache, lens, S)
    cos, sin = rope_tables(max(lens), D, dtype)
    k, v, q = _data(lens, S, H, D, dtype, S, 2.0)
    room = torch.full((len(lens), S + 2, 2 * H + 2, D), 7.0, dtype=dtype, device="cuda")
    out = room[:, 1:-1, 1:-1].transpose(1, 2)
    paged_kv_append(cache, k, v, table, ints(*lens), new_lens=ints(*new), cos=cos, sin=sin, query_states=q, query_out=out)
    cache.check_status()
    pos = torch.stack([(a + torch.arange(S, device="cuda")).clamp(max=max(lens) - 1) for a in starts])
    c, s = cos[pos].float()[:, None], sin[pos].float()[:, None]
    append8(cache, wk, wks, rotate(k.float(), c, s), table, lens, new)
    append8(cache, wv, wvs, v.float(), table, lens, new)
    for got, x in zip(memory, want):
        assert torch.equal(got, x)
    there = torch.arange(S, device="cuda") < ints(*new)[:, None]
    assert torch.equal(out, torch.where(there[:, None, :, None], rotate(q.float(), c, s).to(dtype), 0))
    out.fill_(7.0)
    assert (room == 7).all()


@pytest.mark.parametrize("growth", [1.0, 1.25, 1.5, 2.0, 3.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_tokens_error_is_half_of_each_step_that_it_was_rounded_to(dtype, growth):
    """A token is off by half a step when it is written, and by half a step of then each time that its block's scale grows, no more.  Reciprocals and
    ratios that codes up to 127 are multiplied by are rounded: 127 * 2^-24 of a step each time, taken as 2^-16.  Where the scale doubles with every
    token these halves come to less than one step of the last."""
    from pbs_attn_b200.decode import paged_kv_append
    H, D, n = 4, 256, 16 if growth <= 2 else 7             # (3^6 is a number of eight bits times a power of 2, to within the type's rounding)
    cache = make_cache8(1, 16, H, D, dtype, 16)
    g = torch.Generator(device="cuda").manual_seed(int(growth * 8))
    x = torch.rand(H, n, D, generator=g, device="cuda") * 2 - 1
    x[..., 7] = 1.0
    x = (x * (2.0 ** -6 * growth ** torch.arange(n, device="cuda", dtype=torch.float64))[:, None]).to(dtype)
    steps = torch.zeros(H, n, dtype=torch.float64, device="cuda")
    off = torch.zeros(H, n, dtype=torch.float64, device="cuda")                   # what each token may be off by
    for t in range(n):
        row = x[:, t][None, :, None]
        paged_kv_append(cache, row, row, ints(0)[None], ints(t + 1))
        steps[:, t] = cache.k_params[0, :, 0].double()
        grown = torch.ones(H, dtype=torch.bool, device="cuda") if t == 0 else steps[:, t] > steps[:, t - 1]
        off[:, :t] += torch.where(grown, steps[:, t], 0)[:, None] * (0.5 + 2.0 ** -16)
        off[:, t] += steps[:, t] * (0.5 + 2.0 ** -16)
    for codes, scales in ((cache.k, cache.k_params), (cache.v, cache.v_params)):
        held = values8(cache, codes, scales, ints(0)[None], 0, n)[0]
        assert ((held - x.double()).abs() <= off[..., None]).all()
    if growth == 2.0:
        assert (off < steps[:, -1:] * (1 + 2.0 ** -12)).all()
