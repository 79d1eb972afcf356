"""New keys and values into a paged cache and back, against the formulas in 64 bits."""
import math

import pytest
import torch

from paged_ref import TINY, UNIT, ints, make_cache, make_table, pages_for, rope_tables, rotate

pytestmark = pytest.mark.gpu


def _inputs(B, H, S, D, dtype, seed, major="token"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if major == "token":                                   # what a projection hands over
        return torch.randn(B, S, H, D, generator=g, device="cuda").to(dtype).transpose(1, 2)
    if major == "shared":                                  # one head for all
        return torch.randn(B, 1, S, D, generator=g, device="cuda").to(dtype).expand(B, H, S, D)
    if major == "odd":                                     # rows that the kernel cannot read in place
        return torch.randn(B, H, S, D + 3, generator=g, device="cuda").to(dtype)[..., 1:D + 1]
    return torch.randn(B, H, S, D, generator=g, device="cuda").to(dtype)


def _append(cache, k, v, table, lens, **kw):
    from pbs_attn_b200.decode import paged_kv_append
    got = paged_kv_append(cache, k, v, table, lens, **kw)
    cache.check_status()
    return got


def _gather(cache, table, lens, count, **kw):
    from pbs_attn_b200.decode import paged_kv_gather
    got = paged_kv_gather(cache, table, lens, count, **kw)
    cache.check_status()
    return got


def _quantised(x, group, dtype):
    """The definition in 32 bits, operation by operation: the values that (..., D) stands for."""
    y = x.float().unflatten(-1, (-1, group))
    low, high = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    step = ((high * 0.5 - low * 0.5) * (2 / 15)).to(dtype).float()
    low = low.to(dtype).float()
    codes = ((y - low) * torch.where(step > 0, 1 / step, 0.0)).round().clamp(0, 15)
    return (codes * step + low).flatten(-2).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits,group", [(16, 0), (4, 32), (4, 64)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rope", [None, "positions", "tokens", "shared"])
def test_append_and_gather(dtype, bits, group, D, rope):
    B, H, Hq, S, ps = 3, 2, 6, 7, 16
    lens, new = [7, 40, 129], [7, 3, 5]
    cache = make_cache(pages_for(lens, ps), ps, H, D, dtype, bits, group, token_major=D == 64)
    table = make_table(cache, lens)
    major = {None: "head", "positions": "token", "tokens": "odd", "shared": "shared"}[rope]
    q, k, v = (_inputs(B, h, S, D, dtype, i, major) for i, h in ((1, Hq), (2, H), (3, H)))
    at = (torch.tensor(lens) - torch.tensor(new))[:, None] + torch.arange(S)
    cos = sin = None
    tc, ts = rope_tables(140, D, dtype)
    if rope:
        cos, sin = (tc, ts) if rope == "positions" else (tc[at.cuda()], ts[at.cuda()]) if rope == "tokens" else (tc[5:5 + S][None], ts[5:5 + S][None])
    got_q = _append(cache, k, v, table, ints(*lens), new_lens=ints(*new), cos=cos, sin=sin, query_states=q if rope else None)
    back = _gather(cache, table, ints(*lens), S, new_lens=ints(*new))
    fresh = (torch.arange(S) < torch.tensor(new)[:, None]).cuda()[:, None, :, None]
    c, s = (None, None) if not rope else (t[at.cuda()][:, None] for t in (tc, ts)) if rope == "positions" else (t[:, None] for t in (cos, sin))
    unit, tiny = UNIT[dtype], TINY[dtype]

    def check(got, x, turned, quantised):
        want = rotate(x.double(), c.double(), s.double()) if turned else x.double()
        size = x.double().abs() * c.double().abs() + rotate(x.double().abs(), torch.zeros_like(c).double(), s.double().abs()).abs() if turned else want.abs()
        off = (got.double() - want).abs()
        # two products and a sum in 32 bits, then one rounding
        bound = unit * want.abs() + tiny + 2.0 ** -22 * size
        if quantised:
            y = want.unflatten(-1, (-1, group))
            low, high = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
            step = (high - low) / 15 * (1 + 2 * unit) + tiny
            # half a step; or, where the code is cut off, what step and minimum were rounded by
            cut = unit * low.abs() + tiny + 15 * ((high - low) / 15 * unit + tiny)
            bound = bound + (torch.maximum(step / 2 * (1 + 2.0 ** -20), cut)).expand_as(y).flatten(-2)
            assert torch.equal(torch.where(fresh, _quantised(rotate(x.float(), c.float(), s.float()) if turned else x, group, dtype), 0.0), got)
        assert (off <= bound)[fresh.expand_as(off)].all()
        assert (got[~fresh.expand_as(got)] == 0).all()

    check(back[0], k, bool(rope), bits == 4)
    check(back[1], v, False, bits == 4)
    if rope:
        check(got_q, q, True, False)
    else:
        assert got_q is None


@pytest.mark.parametrize("bits", [16, 4])
def test_nothing_else_is_written(bits):
    ps, H, D = 32, 2, 128
    lens = [33, 64]
    cache = make_cache(6, ps, H, D, torch.bfloat16, bits, 64)
    table = make_table(cache, lens)
    pools = [t for t in (cache.k, cache.v, cache.k_params, cache.v_params) if t is not None]
    for t in pools:
        t.zero_()
    k = torch.ones(2, H, 2, D, device="cuda", dtype=torch.bfloat16) * 3
    k[..., ::2] = -2
    _append(cache, k, k, table, ints(*lens))
    touched = torch.zeros(6, ps, dtype=torch.bool)
    for b, n in enumerate(lens):
        for p in (n - 2, n - 1):
            touched[int(table[b, p // ps]), p % ps] = True
    for t in pools:
        nz = (t != 0).flatten(3).any(-1).any(1).cpu()
        assert torch.equal(nz, touched)


def test_one_token_at_a_time_is_all_at_once():
    ps, H, D, n = 16, 3, 64, 37
    k, v = _inputs(1, H, n, D, torch.float16, 5), _inputs(1, H, n, D, torch.float16, 6)
    a, b = (make_cache(4, ps, H, D, torch.float16, 4, 32) for _ in "ab")
    table = make_table(a, [n])
    cos, sin = rope_tables(n, D, torch.float16)
    _append(a, k, v, table, ints(n), cos=cos, sin=sin)
    for i in range(n):
        _append(b, k[:, :, i:i + 1], v[:, :, i:i + 1], table, ints(i + 1), cos=cos, sin=sin)
    for x, y in zip(_gather(a, table, ints(n), n), _gather(b, table, ints(n), n)):
        assert torch.equal(x, y)


def test_queries_rotated_in_place_and_into_a_given_tensor():
    ps, H, D = 16, 2, 128
    cache = make_cache(3, ps, H, D, torch.bfloat16, 4, 64)
    table = make_table(cache, [20])
    cos, sin = rope_tables(32, D, torch.bfloat16)
    q, k = _inputs(1, 4, 3, D, torch.bfloat16, 1), _inputs(1, H, 3, D, torch.bfloat16, 2)
    want = _append(cache, k, k, table, ints(20), cos=cos, sin=sin, query_states=q)
    wide = torch.zeros(1, 4, 3, D + 1, dtype=torch.bfloat16, device="cuda")[..., 1:]    # rows that the kernel cannot write
    assert _append(cache, k, k, table, ints(20), cos=cos, sin=sin, query_states=q, query_out=wide) is wide and torch.equal(wide, want)
    assert _append(cache, k, k, table, ints(20), cos=cos, sin=sin, query_states=q, query_out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("rope", [True, False])
def test_a_place_for_queries_that_are_not_given_is_refused(rope):
    """It would come back as it was."""
    from pbs_attn_b200.decode import paged_kv_append
    cache = make_cache(3, 16, 2, 128, torch.bfloat16, 4, 64)
    table = make_table(cache, [20])
    k = _inputs(1, 2, 3, 128, torch.bfloat16, 2)
    cos, sin = rope_tables(32, 128, torch.bfloat16) if rope else (None, None)
    with pytest.raises(ValueError, match="query_out"):
        paged_kv_append(cache, k, k, table, ints(20), cos=cos, sin=sin, query_out=torch.zeros(1, 4, 3, 128, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_group_that_is_not_finite_reads_back_as_nan(value, dtype):
    ps, H, D, G = 16, 1, 128, 32
    cache = make_cache(2, ps, H, D, dtype, 4, G)
    table = make_table(cache, [4])
    k = _inputs(1, H, 4, D, dtype, 1, "head").clone()
    k[0, 0, 2, 40] = value
    _append(cache, k, k, table, ints(4))
    for x in _gather(cache, table, ints(4), 4):
        nan = torch.zeros(1, H, 4, D, dtype=torch.bool, device="cuda")
        nan[0, 0, 2, 32:64] = True
        assert torch.equal(x.isnan(), nan)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_groups_without_range_and_at_the_ends_of_the_type(dtype):
    ps, D, G = 16, 64, 32
    cache = make_cache(2, ps, 1, D, dtype, 4, G)
    table = make_table(cache, [6])
    big = torch.finfo(dtype).max
    k = torch.zeros(1, 1, 6, D, dtype=dtype, device="cuda")
    k[0, 0, 1] = -1.7
    k[0, 0, 2, :G:2], k[0, 0, 2, 1:G:2] = big, -big          # a range that the type does not hold
    k[0, 0, 3] = torch.finfo(dtype).smallest_normal
    k[0, 0, 4, 0] = torch.finfo(dtype).smallest_normal
    k[0, 0, 5] = big
    _append(cache, k, k, table, ints(6))
    x = _gather(cache, table, ints(6), 6)[0]
    assert x.isfinite().all()
    for row in (0, 1, 3, 5):
        assert torch.equal(x[0, 0, row], k[0, 0, row])
    # a step of the whole range, and what rounding it and the minimum costs
    assert ((x - k).double().abs()[0, 0, 2, :G] <= 2.0 * big / 15 / 2 + 2 * big * UNIT[dtype] * 2).all()
    assert ((x - k).double().abs()[0, 0, 4] <= torch.finfo(dtype).smallest_normal).all()


def test_keys_that_the_rotation_makes_larger_than_the_type():
    cache = make_cache(2, 16, 1, 64, torch.float16, 4, 32)
    table = make_table(cache, [1])
    k = torch.full((1, 1, 1, 64), 65504.0, dtype=torch.float16, device="cuda")
    h = torch.full((1, 1, 64), 0.7071, dtype=torch.float16, device="cuda")
    _append(cache, k, k, table, ints(1), cos=h, sin=h)
    x = _gather(cache, table, ints(1), 1)[0]
    assert (x[..., 32:] == 65504).all() and (x[..., :32].abs() <= 65504 * 2 ** -10).all()


def test_tokens_left_out():
    """Length 0, fewer tokens than rows, new_lens outside their range: nothing written, no fault."""
    ps, H, D = 16, 1, 64
    cache = make_cache(4, ps, H, D, torch.bfloat16, 16, 0)
    cache.k.zero_(), cache.v.zero_()
    table = torch.full((3, 1), -1, dtype=torch.int32, device="cuda")
    table[1, 0] = 2
    k = torch.ones(3, H, 4, D, dtype=torch.bfloat16, device="cuda")
    cos, sin = rope_tables(16, D, torch.bfloat16)
    q = _append(cache, k, k, table, ints(0, 2, 5), new_lens=ints(4, 9, -3), cos=cos, sin=sin, query_states=k)
    assert (cache.k != 0).flatten(3).any(-1).sum() == 2 and (cache.k[2, 0, :2] != 0).any(-1).all()
    assert (q[0] == 0).all() and (q[1, :, :2] == 0).all() and (q[1, :, 2:] != 0).any() and (q[2] == 0).all()


@pytest.mark.parametrize("table,length,rows,message", [
    ([[9]], 5, 32, "outside the pool"), ([[-1]], 5, 32, "outside the pool"), ([[0]], 40, 64, "longer than its row"), ([[0, 1]], 20, 16, "rotary")])
def test_faults_are_found_and_raised_later(table, length, rows, message):
    from pbs_attn_b200 import _cabi
    from pbs_attn_b200.decode import paged_kv_append, paged_kv_gather
    ps, H, D = 16, 1, 64
    cache = make_cache(2, ps, H, D, torch.bfloat16, 4, 64)
    for t in (cache.k, cache.v, cache.k_params, cache.v_params):
        t.zero_()
    k = torch.ones(1, H, 1, D, dtype=torch.bfloat16, device="cuda")
    cos, sin = rope_tables(rows, D, torch.bfloat16)
    table = torch.tensor(table, dtype=torch.int32, device="cuda")
    paged_kv_append(cache, k, k, table, ints(length), cos=cos, sin=sin)
    torch.cuda.synchronize()
    assert (cache.k_params[:, :, :, :, 1] == 0).all() or message == "rotary"
    with pytest.raises(_cabi.PbsError, match=message):
        paged_kv_append(cache, k, k, table, ints(length), cos=cos, sin=sin)
    cache.check_status()                                   # told once
    if message != "rotary":
        got = paged_kv_gather(cache, table, ints(length), 1)[0]
        with pytest.raises(_cabi.PbsError, match=message):
            cache.check_status()
        assert (got == 0).all()


def test_pages_behind_2_to_the_31_bytes():
    ps, H, D = 64, 8, 128
    cache = make_cache(74000, ps, H, D, torch.bfloat16, 4, 64)       # 2.4 GB of codes for keys
    table = torch.tensor([[73999, 70001, 3]], dtype=torch.int32, device="cuda")
    k, v = _inputs(1, H, 150, D, torch.bfloat16, 1), _inputs(1, H, 150, D, torch.bfloat16, 2)
    _append(cache, k, v, table, ints(150))
    for x, y in zip(_gather(cache, table, ints(150), 150), (k, v)):
        assert torch.equal(x, _quantised(y, 64, torch.bfloat16))


def test_refusals():
    from pbs_attn_b200 import _cabi
    from pbs_attn_b200.decode import PagedKVCache, paged_kv_append, paged_kv_gather
    cache = make_cache(2, 16, 2, 64, torch.bfloat16, 4, 32)
    k = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16, device="cuda")
    table, lens = ints(0)[None], ints(1)
    cos, sin = rope_tables(16, 64, torch.bfloat16)
    for error, args, kw in (
            (TypeError, (k.half(), k, table, lens), {}), (TypeError, (k.cpu(), k, table, lens), {}),
            (TypeError, (k, k, table.long(), lens), {}), (TypeError, (k, k, table, lens.cpu()), {}),
            (ValueError, (k, k[:, :1], table, lens), {}), (ValueError, (k[..., :32], k[..., :32], table, lens), {}),
            (ValueError, (k, k, table, ints(1, 1)), {}), (ValueError, (k, k, table[0], lens), {}),
            (ValueError, (k, k, table, lens), {"cos": cos}), (ValueError, (k, k, table, lens), {"query_states": k}),
            (ValueError, (k, k, table, lens), {"cos": cos[:, :32], "sin": sin[:, :32]}),
            (TypeError, (k, k, table, lens), {"cos": cos.float(), "sin": sin.float()}),
            (ValueError, (k, k, table, lens), {"cos": cos[:0], "sin": sin[:0]}),
            (ValueError, (k, k, table, lens), {"cos": cos, "sin": sin, "query_states": k[:, :, :, :32]}),
            (ValueError, (k, k, table, lens), {"cos": cos, "sin": sin, "query_states": torch.cat([k, k[:, :1]], 1)}),
            (ValueError, (k, k, table, lens), {"cos": cos, "sin": sin, "query_states": k, "query_out": k[:, :1]}),
            (TypeError, (k, k, table, lens), {"new_lens": lens.long()})):
        with pytest.raises(error):
            paged_kv_append(cache, *args, **kw)
    with pytest.raises(ValueError):
        paged_kv_gather(cache, table, ints(1, 1), 1)
    for kw in (dict(head_dim=96), dict(page_size=24), dict(page_size=8), dict(bits=4, group_size=128, head_dim=128), dict(kv_heads=0)):
        with pytest.raises(_cabi.PbsError):
            PagedKVCache(**{**dict(num_pages=2, page_size=16, kv_heads=2, head_dim=64, device="cuda"), **kw})
    with pytest.raises(ValueError):
        PagedKVCache(2, 16, 2, 64, bits=8)
    with pytest.raises(TypeError):
        PagedKVCache(2, 16, 2, 64, dtype=torch.float32)
    with pytest.raises(RuntimeError):
        PagedKVCache(2, 16, 2, 64, device="cpu")
    with pytest.raises(_cabi.PbsError, match="16 bytes"):
        PagedKVCache.from_tensors(*(torch.zeros(2, 2, 16, 65, dtype=torch.bfloat16, device="cuda")[..., :64] for _ in "kv"))
    torch.cuda.synchronize()
    cache.check_status()


def test_no_tokens_at_all():
    from pbs_attn_b200.decode import paged_kv_append, paged_kv_gather
    cache = make_cache(2, 16, 2, 64, torch.bfloat16, 16, 0)
    k = torch.zeros(0, 2, 1, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(0, 1, dtype=torch.int32, device="cuda")
    assert paged_kv_append(cache, k, k, table, table[:, 0]) is None
    assert paged_kv_gather(cache, table, table[:, 0], 3)[0].shape == (0, 2, 3, 64)
    assert paged_kv_gather(cache, ints(0)[None], ints(1), 0)[0].shape == (1, 2, 0, 64)
