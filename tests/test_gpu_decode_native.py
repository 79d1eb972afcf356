"""The calls of decode.py and logits.py without Python in between: same bits as with it, and back to Python for what they do not cover."""
import pytest
import torch

from paged_ref import ints, make_cache, make_table, rope_tables

pytestmark = pytest.mark.gpu


def _case(bits=4):
    g = torch.Generator(device="cuda").manual_seed(bits)
    x = lambda h, s=3: torch.randn(2, s, h, 128, generator=g, device="cuda").to(torch.bfloat16).transpose(1, 2)  # noqa: E731
    cache = make_cache(20, 16, 2, 128, torch.bfloat16, bits, 64)
    return cache, make_table(cache, [100, 40]), ints(100, 40), x(8), x(2), x(2)


def _ran_natively(cache, monkeypatch):
    """Makes the Python code fail: what returns ran without it."""
    from pbs_attn_b200 import decode
    assert cache._native is not None

    def fail(*a):
        raise AssertionError("went through Python")

    monkeypatch.setattr(decode, "_batch", fail)
    monkeypatch.setattr(decode, "_check_rows", fail)


@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("tables", ["positions", "tokens", "shared"])
def test_same_bits_as_through_python(bits, tables, monkeypatch):
    from pbs_attn_b200.decode import paged_attn_fwd, paged_kv_append, paged_kv_gather
    cache, table, lens, q, k, v = _case(bits)
    cos, sin = rope_tables(128, 128, torch.bfloat16)
    if tables != "positions":
        cos, sin = (t[:3].expand(2 if tables == "tokens" else 1, 3, 128).contiguous() for t in (cos, sin))
    past = torch.randn(2, 2, 100, 128, device="cuda").to(torch.bfloat16)
    new = ints(3, 2)

    def step():
        paged_kv_append(cache, past, past, table, lens, new_lens=lens)
        r = paged_kv_append(cache, k, v, table, lens, new_lens=new, cos=cos, sin=sin, query_states=q)
        assert paged_kv_append(cache, k, v, table, lens, new_lens=new, cos=cos, sin=sin) is None
        into = torch.empty_like(r)
        assert paged_attn_fwd(r, cache, table, lens, new_lens=new, scale=0.1, out=into) is into
        return (r, paged_attn_fwd(r, cache, table, lens, new_lens=new), into, *paged_kv_gather(cache, table, lens, 5, new_lens=lens))

    native, cache._native = cache._native, None
    want = step()
    cache._native = native
    with monkeypatch.context() as m:
        _ran_natively(cache, m)
        got = step()
    for a, b in zip(got, want):
        assert torch.equal(a, b) and a.stride() == b.stride()
    cache.check_status()


def test_left_to_python():
    from pbs_attn_b200.decode import paged_attn_fwd
    cache, table, lens, q, k, v = _case()
    past = torch.randn(2, 2, 100, 128, device="cuda").to(torch.bfloat16)
    from pbs_attn_b200.decode import paged_kv_append
    paged_kv_append(cache, past, past, table, lens, new_lens=lens)
    h, want = cache._host, paged_attn_fwd(q, cache, table, lens)
    call = lambda q=q, t=table, n=lens, m=None, s=None, o=None: h.paged_attn(cache._native, q, t, n, m, s, o)  # noqa: E731
    assert torch.equal(call(), want)
    odd = torch.zeros(*q.shape[:3], 129, dtype=q.dtype, device="cuda")[..., 1:]
    odd.copy_(q)
    for r in (call(q=odd), call(q=q.half()), call(q=q.cpu()), call(q=q[:, :7]), call(q=q[:0]), call(t=table.long()), call(n=lens.cpu()),
              call(n=lens[:1]), call(m=lens.long()), call(s=1), call(o=odd), call(o=q[:, :4]), call(t=table[0]), call(t=table[:, :0])):
        assert r is None
    assert torch.equal(paged_attn_fwd(odd, cache, table, lens), want)
    assert h.paged_append(cache._native, k, v, table, lens, None, None, None, q, None) is None
    assert h.paged_append(cache._native, k, v[:, :1], table, lens, None, None, None, None, None) is None
    assert h.paged_gather(cache._native, table, lens, 0, None) is None and h.paged_gather(cache._native, table, lens, 1.0, None) is None
    cache._word.value = 1                                  # a fault is Python's to tell
    assert call() is None and h.paged_gather(cache._native, table, lens, 1, None) is None
    assert h.paged_append(cache._native, k, v, table, lens, None, None, None, None, None) is None
    cache._word.value = 0
    cache.check_status()


def test_workspaces_grow_and_are_given_up():
    from pbs_attn_b200.decode import paged_attn_fwd, paged_kv_append
    caches = [make_cache(40, 16, h, 64, torch.float16, 4, 32) for h in (1, 4)]
    past = torch.randn(1, 4, 600, 64, device="cuda").to(torch.float16)
    want = []
    for c in caches:
        table = make_table(c, [600])
        paged_kv_append(c, past[:, :c.kv_heads], past[:, :c.kv_heads], table, ints(600))
        q = torch.randn(1, 32, 2, 64, device="cuda").to(torch.float16)
        want.append((c, table, q, paged_attn_fwd(q, c, table, ints(600))))
    torch.cuda.synchronize()
    for s in [torch.cuda.Stream() for _ in range(12)]:
        with torch.cuda.stream(s):
            for c, table, q, w in want:
                assert torch.equal(paged_attn_fwd(q, c, table, ints(600)), w)
    torch.cuda.synchronize()


def test_logits_same_bits_as_through_python(monkeypatch):
    from pbs_attn_b200 import logits as module
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3, 999, generator=g, device="cuda").to(torch.bfloat16)
    kw = dict(tokens=torch.randint(0, 999, (3, 50), generator=g, device="cuda"), token_lens=ints(50, 20, 0), prompt_lens=ints(10, 20, 5),
              repetition_penalty=1.2, frequency_penalty=torch.rand(3, device="cuda"), presence_penalty=0.5,
              bias_ids=torch.randint(0, 999, (3, 4), generator=g, device="cuda").int(), bias_values=torch.randn(3, 4, device="cuda"),
              allowed=torch.randint(-2 ** 31, 2 ** 31 - 1, (1, 32), generator=g, device="cuda").int())
    got = module.process_logits(x, **kw)
    assert module._host
    native = module._host.process_logits(module._address, x, *kw.values(), None)
    monkeypatch.setattr(module, "_host", False)
    want = module.process_logits(x, **kw)
    assert torch.equal(got, want) and torch.equal(native, want)


def test_captures_have_their_own_workspace():
    """Two graphs of several calls each, replayed in turn and beside eager calls."""
    from pbs_attn_b200.decode import paged_attn_fwd, paged_kv_append
    cache = make_cache(300, 16, 2, 64, torch.float16, 4, 32)
    past = torch.randn(2, 2, 2000, 64, device="cuda").to(torch.float16)
    table = make_table(cache, [2000, 1500])
    lens = ints(2000, 1500)
    paged_kv_append(cache, past, past, table, lens, new_lens=lens)
    q = [torch.randn(2, 8, 1, 64, device="cuda").to(torch.float16) for _ in range(4)]
    want = [paged_attn_fwd(x, cache, table, lens) for x in q]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for pair in (q[:2], q[2:]):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs += [paged_attn_fwd(x, cache, table, lens) for x in pair]
        graphs.append(g)
    for _ in range(5):
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        again = paged_attn_fwd(q[0], cache, table, lens)
        assert torch.equal(again, want[0]) and all(torch.equal(o, w) for o, w in zip(outs, want))
    cache.check_status()
    torch.cuda.synchronize()
    del graphs


def _captures(n, q, cache, table, lens):
    for _ in range(n):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = paged_attn(q, cache, table, lens)
        g.replay()
        torch.cuda.synchronize()
        del g, out


def paged_attn(*a, **kw):
    from pbs_attn_b200.decode import paged_attn_fwd
    return paged_attn_fwd(*a, **kw)


def _filled(n=2000):
    from pbs_attn_b200.decode import paged_kv_append
    cache = make_cache(300, 16, 2, 64, torch.float16, 4, 32)
    past = torch.randn(1, 2, n, 64, device="cuda").to(torch.float16)
    table, lens = make_table(cache, [n]), ints(n)
    paged_kv_append(cache, past, past, table, lens, new_lens=lens)
    return torch.randn(1, 8, 1, 64, device="cuda").to(torch.float16), cache, table, lens


@pytest.mark.parametrize("native", [True, False])
def test_captures_and_streams_leave_the_memory_of_the_stream_in_use(native):
    """A stream that keeps calling keeps its memory: no call on it allocates, however many captures and other streams come between."""
    q, cache, table, lens = _filled()
    if not native:
        cache._native = None
    out = torch.empty_like(q)
    want = paged_attn(q, cache, table, lens)
    torch.cuda.synchronize()
    count = lambda: torch.cuda.memory_stats()["allocation.all.allocated"]  # noqa: E731
    for s in [torch.cuda.Stream() for _ in range(12)]:
        _captures(1, q, cache, table, lens)
        with torch.cuda.stream(s):
            paged_attn(q, cache, table, lens)
        s.synchronize()
        before = count()
        paged_attn(q, cache, table, lens, out=out)
        assert count() == before and torch.equal(out, want)


def test_memory_of_captures_that_are_gone_is_given_back():
    q, cache, table, lens = _filled()
    cache._host.paged_forget()
    paged_attn(q, cache, table, lens)
    _captures(2, q, cache, table, lens)
    before = torch.cuda.memory_allocated()
    _captures(12, q, cache, table, lens)
    assert torch.cuda.memory_allocated() <= before


def test_dense_tensors_between_the_16_byte_boundaries():
    """Queries, results, keys, values and rotary tables that are dense and begin anywhere."""
    from pbs_attn_b200.decode import paged_kv_append
    cache, table, lens, q, k, v = _case()
    cos, sin = rope_tables(128, 128, torch.bfloat16)

    def shifted(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        return room.copy_(t)

    want = paged_kv_append(cache, k, v, table, lens, cos=cos, sin=sin, query_states=q)
    got = paged_kv_append(cache, shifted(k), shifted(v), table, lens, cos=shifted(cos), sin=shifted(sin), query_states=shifted(q), query_out=shifted(q))
    assert torch.equal(got, want)
    past = torch.randn(2, 2, 100, 128, device="cuda").to(torch.bfloat16)
    paged_kv_append(cache, past, past, table, lens, new_lens=lens)
    out = shifted(q)
    assert paged_attn(shifted(q), cache, table, lens, out=out) is out and torch.equal(out, paged_attn(q, cache, table, lens))
