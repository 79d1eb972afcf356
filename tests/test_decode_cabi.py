"""CPU-only: the C entries of the paged cache and the logits refuse what they cannot do before anything is enqueued."""
import ctypes as C
import os

import pytest

from pbs_attn_b200 import _cabi


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_cabi.lib_path()):
        from pbs_attn_b200.build import build
        build()
    return _cabi.load()


def _cache(**kw):
    d = dict(k=1 << 30, v=2 << 30, k_params=3 << 30, v_params=4 << 30, num_pages=8, page_size=16, kv_heads=2, head_dim=128, dtype=_cabi.BF16, bits=4,
             group_size=64, status=1 << 20)
    d.update(kw)
    row, prow = d["head_dim"] // 2 if d["bits"] == 4 else d["head_dim"], 2 * (d["head_dim"] // 64)
    strides = lambda r: (C.c_int64 * 3)(d["page_size"] * d["kv_heads"] * r, d["page_size"] * r, r)  # noqa: E731
    for n in ("k_strides", "v_strides"):
        d.setdefault(n, strides(row))
    for n in ("k_params_strides", "v_params_strides"):
        d.setdefault(n, strides(prow))
    return _cabi.PagedCache(**{n: (C.c_int64 * 3)(*v) if n.endswith("strides") else v for n, v in d.items()})


def _batch(**kw):
    return _cabi.PagedBatch(**{**dict(block_table=1 << 21, table_stride=4, seq_lens=1 << 22, new_lens=None, max_pages=4, batch=2, new_tokens=1), **kw})


ST = _cabi.Strides4(8 * 128, 128, 128, 1)


def _attn(lib, cache, batch, q_heads=8, q=1 << 24, out=1 << 25, st=ST, ost=ST, space=1 << 26, size=1 << 24):
    return lib.pbs_paged_attn(C.byref(cache), C.byref(batch), q_heads, C.c_void_p(q), st, C.c_void_p(out), ost, 1.0, C.c_void_p(space), size, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=_cabi.FP32), -3), (dict(bits=8), -3), (dict(head_dim=96), -1), (dict(group_size=128), -1), (dict(page_size=24), -1), (dict(page_size=8), -1),
    (dict(page_size=2048), -1), (dict(kv_heads=0), -1), (dict(num_pages=0), -1), (dict(k=None), -3), (dict(v_params=None), -3), (dict(status=None), -3),
    (dict(k=(1 << 30) + 8), -2), (dict(v_strides=(2048, 1024, 72)), -2), (dict(k_strides=(-2048, 1024, 64)), -2), (dict(k_params=(3 << 30) + 4), -2)])
def test_caches_that_are_refused(lib, kw, code):
    before = lib.pbs_launch_count()
    n = C.c_int64()
    assert lib.pbs_paged_attn_workspace(C.byref(_cache(**kw)), C.byref(_batch()), 8, C.byref(n)) == code, lib.pbs_last_error_string()
    assert _attn(lib, _cache(**kw), _batch()) == code
    assert lib.pbs_paged_gather(C.byref(_cache(**kw)), C.byref(_batch()), C.c_void_p(1 << 24), ST, C.c_void_p(1 << 25), ST, None) == code
    assert lib.pbs_paged_append(C.byref(_cache(**kw)), C.byref(_batch()), C.c_void_p(1 << 24), ST, C.c_void_p(1 << 25), ST, 0, None, None, None, None, None, None,
                                None, 0, None) == code
    assert lib.pbs_launch_count() == before


@pytest.mark.parametrize("kw,code", [
    (dict(batch=0), -1), (dict(new_tokens=0), -1), (dict(max_pages=0), -1), (dict(batch=5000), -1), (dict(max_pages=1 << 28), -1), (dict(block_table=None), -3),
    (dict(seq_lens=None), -3), (dict(table_stride=-1), -2), (dict(new_tokens=1 << 30), -1)])
def test_batches_that_are_refused(lib, kw, code):
    assert _attn(lib, _cache(), _batch(**kw)) == code, lib.pbs_last_error_string()


def test_attention_refuses(lib):
    n = C.c_int64()
    assert lib.pbs_paged_attn_workspace(C.byref(_cache()), C.byref(_batch()), 8, C.byref(n)) == 0 and n.value > _cabi.PAGED_COUNTER_BYTES
    assert _attn(lib, _cache(), _batch(), q_heads=7) == -1
    assert _attn(lib, _cache(), _batch(), q=None) == -3
    assert _attn(lib, _cache(), _batch(), q=(1 << 24) + 2) == -2
    assert _attn(lib, _cache(), _batch(), ost=_cabi.Strides4(8 * 128, 0, 128, 1)) == -2 and b"share memory" in lib.pbs_last_error_string()
    assert _attn(lib, _cache(), _batch(), space=None) == -3
    assert _attn(lib, _cache(), _batch(), size=n.value - 1) == -1 and b"workspace" in lib.pbs_last_error_string()
    assert _attn(lib, _cache(num_pages=1 << 26, k_strides=(1 << 20, 1024, 64)), _batch(), size=n.value) == -1 and b"64 GiB" in lib.pbs_last_error_string()


def test_append_refuses(lib):
    cs = (C.c_int64 * 3)(0, 128, 1)

    def call(q=1 << 26, cos=1 << 27, sin=1 << 28, cs=cs, rows=64, heads=8):
        p = lambda x: None if x is None else C.c_void_p(x)  # noqa: E731
        return lib.pbs_paged_append(C.byref(_cache()), C.byref(_batch()), p(1 << 24), ST, p(1 << 25), ST, heads, p(q), ST, p(1 << 29), ST, p(cos), p(sin), cs, rows, None)

    assert call(cos=None) == -3 and call(cos=None, sin=None) == -3 and call(heads=3) == -1 and call(rows=-1) == -1
    assert call(cs=(C.c_int64 * 3)(0, 128, 2)) == -2 and call(cs=(C.c_int64 * 3)(0, 100, 1)) == -2 and call(cos=(1 << 27) + 8) == -2


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=5), -3), (dict(rows=0), -1), (dict(vocab=0), -1), (dict(rows=70000), -1), (dict(logits=None), -3), (dict(out=None), -3), (dict(out_stride=10), -2),
    (dict(logits=(1 << 24) + 1), -2), (dict(token_bytes=2), -3), (dict(history=-1), -1), (dict(bias_ids=1 << 27, biases=3, bias_id_bytes=8), -3)])
def test_logits_refuse(lib, kw, code):
    d = dict(dtype=_cabi.BF16, rows=2, vocab=100, history=10, token_bytes=8, logits=1 << 24, out=1 << 25, logits_stride=100, out_stride=100, tokens=1 << 26,
             tokens_stride=10, repetition_all=1.0)
    before = lib.pbs_launch_count()
    assert lib.pbs_process_logits(C.byref(_cabi.Logits(**{**d, **kw})), None) == code, lib.pbs_last_error_string()
    assert lib.pbs_launch_count() == before


def test_structs_lie_as_in_the_header():
    """Sizes and offsets that the C compiler gives the header's structs."""
    assert C.sizeof(_cabi.PagedCache) == 4 * 8 + 4 * 24 + 8 * 4 + 8 and _cabi.PagedCache.num_pages.offset == 128
    assert C.sizeof(_cabi.PagedBatch) == 4 * 8 + 4 * 4
    assert _cabi.Logits.logits.offset == 32 and _cabi.Logits.repetition_all.offset == 120 and C.sizeof(_cabi.Logits) == 184


def test_numbers_of_biases_that_an_index_cannot_count_are_refused(lib):
    """A thread's index goes on by 256 behind the last of them."""
    for n in (1 << 30, 2 ** 31 - 1):
        d = _cabi.Logits(dtype=_cabi.BF16, rows=1, vocab=100, biases=n, bias_ids=1 << 27, bias_values=1 << 28, bias_id_bytes=8, bias_ids_stride=n,
                         bias_values_stride=n, logits=1 << 24, out=1 << 25, logits_stride=100, out_stride=100, repetition_all=1.0)
        before = lib.pbs_launch_count()
        assert lib.pbs_process_logits(C.byref(d), None) == -1 and b"biases" in lib.pbs_last_error_string()
        assert lib.pbs_launch_count() == before


def test_units_that_the_dealing_cannot_count_are_refused(lib):
    """The last block's share may end behind the last unit: that has to fit 32 bits as well."""
    n = C.c_int64()
    call = lambda pages: lib.pbs_paged_attn_workspace(C.byref(_cache(kv_heads=1)), C.byref(_batch(max_pages=pages, batch=510)), 1, C.byref(n))  # noqa: E731
    assert call((4210752 - 1) * 16) == -1 and b"count" in lib.pbs_last_error_string()       # 510 * 4210752 = 2^31 - 128 units
    assert call((4200000 - 1) * 16) == 0
