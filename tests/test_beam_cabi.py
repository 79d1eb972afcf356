"""CPU-only: the C entries of caches of 8 bits, of beams and of their caches refuse what they cannot do before anything is enqueued."""
import ctypes as C

import pytest

from pbs_attn_b200 import _cabi
from test_decode_cabi import ST, _attn, _batch, lib  # noqa: F401


def _cache8(**kw):
    d = dict(k=1 << 30, v=2 << 30, k_params=3 << 30, v_params=4 << 30, num_pages=8, page_size=64, kv_heads=2, head_dim=128, dtype=_cabi.BF16, bits=8,
             block_size=16, status=1 << 20)
    d.update(kw)
    blocks = d["page_size"] // max(1, d["block_size"])
    for n in ("k_strides", "v_strides"):
        d.setdefault(n, (d["page_size"] * 2 * d["head_dim"], d["page_size"] * d["head_dim"], d["head_dim"]))
    for n in ("k_params_strides", "v_params_strides"):
        d.setdefault(n, (blocks * 2, blocks, 1))
    return _cabi.PagedCache(**{n: (C.c_int64 * 3)(*v) if n.endswith("strides") else v for n, v in d.items()})


@pytest.mark.parametrize("kw,code", [
    (dict(block_size=0), -3), (dict(block_size=8), -3), (dict(block_size=24), -3), (dict(block_size=128), -3), (dict(page_size=16, block_size=32), -3),
    (dict(page_size=48, block_size=16), -1), (dict(head_dim=96), -1), (dict(k_params=None), -3), (dict(v_params=None), -3), (dict(k_params=(3 << 30) + 2), -2),
    (dict(v=(2 << 30) + 8), -2), (dict(k_strides=(16384, 8192, 120)), -2), (dict(v_params_strides=(8, -4, 1)), -2), (dict(dtype=_cabi.FP32), -3)])
def test_caches_of_8_bits_that_are_refused(lib, kw, code):  # noqa: F811
    before = lib.pbs_launch_count()
    cache, n = _cache8(**kw), C.c_int64()
    assert lib.pbs_paged_attn_workspace(C.byref(cache), C.byref(_batch()), 8, C.byref(n)) == code, lib.pbs_last_error_string()
    assert _attn(lib, cache, _batch()) == code
    assert lib.pbs_paged_gather(C.byref(cache), C.byref(_batch()), C.c_void_p(1 << 24), ST, C.c_void_p(1 << 25), ST, None) == code
    assert lib.pbs_paged_append(C.byref(cache), C.byref(_batch()), C.c_void_p(1 << 24), ST, C.c_void_p(1 << 25), ST, 0, None, None, None, None, None, None, None, 0, None) == code
    assert lib.pbs_launch_count() == before


def test_what_a_cache_of_8_bits_needs(lib):  # noqa: F811
    n = C.c_int64()
    assert lib.pbs_paged_attn_workspace(C.byref(_cache8()), C.byref(_batch()), 8, C.byref(n)) == 0 and n.value > _cabi.PAGED_COUNTER_BYTES
    assert _attn(lib, _cache8(), _batch(), size=n.value - 1) == -1 and b"workspace" in lib.pbs_last_error_string()
    assert _attn(lib, _cache8(num_pages=1 << 24, k_strides=(1 << 13, 8192, 128)), _batch(), size=n.value) == -1 and b"64 GiB" in lib.pbs_last_error_string()
    assert _attn(lib, _cache8(num_pages=1 << 26, k_strides=(512, 8192, 128), v_strides=(512, 8192, 128), k_params_strides=(1 << 8, 4, 1)), _batch(), size=n.value) == -1
    # blocks that a unit's number cannot count
    assert lib.pbs_paged_append(C.byref(_cache8(kv_heads=60000)), C.byref(_batch(batch=4096, new_tokens=1)), C.c_void_p(1 << 24), ST, C.c_void_p(1 << 25), ST, 0, None, None,
                                None, None, None, None, None, 0, None) == -1


def _reorder(lib, caches, batch, beams=2, table=1 << 21, parents=1 << 23, stride=2):  # noqa: F811
    pointers = (C.POINTER(_cabi.PagedCache) * max(1, len(caches)))(*(C.pointer(c) for c in caches))
    return lib.pbs_paged_reorder(pointers, len(caches), C.byref(batch), C.c_void_p(table), beams, C.c_void_p(parents), stride, None)


def test_reordering_refuses(lib):  # noqa: F811
    before = lib.pbs_launch_count()
    rows = _batch(batch=4)
    one = [_cache8()]
    assert _reorder(lib, [], rows) == -1
    assert _reorder(lib, one, rows, beams=0) == -1 and _reorder(lib, one, rows, beams=3) == -1 and _reorder(lib, one, _batch(batch=66), beams=33) == -1
    assert _reorder(lib, one, rows, table=None) == -3 and _reorder(lib, one, rows, parents=None) == -3
    assert _reorder(lib, one, rows, stride=-1) == -2 and _reorder(lib, one, _batch(batch=4, table_stride=3)) == -2
    assert _reorder(lib, one, _batch(batch=5000)) == -1 and _reorder(lib, one, _batch(batch=4, seq_lens=None)) == -3
    for other in (dict(page_size=32), dict(block_size=32), dict(kv_heads=1), dict(num_pages=9), dict(head_dim=64), dict(k_strides=(16384, 8192, 256)), dict(v_params_strides=(16, 4, 1)),
                  dict(dtype=_cabi.FP16)):
        assert _reorder(lib, one + [_cache8(k=5 << 30, **other)], rows) == -1 and b"one layout" in lib.pbs_last_error_string()
    assert _reorder(lib, one + [_cache8(k=5 << 30, status=None)], rows) == -3
    assert _reorder(lib, [_cache8(k=(5 + i) << 30) for i in range(3)] + [_cache8(k=6 << 30)], rows) == -3 and b"1 and 3 are one" in lib.pbs_last_error_string()
    assert lib.pbs_launch_count() == before


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), -3), (dict(batch=0), -1), (dict(batch=1025), -1), (dict(beams=0), -1), (dict(beams=33), -1), (dict(vocab=0), -1), (dict(vocab=(1 << 30) + 1), -1), (dict(keep=0), -1),
    (dict(keep=65), -1), (dict(keep=9, vocab=4), -1), (dict(logits=None), -3), (dict(scores=None), -3), (dict(out_scores=None), -3), (dict(out_beams=None), -3), (dict(out_tokens=None), -3),
    (dict(logits=(1 << 24) + 1), -2), (dict(logits_stride=-1), -2), (dict(scores=(1 << 25) + 2), -2), (dict(scores_stride=-1), -2), (dict(out_tokens=(1 << 28) + 4), -2)])
def test_beam_selection_refuses(lib, kw, code):  # noqa: F811
    d = dict(dtype=_cabi.BF16, batch=3, beams=2, vocab=1000, keep=4, logits=1 << 24, logits_stride=1000, scores=1 << 25, scores_stride=2, out_scores=1 << 26, out_beams=1 << 27,
             out_tokens=1 << 28)
    before, n = lib.pbs_launch_count(), C.c_int64()
    a = _cabi.BeamSelect(**{**d, **kw})
    assert lib.pbs_beam_select_workspace(C.byref(a), C.byref(n)) == code, lib.pbs_last_error_string()
    assert lib.pbs_beam_select(C.byref(a), C.c_void_p(1 << 29), 1 << 30, None) == code
    assert lib.pbs_launch_count() == before


def test_beam_selections_workspace(lib):  # noqa: F811
    a = _cabi.BeamSelect(dtype=_cabi.FP32, batch=3, beams=2, vocab=1000, keep=4, logits=1 << 24, logits_stride=1000, scores=1 << 25, scores_stride=2, out_scores=1 << 26,
                         out_beams=1 << 27, out_tokens=1 << 28)
    n = C.c_int64()
    assert lib.pbs_beam_select_workspace(C.byref(a), C.byref(n)) == 0 and n.value > _cabi.PAGED_COUNTER_BYTES
    assert lib.pbs_beam_select(C.byref(a), C.c_void_p(1 << 29), n.value - 1, None) == -1 and b"workspace" in lib.pbs_last_error_string()
    assert lib.pbs_beam_select(C.byref(a), None, n.value, None) == -3 and lib.pbs_beam_select(C.byref(a), C.c_void_p((1 << 29) + 8), n.value, None) == -2


def test_structs_lie_as_in_the_header():
    assert _cabi.PagedCache.block_size.offset == _cabi.PagedCache.group_size.offset + 4 and _cabi.PagedCache.status.offset == 160
    assert C.sizeof(_cabi.BeamSelect) == 6 * 4 + 4 * 8 + 3 * 8 and _cabi.BeamSelect.logits.offset == 24
