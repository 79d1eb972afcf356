"""Rows of a batch that go on from other rows of their group: tables, and pages under way in the caches of all layers."""
import pytest
import torch

from paged_ref import ints, make_cache
from paged_ref8 import make_cache8

pytestmark = pytest.mark.gpu
FORMATS = [(16, 0), (8, 16), (8, 64), (4, 32), (4, 64)]


def _caches(layers, pages, ps, H, D, dtype, bits, share, token_major=False, seed=0):
    """Caches whose memory is all different."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    made = []
    for _ in range(layers):
        c = make_cache8(pages, ps, H, D, dtype, share, token_major) if bits == 8 else make_cache(pages, ps, H, D, dtype, bits, share, token_major)
        for t in (c.k, c.v, c.k_params, c.v_params):
            if t is not None and t.dtype.is_floating_point:
                t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
            elif t is not None:
                t.copy_(torch.randint(-128 if t.dtype == torch.int8 else 0, 128 if t.dtype == torch.int8 else 256, t.shape, generator=g, device="cuda"))
        made.append(c)
    return made


def _tensors(c):
    return [t for t in (c.k, c.v, c.k_params, c.v_params) if t is not None]


def _table(groups, n, per, ps, pages, lens, seed):
    """Full pages at random among the last ones, the page under way a row's own."""
    g = torch.Generator().manual_seed(seed)
    rows = groups * n
    table = torch.randint(rows, pages, (rows, per), generator=g)
    for r in range(rows):
        if lens[r] // ps < per:
            table[r, lens[r] // ps] = r
    return table.int().cuda()


def _expected(caches, table, lens, beams):
    groups, n = beams.shape
    ps = caches[0].page_size
    new, copies = table.clone(), []
    for b in range(groups):
        for i in range(n):
            r, src = b * n + i, b * n + int(beams[b, i])
            full, fill = lens[r] // ps, lens[r] % ps
            new[r, :full] = table[src, :full]
            if fill:
                copies.append((int(table[r, full]), int(table[src, full]), fill))
    held = []
    for c in caches:
        for t in _tensors(c):
            x = t.clone()
            for to, src, fill in copies:
                units = -(-fill // c.block_size) if t.dim() == 3 else fill      # (scales lie by the block)
                x[to, :, :units] = t[src, :, :units]
            held.append(x)
    return new, held


def _run(caches, table, lens, beams):
    from pbs_attn_b200.decode import paged_kv_reorder
    want_table, want = _expected(caches, table, lens, beams.cpu())
    paged_kv_reorder(caches, table, ints(*lens), beams)
    caches[0].check_status()
    assert torch.equal(table, want_table)
    got = [t for c in caches for t in _tensors(c)]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits,share", FORMATS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 16, 32])
def test_formats_and_groups(bits, share, D, n):
    ps, groups, per = 64, 3, 4
    g = torch.Generator().manual_seed(n)
    lens = [x for x in (100, 64, 255) for _ in range(n)]
    pages = groups * n + 9
    caches = _caches(2, pages, ps, 3, D, torch.bfloat16, bits, share, token_major=n % 2 == 1, seed=n)
    beams = torch.stack([torch.randint(0, n, (n,), generator=g), torch.randperm(n, generator=g), torch.arange(n).flip(0)]).int().cuda()
    _run(caches, _table(groups, n, per, ps, pages, lens, n), lens, beams)


@pytest.mark.parametrize("bits,share", [(16, 0), (8, 16), (4, 64)])
@pytest.mark.parametrize("ps", [16, 128, 1024])
@pytest.mark.parametrize("n", [4, 6])
def test_lengths_and_pages(bits, share, ps, n):
    g = torch.Generator().manual_seed(ps)
    lens = [x for x in (0, 1, 15, 16, 17, ps - 1, ps, ps + 1, 2 * ps, 2 * ps + 7, 3 * ps - 1, 3 * ps) for _ in range(n)]
    groups = len(lens) // n
    pages = groups * n + 5
    caches = _caches(1, pages, ps, 2, 64, torch.float16, bits, share)
    _run(caches, _table(groups, n, 3, ps, pages, lens, 1), lens, torch.randint(0, n, (groups, n), generator=g).int().cuda())


@pytest.mark.parametrize("layers", [1, 33, 64, 65, 130])
def test_many_layers(layers):
    n, lens = 4, [21] * 8
    caches = _caches(layers, 12, 16, 1, 64, torch.bfloat16, 8, 16)
    beams = ints(1, 0, 0, 3, 3, 2, 1, 0).view(2, 4)
    _run(caches, _table(2, n, 2, 16, 12, lens, 2), lens, beams)


def test_rows_of_a_group_that_differ_in_length():
    lens = [20, 37, 20, 37, 37, 20]
    caches = _caches(2, 12, 16, 2, 64, torch.bfloat16, 16, 0)
    table = _table(1, 6, 3, 16, 12, lens, 3)
    _run(caches, table, lens, ints(2, 3, 0, 4, 1, 2)[None])


def test_one_cache_strided_beams_and_again():
    """A cache alone, beams as a part of a wider tensor, and a second call on what the first has left."""
    from pbs_attn_b200.decode import paged_kv_reorder
    lens = [21] * 8
    caches = _caches(1, 12, 16, 2, 64, torch.bfloat16, 8, 16)
    table = _table(2, 4, 2, 16, 12, lens, 4)
    wide = torch.full((2, 9), -5, dtype=torch.int32, device="cuda")
    wide[:, :4] = ints(1, 0, 0, 3, 3, 2, 1, 0).view(2, 4)
    _run(caches, table, lens, wide[:, :4])
    want_table, want = _expected(caches, table, lens, wide[:, :4].cpu())
    paged_kv_reorder(caches[0], table, ints(*lens), wide[:, :4])
    assert torch.equal(table, want_table) and all(torch.equal(a, b) for a, b in zip(_tensors(caches[0]), want))


def test_faults_leave_rows_as_they_were():
    from pbs_attn_b200 import _cabi
    from pbs_attn_b200.decode import paged_kv_reorder
    for bad, lens in ((ints(0, 4, -1, 2), [21] * 4), (ints(0, 1, 1, 2), [21, 21, 22, 21])):
        caches = _caches(1, 12, 16, 2, 64, torch.bfloat16, 16, 0)
        table = _table(1, 4, 2, 16, 12, lens, 5)
        # rows whose parent is none stay; the last takes over from row 2 or, where that is longer, stays too
        kept = bad.tolist()
        parents = [p if 0 <= p < 4 and lens[p] == lens[i] else i for i, p in enumerate(kept)]
        want_table, want = _expected(caches, table, lens, torch.tensor([parents]))
        paged_kv_reorder(caches, table, ints(*lens), bad[None])
        with pytest.raises(_cabi.PbsError, match="outside its group"):
            caches[0].check_status()
        assert torch.equal(table, want_table) and all(torch.equal(a, b) for a, b in zip(_tensors(caches[0]), want))
    caches = _caches(1, 12, 16, 2, 64, torch.bfloat16, 16, 0)
    table = _table(1, 2, 2, 16, 12, [21] * 2, 5)
    table[1, 1] = 70
    before = [t.clone() for t in _tensors(caches[0])]
    paged_kv_reorder(caches, table, ints(21, 21), ints(0, 0)[None])
    with pytest.raises(_cabi.PbsError, match="outside the pool"):
        caches[0].check_status()
    assert all(torch.equal(a, b) for a, b in zip(_tensors(caches[0]), before))


def test_through_python_and_captured(monkeypatch):
    from pbs_attn_b200.decode import paged_kv_reorder
    lens = [30] * 4
    caches = _caches(3, 12, 16, 2, 128, torch.bfloat16, 8, 16)
    table = _table(1, 4, 2, 16, 12, lens, 6)
    beams, n = ints(1, 1, 3, 0)[None], ints(*lens)
    monkeypatch.setattr(caches[0], "_native", None)
    _run(caches, table, lens, beams)
    monkeypatch.undo()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_kv_reorder(caches, table, n, beams)
    for other in (ints(3, 2, 1, 0), ints(0, 0, 0, 0), ints(2, 3, 1, 1)):
        beams.copy_(other[None])
        want_table, want = _expected(caches, table, lens, beams.cpu())
        graph.replay()
        assert torch.equal(table, want_table) and all(torch.equal(a, b) for a, b in zip([t for c in caches for t in _tensors(c)], want))


def test_refusals():
    from pbs_attn_b200 import _cabi
    from pbs_attn_b200.decode import paged_kv_reorder
    caches = _caches(2, 12, 16, 2, 64, torch.bfloat16, 16, 0)
    table, lens, beams = _table(2, 4, 2, 16, 12, [21] * 8, 7), ints(*[21] * 8), ints(*range(4), *range(4)).view(2, 4)
    other = _caches(1, 12, 32, 2, 64, torch.bfloat16, 16, 0)
    eight = _caches(1, 12, 16, 2, 64, torch.bfloat16, 8, 16)
    for error, args in ((TypeError, (caches, table, lens, beams.long())), (TypeError, (caches, table.long(), lens, beams)), (ValueError, (caches, table, lens, beams[:, :3])),
                        (ValueError, (caches, table, lens, beams.flatten())), (ValueError, (caches, table, lens[:5], beams)), (ValueError, (caches, table, lens, beams.t())),
                        (_cabi.PbsError, (caches + other, table, lens, beams)), (_cabi.PbsError, (caches + eight, table, lens, beams)),
                        (_cabi.PbsError, (caches, table[:1].expand(8, 2), lens, beams)), (TypeError, (caches, table, lens, beams.cpu())),
                        (_cabi.PbsError, (caches, table.repeat(5, 1)[:33], ints(*[21] * 33), ints(*range(33))[None]))):
        with pytest.raises(error):
            paged_kv_reorder(*args)
    paged_kv_reorder([], table, lens, beams)
    caches[0].check_status()
