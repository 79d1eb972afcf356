"""Plain forms of the paged cache of 8 bits and the attention over it, and caches to test with."""
import math

import torch

from paged_ref import TINY, UNIT, rotate

LEAST = 2.0 ** -120
UNIT_W = 2.0 ** -11                     # weights times scales are rounded to fp16


def make_cache8(pages, page_size, heads, dim, dtype, block, token_major=False):
    """Filled with codes of 99 and scales of NaN: what was not appended must not be read."""
    from pbs_attn_b200.decode import PagedKVCache

    def pool():
        t = torch.full((pages, page_size, heads, dim) if token_major else (pages, heads, page_size, dim), 99, dtype=torch.int8, device="cuda")
        return t.transpose(1, 2) if token_major else t

    def scales():
        n = page_size // block
        t = torch.full((pages, n, heads) if token_major else (pages, heads, n), math.nan, device="cuda")
        return t.transpose(1, 2) if token_major else t

    return PagedKVCache.from_tensors(pool(), pool(), scales(), scales(), dtype=dtype)


def append8(cache, codes, scales, x, table, lens, new):
    """The definition in 32 bits, on copies (codes, scales) of the pages of keys or values: x (B, H, S, D) float32, rotated already."""
    ps, bs = cache.page_size, cache.block_size
    table = table.tolist()
    for b, (n, m) in enumerate(zip(lens, new)):
        first = max(0, n - m)
        for t0 in range(first // bs * bs, n, bs):
            page, slot = table[b][t0 // ps], t0 % ps
            a, e = max(first, t0), min(n, t0 + bs)
            if e <= a:
                continue
            rows = x[b, :, a - (n - m):e - (n - m)]                                       # (H, tokens, D)
            most = rows.abs().amax((1, 2))
            scale = (most * torch.tensor(1 / 127, dtype=torch.float32, device="cuda")).clamp(min=LEAST)
            scale = torch.where(most.isfinite(), scale, math.nan)
            if a > t0:
                old = scales[page, :, slot // bs].clone()
                scale = torch.where(old.isnan() | scale.isnan(), math.nan, torch.maximum(scale, old.abs()))
                ratio = (old / scale).double()[:, None, None]
                kept = codes[page, :, slot:slot + a - t0]
                codes[page, :, slot:slot + a - t0] = torch.where(ratio.isnan(), kept.double(), (kept.double() * ratio).round()).to(torch.int8)
            inv = (1 / scale).double()[:, None, None]
            codes[page, :, slot + a - t0:slot + e - t0] = torch.nan_to_num((rows.double() * inv).round()).to(torch.int8)
            scales[page, :, slot // bs] = scale


def values8(cache, codes, scales, table, b, n):
    """Tokens 0 .. n - 1 of sequence b in 64 bits, (H, n, D), and the largest magnitude that their blocks hold room for."""
    t = torch.arange(n, device="cuda")
    page, slot = table[b].long()[t // cache.page_size], t % cache.page_size
    scale = scales[page, :, slot // cache.block_size].double()
    return torch.einsum("thd,th->htd", codes[page, :, slot].double(), scale), 127 * (scale.abs().amax(0) if n else scale.sum(0))


def attention8(q, cache, table, lens, new=None, scale=None):
    """The result in 64 bits and a bound of the kernel's error, both (B, Hq, S, D).

    Queries are rounded by up to 2^-15 of the row's largest, and scores, sums of D products of integers, a few times in 32 bits (taken as up to
    D / 16 + 4 roundings of 2^-22 of the sum of magnitudes); a score that is e off changes its weight by the factor exp(e), and so the result by
    up to 2 e times the weighted magnitudes.  Weights times scales are rounded to fp16; where they are subnormal, by up to 2^-25, where the largest of them is at
    least 2^7 and the codes are at most 127: over n tokens that comes to n 2^-32 of the largest magnitude that a block has room for."""
    B, Hq, S, D = q.shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    want = torch.zeros(B, Hq, S, D, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    for b in range(B):
        n, m = lens[b], S if new is None else new[b]
        if n == 0:
            continue
        (k, _), (v, room) = values8(cache, cache.k, cache.k_params, table, b, n), values8(cache, cache.v, cache.v_params, table, b, n)
        for i in range(m):
            end = n - m + i + 1
            if end <= 0:
                continue
            x = q[b, :, i].double().view(cache.kv_heads, -1, D)
            s = torch.einsum("hgd,htd->hgt", x, k[:, :end]) * scale
            e = torch.einsum("hgd,htd->hgt", x.abs(), k[:, :end].abs()).amax(-1, keepdim=True) * abs(scale) * (D / 16 + 4) * 2.0 ** -22
            e = e + (x.abs().amax(-1, keepdim=True) * k[:, :end].abs().sum(-1).amax(-1)[:, None, None]) * abs(scale) * 2.0 ** -15
            p = torch.softmax(s, -1)
            o, a = torch.einsum("hgt,htd->hgd", p, v[:, :end]), torch.einsum("hgt,htd->hgd", p, v[:, :end].abs())
            want[b, :, i] = o.reshape(Hq, D)
            few = end * 2.0 ** -32 * room[:, None, None]
            bound[b, :, i] = ((2 * e + UNIT_W + 2.0 ** -18) * a + few + UNIT[q.dtype] * o.abs() + TINY[q.dtype]).reshape(Hq, D)
    return want, bound


__all__ = ["LEAST", "make_cache8", "append8", "values8", "attention8", "rotate"]
