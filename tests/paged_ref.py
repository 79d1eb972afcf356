"""Plain forms in 64 bits of the paged cache and the attention over it, and caches to test with."""
import math

import torch

# unit roundoff of the storage types
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# half the distance of two numbers next to 0
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def make_cache(pages, page_size, heads, dim, dtype, bits, group, token_major=False):
    """Filled with NaN (or codes whose params are NaN): what was not appended must not be read.  token_major: (pages, page_size, heads, row) memory."""
    from pbs_attn_b200.decode import PagedKVCache

    def pool(row, dt):
        shape = (pages, page_size, heads, *row) if token_major else (pages, heads, page_size, *row)
        t = torch.full(shape, 255 if dt == torch.uint8 else math.nan, dtype=dt, device="cuda")
        return t.transpose(1, 2) if token_major else t

    if bits == 16:
        return PagedKVCache.from_tensors(pool((dim,), dtype), pool((dim,), dtype))
    return PagedKVCache.from_tensors(pool((dim // 2,), torch.uint8), pool((dim // 2,), torch.uint8), pool((dim // group, 2), dtype),
                                     pool((dim // group, 2), dtype))


def make_table(cache, lens, seed=0, spare=0):
    """A table with pages in no order; entries behind a sequence's end name no page."""
    per = max(1, max(-(-n // cache.page_size) for n in lens)) + spare
    order = torch.randperm(cache.num_pages, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((len(lens), per), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        k = -(-n // cache.page_size)
        table[b, :k] = order[at:at + k]
        at += k
    assert at <= cache.num_pages
    return table.cuda()


def pages_for(lens, page_size):
    return sum(-(-n // page_size) for n in lens) + 2


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def held(cache, table, b, n):
    """Tokens 0 .. n - 1 of sequence b in 64 bits: k, v and the magnitudes of their parts, each (H, n, D)."""
    out = []
    t = torch.arange(n, device="cuda")
    page, slot = table[b].long()[t // cache.page_size], t % cache.page_size
    for x, params in ((cache.k, cache.k_params), (cache.v, cache.v_params)):
        x = x[page, :, slot].transpose(0, 1)
        if cache.bits == 16:
            x = x.double()
            out.append((x, x.abs()))
            continue
        codes = torch.stack([x & 15, x >> 4], -1).flatten(-2).double().unflatten(-1, (-1, cache.group_size))
        step, low = params[page, :, slot].transpose(0, 1).double().split(1, -1)
        out.append(((codes * step + low).flatten(-2), (codes * step.abs() + low.abs()).flatten(-2)))
    return out


def attention(q, cache, table, lens, new=None, scale=None):
    """The result in 64 bits and a bound of the kernels' error, both (B, Hq, S, D).

    Scores are sums of D products (held in 32 bits, up to D / 16 + 4 of its roundings deep, each of them up to 2^-22 of the sum of
    magnitudes); a score that is e off changes its weight by the factor exp(e), and so the result by up to 2 e times the weighted
    magnitudes.  Weights are rounded to the type that they are multiplied in (bf16 pages: bf16; else fp16), and the result to its own."""
    B, Hq, S, D = q.shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    unit_p = 2.0 ** -8 if cache.bits == 16 and cache.dtype == torch.bfloat16 else 2.0 ** -11
    want = torch.zeros(B, Hq, S, D, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    for b in range(B):
        n = lens[b]
        m = S if new is None else new[b]
        if n == 0:
            continue
        (k, ka), (v, va) = held(cache, table, b, n)
        for i in range(m):
            end = n - m + i + 1
            if end <= 0:
                continue
            x = q[b, :, i].double().view(cache.kv_heads, -1, D)
            s = torch.einsum("hgd,htd->hgt", x, k[:, :end]) * scale
            e = torch.einsum("hgd,htd->hgt", x.abs(), ka[:, :end]).amax(-1, keepdim=True) * scale * (D / 16 + 4) * 2.0 ** -22
            p = torch.softmax(s, -1)
            o, a = torch.einsum("hgt,htd->hgd", p, v[:, :end]), torch.einsum("hgt,htd->hgd", p, va[:, :end])
            want[b, :, i] = o.reshape(Hq, D)
            bound[b, :, i] = ((2 * e + unit_p + 2.0 ** -18) * a + UNIT[q.dtype] * o.abs() + TINY[q.dtype]).reshape(Hq, D)
    return want, bound


def assert_within(got, want, bound):
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan())
    off = (got - want).abs()
    bad = (off > bound) & ~want.isnan()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off / bound.clamp(min=1e-300))[bad].max()):.3g} times the bound"


def rotate(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin


def rope_tables(n, dim, dtype, theta=10000.0):
    inv = 1.0 / (theta ** (torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim))
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    ang = torch.cat([ang, ang], -1)
    return ang.cos().to(dtype), ang.sin().to(dtype)
