"""Values far from 1 in the attention over a paged cache, against the formula in 64 bits on the values that the cache stands for."""
import math

import pytest
import torch

from paged_ref import assert_within, attention, ints, make_cache, make_table, pages_for

pytestmark = pytest.mark.gpu


def _run(q, k, v, bits, group, dtype, scale=None, ps=16):
    """Attention of the queries (1, Hq, S, D) over keys and values (1, 1, n, D)."""
    from pbs_attn_b200.decode import paged_attn_fwd, paged_kv_append
    n, D = k.shape[2:]
    cache = make_cache(pages_for([n], ps), ps, 1, D, dtype, bits, group)
    table = make_table(cache, [n])
    q, k, v = (t.to(dtype) for t in (q, k, v))
    paged_kv_append(cache, k, v, table, ints(n))
    got = paged_attn_fwd(q, cache, table, ints(n), scale=scale)
    cache.check_status()
    assert_within(got, *attention(q, cache, table, [n], None, scale))
    return got


def _random(n, D=128, S=1, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(1, h, s, D, generator=g, device="cuda") for h, s in ((4, S), (1, n), (1, n))]


@pytest.mark.parametrize("S", [1, 5])
@pytest.mark.parametrize("n", [1, 100, 20000])
def test_values_up_to_the_largest_that_16_bits_hold(n, S):
    """The weights' sum is not 1 while the sums grow: that must not cost the values their range."""
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = _random(n, S=S if n > 1 else 1)
        _run(q * 0.1, k, v.clamp(-1, 1).sign() * torch.finfo(dtype).max * 0.9, 16, 0, dtype)
        same = torch.linspace(-0.9, 0.9, 128, device="cuda").expand_as(v) * torch.finfo(dtype).max
        _run(q * 0.1, k, same, 16, 0, dtype)
        rise = torch.linspace(0, 2, n, device="cuda")[:, None] * q[0, 0, 0] / q[0, 0, 0].norm()
        _run(q, k + 4 * rise, same, 16, 0, dtype)


@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("S", [1, 3])
@pytest.mark.parametrize("first", ["nothing", "zeros", "small"])
def test_large_groups_without_a_range(group, S, first):
    """All channels of a group alike: its step is 0 and its minimum large, and the weights, which steps hold back, must not outgrow it."""
    n = 900
    for size in (2.0 ** 60, 2.0 ** 80, 2.0 ** 99):
        q, k, v = _random(n, S=S)
        flat = v.unflatten(-1, (-1, group))[..., :1].sign().expand(-1, -1, -1, -1, group).flatten(-2) * size
        if first == "zeros":
            flat[:, :, :400] = 0
        if first == "small":
            flat[:, :, :400] = v[:, :, :400] * 2.0 ** -70
        _run(q, k, flat, 4, group, torch.bfloat16)
        rise = torch.linspace(-2, 2, n, device="cuda")[:, None] * q[0, 0, 0] / q[0, 0, 0].norm()
        _run(q, k + 4 * rise, flat, 4, group, torch.bfloat16)


@pytest.mark.parametrize("dtype,large,small", [(torch.float16, 60000.0, 2.0 ** -13), (torch.bfloat16, 2.0 ** 40, 2.0 ** -20)])
@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("S", [1, 3])
def test_small_values_beside_large_ones_that_hardly_weigh(dtype, large, small, group, S):
    """Every other token is large, but its score is so far below that it leaves nothing: the small ones keep their codes."""
    n = 700
    q, k, v = _random(n, S=S)
    shared = torch.randn(128, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")
    shared /= shared.norm()
    odd = (torch.arange(n, device="cuda") % 2 == 1)[:, None]
    # scores of the two differ by 2 * 20 * 40 / sqrt(128) = 141 and more than 2^200 in weight
    q, k = q * 0.1 + 40 * shared, k + torch.where(odd, -20.0, 20.0) * shared
    _run(q, k, torch.where(odd, v.sign() * large, v * small), 4, group, dtype)


@pytest.mark.parametrize("bits,group", [(16, 0), (4, 32), (4, 64)])
def test_values_that_are_all_small(bits, group):
    """Weights make up for it, as far as the header's range goes."""
    for size in (2.0 ** -30, 2.0 ** -60, 2.0 ** -78):
        q, k, v = _random(900, S=3)
        _run(q, k, v * size, bits, group, torch.bfloat16)
    _run(q, k, v * 2.0 ** -13, bits, group, torch.float16)


@pytest.mark.parametrize("n", [100, 900, 9000])
@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("small", [0.0, 2.0 ** -76])
def test_runs_of_very_different_sizes_keep_their_weights(small, group, n):
    """Stretches of large values and of none at all: the latter leave nothing but their weights, whose sums are as far apart as the values."""
    for large in (2.0 ** 50, 2.0 ** 90):
        for run in (32, 128, 3000):
            q, k, v = _random(n, S=3)
            few = (torch.arange(n, device="cuda") // run % 2 == 0)[:, None]
            for one in (few, ~few):
                _run(q * 0.3, k, torch.where(one, v * small, v * large), 4, group, torch.bfloat16)
