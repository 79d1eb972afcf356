"""The choice among beams' continuations, against log-softmax and a full sort in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _scores64(logits, scores):
    """(B, N, V) in 64 bits, with the rules for what is not finite."""
    x = logits.double().nan_to_num(-math.inf, torch.finfo(torch.float32).max, -math.inf)
    x = torch.where(logits.isposinf(), torch.finfo(torch.float32).max, x)
    top = x.amax(-1, keepdim=True).clamp(min=-torch.finfo(torch.float32).max)
    y = x - top - (x - top).exp().sum(-1, keepdim=True).log()
    y = torch.where(x.isneginf(), -math.inf, y)
    own = torch.where(scores.isnan(), -math.inf, scores).double()
    return torch.where(own[..., None] == -math.inf, -math.inf, y.view(*scores.shape, -1) + own[..., None])


def _check(logits, scores, keep=None):
    from pbs_attn_b200.beam import beam_select
    B, N = scores.shape
    V = logits.shape[1]
    got, beams, tokens = beam_select(logits, scores, keep)
    K = 2 * N if keep is None else keep
    assert got.shape == beams.shape == tokens.shape == (B, K)
    assert (got.dtype, beams.dtype, tokens.dtype) == (torch.float32, torch.int32, torch.int64)
    want = _scores64(logits, scores)
    # what the tokens' places in order (score, beam, logit, token) are
    flat = want.flatten(1)
    order = flat.sort(dim=1, descending=True, stable=True)
    # sums of exponentials: their terms and the adding up in 32 bits, up to 80 one after the other; the score is rounded once
    off = 2.0 ** -22 + 80 * 2.0 ** -24
    place = beams.long() * V + tokens
    assert ((tokens >= 0) & (tokens < V) & (beams >= 0) & (beams < N)).all()
    assert (place.sort(1).values.diff(dim=1) != 0).all(), "a continuation twice"
    mine = flat.gather(1, place)
    near = lambda a, b: (a == b) | ((a - b).abs() <= off * 2 + b.abs() * 2.0 ** -23)  # noqa: E731
    assert near(got.double(), mine).all()
    assert near(mine, order.values[:, :K]).all()
    # beams apart by more than that, and tokens of one beam, come in one order only
    same = mine == order.values[:, :K]
    wrong = same & (place != order.indices[:, :K])
    assert not wrong.any(), (place[wrong][:5], order.indices[:, :K][wrong][:5])
    far = (order.values[:, :K] - mine).abs() > 0
    if far.any():                                          # (two beams' scores next to one another)
        assert ((order.indices[:, :K] // V) != beams)[far].all()
    return got, beams, tokens


def _logits(B, N, V, dtype, seed=0, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    scores = (-torch.rand(B, N, generator=g, device="cuda") * 10).sort(1, descending=True).values
    return (torch.randn(B * N, V, generator=g, device="cuda") * spread).to(dtype), scores


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,N,V,keep", [(1, 1, 1, 1), (1, 2, 2, 4), (3, 4, 33, 8), (2, 5, 1000, 10), (1, 4, 4097, 8), (7, 3, 20011, 6), (1, 32, 5003, 64), (2, 8, 128256, 16),
                                        (1, 1, 152064, 64), (40, 16, 9000, 33), (130, 1, 300, 2), (1024, 2, 65, 3)])
def test_types_and_sizes(dtype, B, N, V, keep):
    _check(*_logits(B, N, V, dtype, V + keep), keep)


@pytest.mark.parametrize("V", list(range(1, 20)) + [31, 63, 64, 65, 255, 257, 511, 1023, 1025, 2047, 2049, 8191])
def test_vocabularies(V):
    for dtype in (torch.bfloat16, torch.float32):
        _check(*_logits(2, 3, V, dtype, V), min(6, 3 * V))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_start_between_boundaries(dtype):
    logits, scores = _logits(3, 4, 5001, dtype, 3)
    for shift, stride in ((0, 5001), (1, 5001), (3, 5007), (5, 6000)):
        memory = torch.full((12 * stride + 16,), 99.0, dtype=dtype, device="cuda")
        view = memory[shift:shift + 12 * stride].view(12, stride)[:, :5001]
        view.copy_(logits)
        want, got = _check(logits, scores), _check(view, scores)
        # (slices are cut elsewhere: the sums' last bits may differ)
        assert torch.equal(want[2], got[2]) and torch.equal(want[1], got[1])
    wide = torch.zeros(3, 9, device="cuda")
    wide[:, :4] = scores
    assert all(torch.equal(a, b) for a, b in zip(_check(logits, scores), _check(logits, wide[:, :4])))
    _check(logits[:1].expand(12, -1), scores)


def test_ties():
    """Equal logits by their tokens, equal beams by their number; all equal, and few values."""
    for V in (5, 700, 30011):
        logits = torch.zeros(6, V, device="cuda")
        scores = torch.zeros(2, 3, device="cuda")
        got, beams, tokens = _check(logits, scores, min(12, 3 * V))
        K = got.shape[1]
        assert torch.equal(beams[0].long() * V + tokens[0], torch.arange(K, device="cuda"))
        g = torch.Generator(device="cuda").manual_seed(V)
        for dtype in (torch.bfloat16, torch.float32):
            _check(torch.randint(0, 3, (6, V), generator=g, device="cuda").to(dtype), scores, min(12, 3 * V))
            signs = torch.where(torch.rand(6, V, generator=g, device="cuda") < 0.5, -0.0, 0.0).to(dtype)
            assert torch.equal(_check(signs, scores, min(12, 3 * V))[2], _check(signs.abs(), scores, min(12, 3 * V))[2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [8, 40])
def test_large_ones_that_lie_together(dtype, K):
    """The largest in few threads' hands, more of them than are listed: neighbours, and the pieces of one thread."""
    V = 70000
    n = 8 if dtype == torch.bfloat16 else 4
    for make in (lambda i: i < 3000, lambda i: i // n % 256 == 77, lambda i: i // n % 256 < 40, lambda i: i >= V - 900):
        logits, scores = _logits(1, 2, V, dtype, 9, 1.0)
        logits = logits + 20 * make(torch.arange(V, device="cuda"))
        _check(logits, scores, K)
        up = torch.where(make(torch.arange(V, device="cuda")), torch.arange(V, device="cuda") / V, -5.0).to(dtype)
        _check(up[None].expand(2, -1), scores, K)


def test_masked_tokens_and_dead_beams():
    logits, scores = _logits(4, 4, 12000, torch.bfloat16, 4)
    scores[0, 1:] = -math.inf                              # a first step
    scores[1, 2] = math.nan
    scores[2] = -math.inf
    g = torch.Generator(device="cuda").manual_seed(5)
    logits[torch.rand(logits.shape, generator=g, device="cuda") < 0.99] = -math.inf
    logits[13] = -math.inf                                 # a beam that can not go on
    logits[12, 500:], logits[14:, 3:] = -math.inf, -math.inf
    got, beams, tokens = _check(logits, scores)
    assert (beams[0] == 0).all() and got[2].isneginf().all()
    assert torch.equal(tokens[2], torch.arange(8, device="cuda")) and (beams[2] == 0).all()
    # (entry 3 has fewer tokens left than are kept: -inf fills up, which beam 1 has nothing but)
    assert not (beams[1] == 2).any() and not ((beams[3] == 1) & got[3].isfinite()).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_what_is_not_finite(dtype):
    logits, scores = _logits(3, 2, 9001, dtype, 6)
    logits[0, 7], logits[1, ::3], logits[2, 5:] = math.nan, math.nan, math.nan
    logits[3, [4, 8000]] = math.inf
    logits[4, :] = math.nan
    logits[5, 100] = -math.inf
    got, beams, tokens = _check(logits, scores)
    assert not got.isnan().any()
    r = (beams[1] == 1).nonzero().flatten()[:2]
    assert tokens[1][r].tolist() == [4, 8000] and (got[1][r] - (scores[1, 1] - math.log(2))).abs().max() < 1e-5


def test_large_and_small_logits():
    for size in (1e-6, 100.0, 1e4, 1e30):
        _check(*_logits(2, 4, 3001, torch.float32, 7, size))
        _check(*_logits(2, 4, 3001, torch.bfloat16, 7, size))


def test_again_through_python_and_captured(monkeypatch):
    import pbs_attn_b200.beam as module
    logits, scores = _logits(5, 4, 50021, torch.bfloat16, 8)
    want = _check(logits, scores)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(want, module.beam_select(logits, scores)))
    monkeypatch.setattr(module, "_host", False)
    assert all(torch.equal(a, b) for a, b in zip(want, module.beam_select(logits, scores)))
    monkeypatch.undo()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = module.beam_select(logits, scores)
        out2 = module.beam_select(logits, out[0][:, :4].contiguous())
    other, other_scores = _logits(5, 4, 50021, torch.bfloat16, 9)
    side = torch.cuda.Stream()
    for _ in range(3):
        logits.copy_(other)
        scores.copy_(other_scores)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):                      # another stream has its own workspace
            beside = module.beam_select(other, other_scores)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, beside))
    assert all(torch.equal(a, b) for a, b in zip(out2, _check(other, out[0][:, :4].contiguous())))


def test_refusals():
    from pbs_attn_b200 import _cabi
    from pbs_attn_b200.beam import beam_select
    logits, scores = _logits(2, 3, 50, torch.bfloat16)
    for error, args in ((TypeError, (logits.double(), scores)), (TypeError, (logits, scores.double())), (ValueError, (logits, scores[:1])), (ValueError, (logits, scores[0])),
                        (ValueError, (logits.t(), scores)), (ValueError, (logits, scores, 0)), (RuntimeError, (logits.cpu(), scores.cpu())), (TypeError, (logits, scores.cpu())),
                        (ValueError, (logits[None], scores)), (_cabi.PbsError, (logits, scores, 65)), (_cabi.PbsError, (logits, scores, 2 ** 32 + 4)), (_cabi.PbsError, (logits[:, :3], scores, 10)),
                        (_cabi.PbsError, (logits[:, :0], scores, 1)), (_cabi.PbsError, (logits.expand(6, 50)[:1].expand(33, 50), scores.new_zeros(1, 33), 4)),
                        (_cabi.PbsError, (logits[:1].expand(1025, 50), scores.new_zeros(1025, 1), 4)), (ValueError, (logits[:0], scores.new_zeros(2, 0)))):
        with pytest.raises(error):
            beam_select(*args)
    assert beam_select(logits[:0], scores[:0], 4)[0].shape == (0, 4)


def _time_of(call, rounds=15):
    """Median of a call's time on the device, among others."""
    for _ in range(3):
        call()
    times = []
    for _ in range(rounds):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        start.record()
        for _ in range(8):
            call()
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end))
    return sorted(times)[rounds // 2]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_first_step_takes_no_longer_than_a_later_one(dtype):
    """Of beams that are not alive nothing is looked at; what comes out is the order of their tokens."""
    from pbs_attn_b200.beam import beam_select
    logits, scores = _logits(64, 8, 100003, dtype, 12)
    first, dead = scores.clone(), torch.full_like(scores, -math.inf)
    first[:, 1:] = -math.inf
    _check(logits, first)
    got, beams, tokens = _check(logits, dead)
    assert got.isneginf().all() and (beams == 0).all() and (tokens == torch.arange(16, device="cuda")).all()
    later = _time_of(lambda: beam_select(logits, scores))
    assert _time_of(lambda: beam_select(logits, first)) <= later and _time_of(lambda: beam_select(logits, dead)) <= later


@pytest.mark.parametrize("N,V,keep", [(1, 5, 5), (1, 64, 64), (4, 3, 12), (2, 4099, 64), (3, 130001, 64)])
def test_beams_that_are_all_dead(N, V, keep):
    """The first tokens of the first beams, whatever the logits are, at the ends of segments and of rows that start anywhere."""
    for dtype in (torch.bfloat16, torch.float32):
        for shift in (0, 1, 3):
            memory = torch.full((2 * N * V + 8,), math.nan, dtype=dtype, device="cuda")
            from pbs_attn_b200.beam import beam_select
            got, beams, tokens = beam_select(memory[shift:shift + 2 * N * V].view(2 * N, V), torch.full((2, N), -math.inf, device="cuda"), keep)
            assert got.isneginf().all()
            place = beams.long() * V + tokens
            assert torch.equal(place, torch.arange(keep, device="cuda").expand(2, -1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("left", [0, 1, 5, 16, 2000])
def test_masks_of_the_lowest_finite_number(dtype, left):
    """More logits that are equal than there is room for, beside the few that are not banned, in long segments and short ones."""
    for B, N, V, keep in ((64, 8, 20011, 16), (1, 2, 150001, 64), (200, 2, 6000, 33)):
        logits, scores = _logits(B, N, V, dtype, left, 2.0)
        g = torch.Generator(device="cuda").manual_seed(left)
        banned = torch.rand(B * N, V, generator=g, device="cuda").argsort(1) >= left
        logits[banned] = torch.finfo(dtype).min
        _check(logits, scores, keep)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_equal_logits_do_not_take_many_times_as_long(dtype):
    """Rows of one segment each, all but five tokens banned by the lowest finite number: a few passes over them, not one for each that is kept."""
    from pbs_attn_b200.beam import beam_select
    logits, scores = _logits(64, 8, 100003, dtype, 13)
    usual = _time_of(lambda: beam_select(logits, scores))
    logits[:, 5:] = torch.finfo(dtype).min
    assert _time_of(lambda: beam_select(logits, scores)) <= 8 * usual
