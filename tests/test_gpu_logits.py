"""Penalties, biases and grammar masks on logits, against the formulas in 64 bits."""
import math

import pytest
import torch

from paged_ref import TINY, UNIT, ints

pytestmark = pytest.mark.gpu


def _want(logits, tokens=None, token_lens=None, prompt_lens=None, repetition_penalty=None, frequency_penalty=None, presence_penalty=None,
          bias_ids=None, bias_values=None, allowed=None):
    B, V = logits.shape
    x, size = logits.double().cpu(), logits.double().abs().cpu()
    of = lambda p, b, none: none if p is None else float(p[b]) if isinstance(p, torch.Tensor) else float(torch.tensor(p))  # noqa: E731
    for b in range(B):
        if tokens is not None:
            n = tokens.shape[1] if token_lens is None else min(max(int(token_lens[b]), 0), tokens.shape[1])
            m = 0 if prompt_lens is None else int(prompt_lens[b])
            row = tokens[b, :n].tolist()
            r, f, p = (of(t, b, none) for t, none in ((repetition_penalty, 1.0), (frequency_penalty, 0.0), (presence_penalty, 0.0)))
            counts = {}
            for i, t in enumerate(row):
                if 0 <= t < V:
                    counts[t] = counts.get(t, 0) + (i >= m)
            for t, c in counts.items():
                x[b, t] = x[b, t] / r if x[b, t] > 0 else x[b, t] * r
                size[b, t] = abs(x[b, t])
                if c:
                    x[b, t] -= f * c + p
                    size[b, t] += abs(f) * c + abs(p)
        if bias_ids is not None:
            for t, v in zip(bias_ids[b].tolist(), bias_values[b].tolist()):
                if 0 <= t < V:
                    x[b, t] += v
                    size[b, t] += abs(v)
        if allowed is not None:
            v = torch.arange(V)
            words = allowed[b if allowed.shape[0] > 1 else 0].cpu().long()
            x[b, (words[v // 32] >> (v % 32)) & 1 == 0] = -math.inf
    return x, size


def _check(logits, **kw):
    from pbs_attn_b200.logits import process_logits
    before = logits.clone()
    got = process_logits(logits, **kw)
    torch.cuda.synchronize()
    assert torch.equal(logits.view(torch.uint8) if logits.is_contiguous() else logits, before.view(torch.uint8) if logits.is_contiguous() else before)
    want, size = _want(logits, **kw)
    got64, dt = got.double().cpu(), logits.dtype
    fine = want.isfinite()
    assert torch.equal(got64.isfinite(), fine) and torch.equal(got64[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    # up to six roundings in 32 bits, then one of the type
    bound = UNIT[dt] * want.abs() + 2.0 ** -21 * size + TINY[dt]
    assert ((got64 - want).abs() <= bound)[fine].all()
    return got


def _inputs(B, V, L, dtype, seed=0, ids=torch.int64, biases=9):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda hi, *s: torch.randint(0, hi, s, generator=g, device="cuda")  # noqa: E731
    f = lambda lo, hi: torch.rand(B, generator=g, device="cuda") * (hi - lo) + lo  # noqa: E731
    words = r(1 << 32, B, -(-V // 32))
    return (torch.randn(B, V, generator=g, device="cuda") * 4).to(dtype), dict(
        tokens=(r(max(1, V // 3), B, L) * 2 - 3).to(ids),              # repeated, some outside
        token_lens=r(L + 1, B).int(), prompt_lens=r(L + 1, B).int(), repetition_penalty=f(0.7, 1.6), frequency_penalty=f(-0.5, 1),
        presence_penalty=f(-0.5, 1), bias_ids=(r(V + 2, B, biases) - 1).to(ids), bias_values=torch.randn(B, biases, generator=g, device="cuda") * 3,
        allowed=torch.where(words >= 1 << 31, words - (1 << 32), words).int())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,V,L", [(1, 1, 1), (2, 7, 5), (3, 31, 40), (2, 33, 3), (1, 1000, 300), (4, 4095, 100), (3, 4097, 1000), (2, 32001, 777),
                                   (1, 128256, 2000), (5, 50257, 63)])
@pytest.mark.parametrize("ids", [torch.int64, torch.int32])
def test_all_at_once(dtype, B, V, L, ids):
    logits, kw = _inputs(B, V, L, dtype, seed=V, ids=ids)
    _check(logits, **kw)


PARTS = ["repetition_penalty", "frequency_penalty", "presence_penalty", "bias", "allowed"]


@pytest.mark.parametrize("part", PARTS + ["nothing"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_each_alone(part, dtype):
    logits, kw = _inputs(3, 5003, 200, dtype)
    keep = {"bias": ["bias_ids", "bias_values"], "allowed": ["allowed"], "nothing": []}.get(part, [part, "tokens", "token_lens", "prompt_lens"])
    got = _check(logits, **{k: v for k, v in kw.items() if k in keep})
    if part == "nothing":
        assert torch.equal(got, logits)


def test_numbers_for_penalties_and_whole_rows():
    logits, kw = _inputs(3, 900, 64, torch.float32)
    a = _check(logits, tokens=kw["tokens"], repetition_penalty=1.3, frequency_penalty=0.25, presence_penalty=-0.5)
    full = lambda v: torch.full((3,), v, device="cuda")  # noqa: E731
    b = _check(logits, tokens=kw["tokens"], token_lens=ints(64, 64, 64), prompt_lens=ints(0, 0, -5), repetition_penalty=full(1.3),
               frequency_penalty=full(0.25), presence_penalty=full(-0.5))
    assert torch.equal(a, b)


@pytest.mark.parametrize("repetition", [None, 1.3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompts_longer_than_any_history(repetition, dtype):
    """A prompt length of 2^31 - 1 says that all of the row is the prompt, as that of its history does; one of -2^31, none of it."""
    most, L = 2 ** 31 - 1, 700
    logits, kw = _inputs(6, 3000, L, dtype, seed=4)
    args = dict(tokens=kw["tokens"], token_lens=ints(L, 600, 0, L, 300, most), repetition_penalty=repetition, frequency_penalty=kw["frequency_penalty"],
                presence_penalty=kw["presence_penalty"])
    got = _check(logits, prompt_lens=ints(most, most - 255, most, -most - 1, 301, most - 100), **args)
    assert torch.equal(got, _check(logits, prompt_lens=ints(L, 600, 0, 0, 300, L), **args))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lead,out_lead", [(0, 0), (1, 1), (3, 3), (1, 2), (0, 5)])
def test_rows_that_start_anywhere(dtype, lead, out_lead):
    from pbs_attn_b200.logits import process_logits
    logits, kw = _inputs(4, 3001, 100, dtype)
    want = _check(logits, **kw)
    room = torch.full((4, 3050), 7.0, dtype=dtype, device="cuda")
    room[:, lead:lead + 3001] = logits
    into = torch.full((4, 3050), 9.0, dtype=dtype, device="cuda")
    out = into[:, out_lead:out_lead + 3001]
    assert process_logits(room[:, lead:lead + 3001], out=out, **kw) is out
    assert torch.equal(out, want)
    assert (into[:, :out_lead] == 9).all() and (into[:, out_lead + 3001:] == 9).all()


def test_in_place_and_shared_rows():
    from pbs_attn_b200.logits import process_logits
    logits, kw = _inputs(3, 2500, 50, torch.bfloat16)
    kw["allowed"] = kw["allowed"][:1]
    want = _check(logits, **kw)
    assert process_logits(logits, out=logits, **kw) is logits and torch.equal(logits, want)
    one = torch.randn(1, 2500, device="cuda").expand(3, 2500)
    kw["tokens"], kw["bias_ids"], kw["bias_values"] = (kw[n][:1].expand(3, -1) for n in ("tokens", "bias_ids", "bias_values"))
    _check(one, **kw)


def test_infinities_and_nan_in_logits():
    logits, kw = _inputs(2, 600, 50, torch.float32)
    logits[:, 5], logits[:, 6], logits[:, 7] = math.inf, -math.inf, math.nan
    kw["tokens"][:, :3] = torch.tensor([5, 6, 7], device="cuda")
    kw["token_lens"], kw["bias_ids"][:, :3] = ints(50, 50), torch.tensor([5, 6, 7], device="cuda")
    _check(logits, **kw)


def test_a_row_with_nothing_allowed():
    logits, _ = _inputs(2, 70, 1, torch.bfloat16)
    allowed = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    allowed[1] = -1
    got = _check(logits, allowed=allowed)
    assert (got[0] == -math.inf).all() and torch.equal(got[1], logits[1])


def test_a_token_written_very_often():
    logits, _ = _inputs(1, 5000, 1, torch.float32)
    tokens = torch.full((1, 200000), 4321, device="cuda")
    _check(logits, tokens=tokens, frequency_penalty=0.01, prompt_lens=ints(100))


def test_biases_listed_more_than_once_add_up_in_order():
    logits, _ = _inputs(1, 300, 1, torch.float32)
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, 4, (1, 400), generator=g, device="cuda") * 70
    values = torch.randn(1, 400, generator=g, device="cuda") * 10
    from pbs_attn_b200.logits import process_logits
    got = process_logits(logits, bias_ids=ids, bias_values=values)
    for t in (0, 70, 140, 210):
        s = torch.zeros((), dtype=torch.float32)
        for v in values[0][ids[0] == t].cpu():
            s = s + v
        assert got[0, t].item() == (logits[0, t].cpu() + s).item()
    for _ in range(5):
        assert torch.equal(process_logits(logits, bias_ids=ids, bias_values=values), got)


def test_refusals():
    from pbs_attn_b200.logits import process_logits
    logits, kw = _inputs(2, 64, 8, torch.bfloat16)
    for error, args, more in (
            (RuntimeError, (logits.cpu(),), {}), (TypeError, (logits.double(),), {}), (ValueError, (logits[0],), {}),
            (ValueError, (logits.t(),), {}), (ValueError, (logits,), {"out": logits[:, :5]}),
            (ValueError, (logits,), {"repetition_penalty": 1.2}), (ValueError, (logits,), {"tokens": kw["tokens"], "repetition_penalty": 0.0}),
            (TypeError, (logits,), {"tokens": kw["tokens"].float()}), (TypeError, (logits,), {"tokens": kw["tokens"].cpu()}),
            (ValueError, (logits,), {"tokens": kw["tokens"][:1]}), (TypeError, (logits,), {"tokens": kw["tokens"], "token_lens": kw["token_lens"].long()}),
            (ValueError, (logits,), {"bias_ids": kw["bias_ids"]}), (ValueError, (logits,), {"bias_ids": kw["bias_ids"], "bias_values": kw["bias_values"][:, 1:]}),
            (TypeError, (logits,), {"bias_ids": kw["bias_ids"], "bias_values": kw["bias_values"].half()}),
            (ValueError, (logits,), {"allowed": kw["allowed"][:, :1]}), (TypeError, (logits,), {"allowed": kw["allowed"].long()})):
        with pytest.raises(error):
            process_logits(*args, **more)
    from pbs_attn_b200 import _cabi
    with pytest.raises(_cabi.PbsError):
        process_logits(logits, out=logits[:1].expand(2, 64))
    assert process_logits(logits[:0]).shape == (0, 64)
