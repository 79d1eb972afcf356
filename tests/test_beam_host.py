"""CPU-only: what generation keeps of its beams, with the kernels replaced by plain forms."""
import itertools
import math
import types

import pytest
import torch

import pbs_attn_b200.generate as module


def _select(logits, scores, keep):
    x = torch.log_softmax(logits.double(), -1).view(*scores.shape, -1) + scores.double()[..., None]
    value, at = x.flatten(1).sort(dim=1, descending=True, stable=True)
    return value[:, :keep].float(), (at[:, :keep] // logits.shape[1]).int(), at[:, :keep] % logits.shape[1]


@pytest.fixture
def seen(monkeypatch):
    calls = []
    monkeypatch.setattr(module, "beam_select", _select)
    monkeypatch.setattr(module, "paged_kv_reorder", lambda layers, table, lens, beams: calls.append((lens.tolist(), beams.clone())))
    return calls


def _logits(text, V):
    """Of the token after `text`, made of it alone."""
    g = torch.Generator().manual_seed(sum((i + 1) * 131 * (t + 3) for i, t in enumerate(text)) % 10007)
    return torch.randn(V, generator=g) * 1.5


@pytest.mark.parametrize("N,ends,power", [(2, (), 1.0), (3, (0,), 1.0), (3, (0, 4), 0.0), (4, (2,), 2.0), (20, (1,), 0.7)])
def test_beams_are_those_of_a_search_by_hand(seen, N, ends, power):
    B, S, V, steps = 2, 3, 6, 4
    prompts = torch.randint(0, V, (B, S), generator=torch.Generator().manual_seed(N))
    beams = module._Beams(prompts, steps, N, list(ends), power)
    cache = types.SimpleNamespace(seq_lens=torch.full((B * N,), S, dtype=torch.int32), layers=[], block_table=None)
    running = [[([], 0.0)] for _ in range(B)]
    done = [[] for _ in range(B)]
    for t in range(steps):
        rows = torch.stack([_logits(beams.history[r, :S + t].tolist(), V) for r in range(B * N)])
        before = beams.history.clone()
        token = beams.choose(rows, cache)
        assert torch.equal(beams.history[torch.arange(B * N), S + t][:, None], token)
        # the caches follow the histories
        lens, parents = seen.pop()
        assert lens == [S + t] * (B * N) and parents.dtype == torch.int32 and parents.shape == (B, N)
        rows_of = (torch.arange(B)[:, None] * N + parents).flatten()
        alive = beams.scores.flatten() > -math.inf
        assert torch.equal(beams.history[alive, :S + t], before[rows_of][alive, :S + t])
        cache.seq_lens += 1
        for b in range(B):
            following = []
            for (text, score), v in itertools.product(running[b], range(V)):
                following.append((text + [v], score + float(torch.log_softmax(_logits(prompts[b].tolist() + text, V).double(), -1)[v])))
            following.sort(key=lambda x: -x[1])
            following = following[:N * (1 + len(ends))]
            done[b] += [(text, score / (t + 1) ** power) for text, score in following[:N] if text[-1] in ends]
            running[b] = [x for x in following if x[0][-1] not in ends][:N]
            got = {(tuple(beams.history[b * N + i, S:S + t + 1].tolist()), round(float(beams.scores[b, i]), 3)) for i in range(N) if beams.scores[b, i] > -math.inf}
            assert got == {(tuple(text), round(score, 3)) for text, score in running[b]}
    out = beams.best(prompts)
    for b in range(B):
        texts = done[b] + [(text, score / steps ** power) for text, score in running[b]]
        best = max(texts, key=lambda x: x[1])[0]
        assert out[b].tolist() == prompts[b].tolist() + best + [beams.pad] * (steps - len(best))


def test_a_cache_that_forks():
    """Full pages of the prompt are shared, all others are a row's own."""
    cache = object.__new__(module.PagedModelCache)
    per, N, prompt, page = 5, 3, 37, 16
    cache.block_table, cache.seq_lens = torch.arange(2 * per, dtype=torch.int32).view(2, per), torch.tensor([prompt, prompt], dtype=torch.int32)
    cache._beams, cache._shared = N, prompt // page
    cache.fork()
    table = cache.block_table.view(2, N, per)
    assert cache.seq_lens.tolist() == [prompt] * 6 and cache.block_table.dtype == torch.int32
    assert (table[:, :, :2] == table[:, :1, :2]).all()
    own = table[:, :, 2:].flatten().tolist()
    assert len(set(own)) == len(own) and not set(own) & set(table[:, :, :2].flatten().tolist())
    assert set(own) | set(table[:, :, :2].flatten().tolist()) == set(range(2 * (per + (N - 1) * (per - 2))))


def test_what_is_given_by_the_sequence_goes_to_its_rows():
    x = torch.arange(4).view(2, 2)
    assert module._for_beams(x, 3, 2).tolist() == [[0, 1]] * 3 + [[2, 3]] * 3
    assert module._for_beams(x[:1], 3, 2).shape == (1, 2) and module._for_beams(x[:1], 3, 1).shape == (3, 2)
    assert module._for_beams(1.5, 3, 2) == 1.5 and module._for_beams(None, 3, 2) is None
