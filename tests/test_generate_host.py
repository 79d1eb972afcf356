"""CPU-only: the host side of generation, with the model's layers and CUDA replaced by fakes."""
import contextlib
import types

import pytest
import torch

import pbs_attn_b200.generate as module


@pytest.fixture
def fakes(monkeypatch):
    """Fakes that note (what, device that was current, device of the stream that was given)."""
    seen, current = [], [None]

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], d
        yield
        current[0] = before

    @contextlib.contextmanager
    def graph(g, stream=None, **kw):
        seen.append(("graph", current[0], getattr(stream, "device", None)))
        yield

    class Event:
        def __init__(self, **kw):
            seen.append(("event", current[0], None))

        def record(self):
            pass

        def synchronize(self):
            pass

        def elapsed_time(self, other):
            return 1.0

    class Cache:
        def __init__(self, model, batch, *a):
            self.seq_lens = torch.zeros(batch, dtype=torch.int32)

        def add(self, n):
            self.seq_lens += n

        def check_status(self):
            pass

    for name, x in (("device", device), ("graph", graph), ("Event", Event), ("synchronize", lambda d=None: None),
                    ("Stream", lambda d=None: types.SimpleNamespace(device=d)), ("CUDAGraph", lambda: types.SimpleNamespace(replay=lambda: None))):
        monkeypatch.setattr(torch.cuda, name, x)
    monkeypatch.setattr(module, "_STREAMS", {})
    monkeypatch.setattr(module, "PagedModelCache", Cache)
    monkeypatch.setattr(module, "is_model_supported", lambda m: True)
    monkeypatch.setattr(module, "process_logits", lambda x, **kw: x)

    def layers(model, ids, cache):
        seen.append(("layers", current[0], None))
        return torch.zeros(ids.shape[0], 5)

    monkeypatch.setattr(module, "_run_layers", layers)
    return seen


def test_everything_runs_with_the_inputs_device_current(fakes):
    """The current device is not the model's: streams, graphs and events are those of the model's all the same."""
    model = types.SimpleNamespace(model=types.SimpleNamespace(layers=[]))
    ids = torch.zeros(1, 4, dtype=torch.long)
    timings = {}
    assert module.generate(model, ids, 5, timings=timings).shape == (1, 9) and timings["ms_per_token"] > 0
    assert [w for w, _, _ in fakes] == ["layers", "layers", "graph", "layers", "event", "event"]
    assert all(d == ids.device for _, d, _ in fakes)
    assert all(s == ids.device for w, _, s in fakes if w == "graph")


@pytest.mark.parametrize("grouped", [False, True])
def test_a_prefill_function_is_told_its_layer_in_front_of_a_paged_cache_too(grouped):
    from pbs_attn_b200.hf_patch import patched_attention_forward
    told = []

    def fn(q, k, v, layer_idx):
        told.append((layer_idx, k.shape[1], v.shape[1]))
        return q

    fn.takes_grouped_kv = grouped

    class Cache:
        def attend(self, attn, hidden, prefill_fn):
            return prefill_fn(torch.zeros(1, 8, 5, 4), torch.zeros(1, 2, 5, 4), torch.zeros(1, 2, 5, 4))

    layer = types.SimpleNamespace(layer_idx=3)
    out, _ = patched_attention_forward(layer, torch.zeros(1, 5, 32), None, None, past_key_values=Cache(), prefill_fn=fn)
    assert out.shape == (1, 8, 5, 4) and told == [(3, 2, 2) if grouped else (3, 8, 8)]


def _llama(**kw):
    from transformers import LlamaConfig, LlamaForCausalLM
    return LlamaForCausalLM(LlamaConfig(vocab_size=300, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                                        num_key_value_heads=2, head_dim=64, max_position_embeddings=64, **kw)).to(torch.bfloat16)


@pytest.mark.parametrize("rope,changes", [("default", False), ("dynamic", True)])
def test_rotary_tables_that_change_with_the_length_are_refused(rope, changes):
    """A cached key was rotated by the tables of its time; where they change as the sequence grows, one set of tables is not the model's."""
    model = _llama(rope_parameters={"rope_type": rope, "rope_theta": 10000.0, "factor": 2.0})
    before = model.model.rotary_emb.inv_freq.clone()
    with pytest.raises(RuntimeError, match="CUDA"):        # (within the length that it was made for: as far as the cache itself)
        module.PagedModelCache(model, 1, 60)
    with pytest.raises(ValueError if changes else RuntimeError, match="rotary" if changes else "CUDA"):
        module.PagedModelCache(model, 1, 200)
    assert torch.equal(model.model.rotary_emb.inv_freq, before)


def test_layers_that_see_a_window_alone_are_refused_beyond_it():
    """The steps attend to everything that is cached."""
    from transformers import Qwen2Config, Qwen2ForCausalLM
    model = Qwen2ForCausalLM(Qwen2Config(vocab_size=300, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                                         num_key_value_heads=2, use_sliding_window=True, sliding_window=16, max_window_layers=1)).to(torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        module.PagedModelCache(model, 1, 16)
    with pytest.raises(ValueError, match="window"):
        module.PagedModelCache(model, 1, 17)
