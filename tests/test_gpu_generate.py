"""Generation on a patched model through the paged cache, against the model itself."""
import json

import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(kind="llama", dtype=torch.bfloat16):
    from transformers import LlamaConfig, LlamaForCausalLM, Qwen2Config, Qwen2ForCausalLM
    kw = dict(vocab_size=300, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
              num_key_value_heads=2, max_position_embeddings=2048)
    torch.manual_seed(0)
    m = LlamaForCausalLM(LlamaConfig(head_dim=64, **kw)) if kind == "llama" else Qwen2ForCausalLM(Qwen2Config(**kw))
    return m.to(dtype).cuda().eval()


def _patched(model):
    from pbs_attn.patch.huggingface import apply_patch_with_prefill, get_permuted_block_sparse_attn_fwd
    # every block: the prompt's attention is the model's own
    return apply_patch_with_prefill(model, get_permuted_block_sparse_attn_fwd(block_size=64, segment_size=128, threshold=1, force_select_first_block=False))


@pytest.mark.parametrize("kind", ["llama", "qwen2"])
@pytest.mark.parametrize("batch,prompt", [(1, 200), (3, 65), (2, 1)])
def test_steps_follow_the_model(kind, batch, prompt):
    """Each step's logits, with a cache of 16 bits, are those of the model on the whole sequence.  Both round to bf16 some fifteen times
    a layer, and twice at the end, by up to 2^-8 of what they round; errors of two layers of independent signs, taken five deep."""
    from pbs_attn_b200.generate import generate
    from pbs_attn_b200.hf_patch import remove_patch
    model = _model(kind)
    ids = torch.randint(0, 300, (batch, prompt), device="cuda")
    steps = []
    out = generate(_patched(model), ids, 7, bits=16, page_size=16, cuda_graph=False, step_logits=steps)
    assert out.shape == (batch, prompt + 7) and torch.equal(out[:, :prompt], ids) and len(steps) == 7
    remove_patch(model)
    with torch.no_grad():
        want = model(out).logits.float()[:, prompt - 1:-1]
    got = torch.stack(steps, 1).float()
    bound = 5 * (32 ** 0.5) * 2.0 ** -8 * want.abs().amax(-1, keepdim=True)
    assert ((got - want).abs() <= bound).all()
    # the chosen token is among those that the bound cannot tell from the best
    best = want.amax(-1, keepdim=True)
    assert (want.gather(-1, out[:, prompt:, None]) >= best - 2 * bound).all()


@pytest.mark.parametrize("bits", [4, 16])
def test_graph_and_eager_choose_the_same(bits):
    from pbs_attn_b200.generate import generate
    model = _patched(_model())
    ids = torch.randint(0, 300, (2, 150), device="cuda")
    kw = dict(bits=bits, group_size=32, repetition_penalty=1.3, frequency_penalty=0.1, presence_penalty=0.2)
    a, b = generate(model, ids, 20, **kw), generate(model, ids, 20, cuda_graph=False, **kw)
    assert torch.equal(a, b)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_on_a_device_that_is_not_current():
    from pbs_attn_b200.generate import generate
    model, first = _patched(_model()).to("cuda:1"), _patched(_model())
    ids = torch.randint(0, 300, (2, 150), device="cuda")
    want = generate(first, ids, 20, repetition_penalty=1.3)              # (a capture on the current device comes first)
    for graph in (True, False):
        assert torch.equal(generate(model, ids.to("cuda:1"), 20, repetition_penalty=1.3, cuda_graph=graph).to("cuda"), want)


def test_call_after_call_keeps_no_memory():
    """What libraries keep for the stream of a capture they keep once."""
    from pbs_attn_b200.generate import generate
    model = _patched(_model())
    ids = torch.randint(0, 300, (2, 150), device="cuda")
    held = []
    for _ in range(4):
        generate(model, ids, 6, repetition_penalty=1.3)
        held.append(torch.cuda.memory_allocated())
    assert held[3] <= held[0]


def test_masks_and_penalties_reach_the_choice():
    from pbs_attn_b200.generate import generate
    model = _patched(_model())
    ids = torch.randint(0, 300, (1, 80), device="cuda")
    allowed = torch.zeros(1, 10, dtype=torch.int32, device="cuda")
    allowed[0, 3] = 0b1111 << 4                            # tokens 100 .. 103
    out = generate(model, ids, 12, bits=4, allowed=allowed)[0, 80:]
    assert ((out >= 100) & (out < 104)).all()
    out = generate(model, ids, 4, bits=4, allowed=allowed, presence_penalty=1e4)[0, 80:]
    assert sorted(out.tolist()) == [100, 101, 102, 103]
    bias = torch.full((1, 1), 1e4, device="cuda")
    assert (generate(model, ids, 5, bits=16, bias_ids=torch.tensor([[77]], device="cuda"), bias_values=bias)[0, 80:] == 77).all()


def test_refusals():
    from pbs_attn_b200.generate import PagedModelCache, generate
    model = _model()
    ids = torch.zeros(1, 4, dtype=torch.long, device="cuda")
    with pytest.raises(ValueError, match="patched"):
        generate(model, ids, 2)
    _patched(model)
    with pytest.raises(ValueError, match="at least one"):
        generate(model, ids, 0)
    with pytest.raises(ValueError, match="eager"):
        generate(model, ids, 2, step_logits=[])
    cache = PagedModelCache(model, 1, 8)
    cache.add(8)
    with pytest.raises(ValueError, match="holds 8"):
        cache.add(1)


def test_other_calls_of_a_patched_model_stay_as_they_were():
    model = _patched(_model())
    ids = torch.randint(0, 300, (1, 130), device="cuda")
    with torch.no_grad():
        out = model.generate(ids, max_new_tokens=4, do_sample=False)
    assert out.shape == (1, 134)


def test_efficiency_reports_the_time_of_a_token(tmp_path):
    from pbs_attn_b200 import efficiency
    efficiency.ARCHS["tiny-llama"] = dict(kind="llama", vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                                          num_attention_heads=4, num_key_value_heads=2, head_dim=64, rope_theta=10000.0,
                                          max_position_embeddings=4096, rms_norm_eps=1e-5)
    out = tmp_path / "r.jsonl"
    try:
        efficiency.main(["--arch", "tiny-llama", "--lens", "1024", "--block-size", "64", "--segment-size", "128", "--warmup", "1", "--iters", "1",
                         "--decode", "8", "--out", str(out)])
    finally:
        efficiency.ARCHS.pop("tiny-llama", None)
    rec = json.loads(out.read_text())
    assert rec["decode_tokens"] == 8 and rec["cache_bits"] == 4 and rec["decode_ms_per_token"] < 1000
