"""The engine's option that attends to the prompts of latent-attention models in expanded form: what decides it, on the host."""
import pytest
import torch

from metrale_inference_alpha_b200.config.model_config import from_hf_config, preset
from metrale_inference_alpha_b200.engine.batch import ForwardBatch
from metrale_inference_alpha_b200.engine.llm_engine import EngineArgs, LLMEngine
from metrale_inference_alpha_b200.engine.runner import ModelRunner
from metrale_inference_alpha_b200.models import mla
from metrale_inference_alpha_b200.scheduler.policy import SchedulerConfig
from metrale_inference_alpha_b200.weights.loader import load_weights
from metrale_inference_alpha_b200.weights.source import SyntheticSource


def _batch(portions, pad_seqs=0):
    """portions: (rows, cached tokens in front)."""
    return ForwardBatch.build([dict(tokens=[1] * n, start_pos=p, blocks=list(range(1, (p + n) // 16 + 2))) for n, p in portions], 16, pad_seqs=pad_seqs)


@pytest.mark.parametrize("portions", [[(1, 0)], [(5, 0)], [(3, 9)], [(64, 0), (1, 40), (17, 5)]])
def test_a_batch_counts_its_pairs(portions):
    b = _batch(portions)
    assert b.total_ctx == sum(n + p for n, p in portions) == int(b.ctx_len.sum())
    assert b.total_pairs == sum(p + i + 1 for n, p in portions for i in range(n))
    assert _batch(portions, pad_seqs=8).total_ctx == 0


@pytest.mark.parametrize("portions,pays", [([(31, 0)], False), ([(32, 0)], True), ([(1, 0)] * 40, False), ([(600, 0)], True), ([(32, 4000)], False),
                                           ([(200, 4000)], True), ([(1, 4000)] * 64 + [(64, 0)], False), ([(1, 40)] * 64 + [(1024, 0)], True)])
def test_when_the_expanded_form_is_taken(portions, pays):
    assert mla._expanded_pays(_batch(portions)) is pays
    assert not mla._expanded_pays(_batch(portions, pad_seqs=80))             # a shape that is captured and replayed with other lengths


def test_the_option_is_checked_and_other_layers_stay_as_they_are():
    with pytest.raises(ValueError, match="latent_prompts"):
        LLMEngine(EngineArgs(model=preset("tiny-dense"), device="cpu", latent_prompts="both", num_kv_blocks=8))
    cfg = from_hf_config(dict(model_type="deepseek_v3", vocab_size=256, hidden_size=128, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=2,
                              intermediate_size=256, moe_intermediate_size=128, n_routed_experts=0, first_k_dense_replace=1, kv_lora_rank=64, q_lora_rank=64,
                              qk_nope_head_dim=32, qk_rope_head_dim=16, v_head_dim=32, rms_norm_eps=1e-6, rope_theta=1e4, max_position_embeddings=256),
                         name="tiny-mla")
    logits = {}
    for how in ("absorbed", "expanded"):
        w = load_weights(cfg, SyntheticSource(cfg, seed=3, device="cpu"), device="cpu")
        r = ModelRunner(cfg, w, "cpu", num_blocks=16, sched=SchedulerConfig(max_num_seqs=2, max_model_len=128), use_graphs=False, latent_prompts=how)
        assert not hasattr(w.layers[0].mixer, "_w_kv_bf16")
        logits[how] = r.decoder.forward(_batch([(40, 0)]), r.caches, out_f32=True)[0]
    assert torch.equal(logits["absorbed"], logits["expanded"])
