"""Prompts of latent-attention models in expanded form, through the model and the engine."""
import pytest
import torch

from metrale_inference_alpha_b200 import ops
from metrale_inference_alpha_b200.config.model_config import from_hf_config
from metrale_inference_alpha_b200.engine.batch import ForwardBatch
from metrale_inference_alpha_b200.engine.llm_engine import EngineArgs, LLMEngine
from metrale_inference_alpha_b200.engine.runner import ModelRunner
from metrale_inference_alpha_b200.ops import mla_cuda
from metrale_inference_alpha_b200.sampling.params import SamplingParams
from metrale_inference_alpha_b200.scheduler.policy import SchedulerConfig
from metrale_inference_alpha_b200.weights.loader import load_weights
from metrale_inference_alpha_b200.weights.source import SyntheticSource

pytestmark = pytest.mark.gpu


def _config(layers=2):
    return from_hf_config(dict(model_type="deepseek_v3", vocab_size=1024, hidden_size=512, num_hidden_layers=layers, num_attention_heads=16,
                               num_key_value_heads=16, intermediate_size=512, moe_intermediate_size=128, n_routed_experts=0, first_k_dense_replace=layers,
                               kv_lora_rank=512, q_lora_rank=192, qk_nope_head_dim=128, qk_rope_head_dim=64, v_head_dim=128, rms_norm_eps=1e-6,
                               rope_theta=1e4, max_position_embeddings=1024), name="tiny-mla")


def _tokens(n, seed):
    return torch.randint(1, 1024, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("H", [1, 8, 13])
def test_the_rotation_in_place_is_that_of_the_absorbed_rows(H):
    g = torch.Generator().manual_seed(H)
    T, slots = 37, 64
    q, ckv = torch.randn(T, H, 192, generator=g).bfloat16().cuda(), torch.randn(T, 576, generator=g).bfloat16().cuda()
    norm, ang = torch.randn(512, generator=g).bfloat16().cuda(), torch.rand(100, 32, generator=g).cuda() * 6
    pos, slot = torch.randint(0, 100, (T,), generator=g).int().cuda(), torch.randperm(slots, generator=g)[:T].cuda()
    slot[5] = -1
    c1, c2 = (torch.zeros(slots // 16, 16, 1, 576, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q_lat = torch.randn(H, T, 512, generator=g).bfloat16().cuda()
    qq = mla_cuda.prepare(q, q_lat, ckv, norm, ang.cos(), ang.sin(), pos, slot, c1, 128, 1e-6)
    mine = q.clone()
    mla_cuda.prepare_prompt(mine, ckv, norm, ang.cos(), ang.sin(), pos, slot, c2, 128, 1e-6)
    assert torch.equal(c1, c2) and torch.equal(mine[..., 128:], qq[..., 512:]) and torch.equal(mine[..., :128], q[..., :128])


def test_both_forms_of_a_prompt_give_the_logits_of_the_restatement(monkeypatch):
    """Two prompts (300 tokens in portions of 200 and 100, and one of 37 beside the second portion), then a token each: absorbed and expanded on the GPU
    against the 32-bit restatement. The bound is that of the absorbed block's own comparison (4 % of the largest logit): both forms round as many values to
    bf16 on the way (query latents and weighted latents there, keys and values here), by half a step of 2^-8 each."""
    cfg = _config()
    calls = []
    inner = ops.mla_prompt_attention
    monkeypatch.setattr(ops, "mla_prompt_attention", lambda q, *a, **k: calls.append(q.shape[0]) or inner(q, *a, **k))
    one, two, logits = _tokens(300, 1), _tokens(37, 2), {}
    b1, b2 = list(range(1, 21)), list(range(21, 25))
    steps = [[dict(tokens=one[:200], start_pos=0, blocks=b1)], [dict(tokens=one[200:], start_pos=200, blocks=b1), dict(tokens=two, start_pos=0, blocks=b2)],
             [dict(tokens=[7], start_pos=300, blocks=b1), dict(tokens=[9], start_pos=37, blocks=b2)]]
    for dev, how in (("cpu", "absorbed"), ("cuda", "absorbed"), ("cuda", "expanded")):
        w = load_weights(cfg, SyntheticSource(cfg, seed=3, device="cpu"), device=dev)
        r = ModelRunner(cfg, w, dev, num_blocks=32, sched=SchedulerConfig(max_num_seqs=2, max_model_len=512), use_graphs=False, latent_prompts=how)
        logits[dev, how] = [r.decoder.forward(ForwardBatch.build(s, 16, device=dev, max_blocks=r.max_blocks), r.caches, out_f32=True)[0].float().cpu()
                            for s in steps]
        assert calls == ([] if how == "absorbed" else [200, 200, 137, 137])
    ops.check_status("cuda")
    for a, b, c in zip(*logits.values()):
        for mine in (b, c):
            assert (a - mine).abs().max() <= 0.04 * a.abs().max() + 2e-3


def test_the_engine_answers_in_expanded_form_with_graphs_and_without(monkeypatch):
    cfg, outs, calls = _config(3), {}, []
    inner = ops.mla_prompt_attention
    monkeypatch.setattr(ops, "mla_prompt_attention", lambda q, *a, **k: calls.append(q.shape[0]) or inner(q, *a, **k))
    for graphs in (False, True):
        eng = LLMEngine(EngineArgs(model=cfg, device="cuda", max_num_seqs=4, max_model_len=512, num_kv_blocks=128, use_cuda_graphs=graphs,
                                   enable_prefix_caching=False, latent_prompts="expanded"))
        rids, done = [eng.add_request(_tokens(n, n), SamplingParams(max_tokens=6)) for n in (300, 40, 3)], {}
        while eng.has_work():
            done.update((o.request_id, o.output_ids) for o in eng.step() if o.finished)
        outs[graphs] = [done[r] for r in rids]
    assert outs[False] == outs[True] and all(len(o) == 6 for o in outs[True])
    assert calls
