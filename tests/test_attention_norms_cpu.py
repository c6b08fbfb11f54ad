"""The bounds of attention_norms.py let no wrong result pass: masks that are a token off, tiles that are lost, scores without their rotation, zeros, weights of fewer bits."""
import pytest
import torch

import attention_norms as norms
import shared_attn_oracle as oracle
from shared_attn_oracle import run_latent, run_shared


@pytest.mark.parametrize("case", norms.LATENT, ids=range(len(norms.LATENT)))
def test_no_wrong_latent_prompt_is_within_the_bound(case):
    c = oracle.latent(200, **case)
    want, bound = norms.latent(c)
    assert 0.0015 < bound < 0.02
    first = min(c["ctx"].tolist())
    wrong = dict(less=dict(shift=-1), more=dict(shift=1), tile=dict(without=slice(0, min(128, first))), key=dict(without=slice(first // 2, first // 2 + 1)), rotation=dict(rope=False))
    for name, kw in wrong.items():
        got = norms.latent(c, **kw)[0].bfloat16()
        assert norms.distance(got, want) > 1.2 * bound, (name, norms.distance(got, want), bound)
    assert norms.distance(torch.zeros_like(want), want) > bound


@pytest.mark.parametrize("case", [norms.LATENT[0], norms.LATENT[-1]], ids=["one", "three"])
def test_the_restatement_of_a_latent_prompt_is(case):
    c = oracle.latent(200, **case)
    want, bound = norms.latent(c)
    assert norms.distance(run_latent(c), want) <= bound


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("case", norms.SHARED, ids=range(len(norms.SHARED)))
def test_no_wrong_shared_prefix_is_within_the_bound(case, fp8):
    c = oracle.shared(201, fp8=fp8, **case)
    want, bound = norms.shared(c)
    assert 0.0014 < bound < 0.01
    first = min(c["prefix"].tolist())
    wrong = dict(less=dict(shift=-1), tile=dict(without=slice(128, 256)), key=dict(without=slice(first // 2, first // 2 + 1)))
    if c["n"] > 1:
        wrong["more"] = dict(shift=1)                      # the others' last token sees all there is
    if fp8:
        wrong["weights"] = dict(round_weights=torch.bfloat16)
    for name, kw in wrong.items():
        got = norms.shared(c, **kw)[0].bfloat16()
        assert norms.distance(got, want) > 1.05 * bound, (name, norms.distance(got, want), bound)
    kept = norms.shared(c, round_weights=torch.float16 if fp8 else torch.bfloat16)[0].bfloat16()
    assert norms.distance(kept, want) <= bound
    assert norms.distance(torch.zeros_like(want), want) > bound


@pytest.mark.parametrize("fp8", [False, True])
def test_the_restatement_of_a_shared_prefix_is(fp8):
    c = oracle.shared(201, fp8=fp8, **norms.SHARED[1])
    want, bound = norms.shared(c)
    assert norms.distance(run_shared(c)[0], want) <= bound
