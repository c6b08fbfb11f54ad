"""Expanded latent prompts where their rows go from one product to the other: 128 gathered rows and fewer, 256, odd numbers of 128 behind these."""
import pytest
import torch

import attention_norms as norms
import shared_attn_oracle as oracle
from metrale_inference_alpha_b200 import ops
from shared_attn_oracle import run_latent

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,ctx", [([128], [128]), ([129], [129]), ([100, 28], [128, 30]), ([256], [256]), ([90, 60, 40], [120, 100, 128])], ids=str)
@pytest.mark.parametrize("heads", [1, 5, 16])
def test_latent_prompt(new, ctx, heads):
    c = oracle.latent(210, new, ctx, heads)
    want, bound = norms.latent(c)
    got = run_latent({k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()})
    ops.check_status("cuda")
    assert norms.distance(got, want) <= bound
