"""Kernels of attention over shared prefixes and of expanded latent prompts, held to the 2-norms of attention_norms.py, which no mask that is a token off passes."""
import pytest
import torch

import attention_norms as norms
import shared_attn_oracle as oracle
from metrale_inference_alpha_b200 import ops
from shared_attn_oracle import run_latent, run_shared

pytestmark = pytest.mark.gpu


def cuda(c):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}


@pytest.fixture(autouse=True)
def _status():
    yield
    ops.check_status("cuda")


@pytest.mark.parametrize("case", norms.LATENT, ids=range(len(norms.LATENT)))
def test_latent_prompt(case):
    c = oracle.latent(200, **case)
    want, bound = norms.latent(c)
    assert norms.distance(run_latent(cuda(c)), want) <= bound


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("case", norms.SHARED, ids=range(len(norms.SHARED)))
def test_shared_prefix(case, fp8):
    c = oracle.shared(201, fp8=fp8, **case)
    want, bound = norms.shared(c)
    assert norms.distance(run_shared(cuda(c))[0], want) <= bound
