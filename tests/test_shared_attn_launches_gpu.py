"""Attention over shared prefixes, joins and expanded latent prompts give the same bits however their kernels are launched, and call after call."""
import pytest
import torch

import shared_attn_oracle as oracle
from metrale_inference_alpha_b200 import ops
from metrale_inference_alpha_b200.ops import _native
from shared_attn_oracle import run_latent, run_shared

pytestmark = pytest.mark.gpu

SHARED = [dict(ctx=[20, 9, 33, 4, 700], prefix=[600], start=[0, 4], heads=40, kv_heads=8, dim=128, fp8=True), dict(ctx=[3] * 90, prefix=[900, 70], start=[0, 50, 90], heads=10, kv_heads=2, dim=128, fp8=False),
          dict(ctx=[50, 1], prefix=[90, 30], start=[0, 1, 2], heads=40, kv_heads=1, dim=256, fp8=True, n=3), dict(ctx=[9, 0], prefix=[], start=[0], heads=4, kv_heads=2, dim=64, fp8=False)]
LATENT = [dict(new=[140, 30], ctx=[200, 60], heads=16), dict(new=[100, 300], ctx=[129, 641], heads=3)]


def cuda(c):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}


def test_the_same_bits_however_kernels_are_launched():
    shared, latent = [cuda(oracle.shared(300, **a)) for a in SHARED], [cuda(oracle.latent(301, **a)) for a in LATENT]
    lib = _native.lib()
    default = lib.mb_pdl_enabled()
    results = []
    try:
        for mode in (0, 1, 2, default):
            lib.mb_set_pdl(mode)
            for _ in range(3):
                r = []
                for c in shared:
                    r += run_shared(c)
                    r += ops.merge_attention([r[-2], r[-2]], [r[-1], r[-1]])
                    if not c["prefix"].numel():
                        continue
                    r += run_shared({**c, "ctx": torch.zeros_like(c["ctx"])}, max_ctx=0)
                    r += run_shared({**c, "prefix": torch.zeros_like(c["prefix"])}, max_prefix=0)
                r += [run_latent(c) for c in latent]
                results.append([t.clone() for t in r])
                torch.cuda.synchronize()
    finally:
        lib.mb_set_pdl(default)
    ops.check_status("cuda")
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], r))
