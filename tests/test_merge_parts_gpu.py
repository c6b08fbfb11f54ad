"""Every number of parts that merge_attention takes, over all of its kernels, against 64 bits; and what a part of weight zero holds."""
import pytest
import torch

import shared_attn_oracle as oracle
from metrale_inference_alpha_b200 import ops
from shared_attn_oracle import within

pytestmark = pytest.mark.gpu


def _parts(parts, rows, heads, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    outs = [torch.randn(rows, heads, dim, generator=g).to(dtype) for _ in range(parts)]
    lses = [torch.randn(rows, heads, generator=g) * 5 for _ in range(parts)]
    for o, l in zip(outs, lses):
        none = torch.rand(rows, heads, generator=g) < 0.2
        l[none], o[none] = -float("inf"), float("nan")
    return outs, lses


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("parts", range(1, 17))
@pytest.mark.parametrize("rows,heads,dim", [(77, 3, 128), (9, 5, 20), (5, 2, 515), (600, 4, 64)])
def test_merge(dtype, parts, rows, heads, dim):
    """Rows of whole 16-byte pieces and others, more of them than a CTA takes."""
    outs, lses = _parts(parts, rows, heads, dim, dtype, 41 + parts)
    out, tol, lse, ltol = oracle.merge_exact(outs, lses)
    a, b = ops.merge_attention([o.cuda() for o in outs], [l.cuda() for l in lses])
    within(a, out, tol, "outputs")
    within(b, lse, ltol, "log-sum-exps")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("parts", [4, 5, 8, 12])
@pytest.mark.parametrize("late", [0, 1])
def test_merge_in_a_graph_of_rows_off_their_alignment(dtype, parts, late):
    """`late`: the last part begins between vectors, which sends all of them element by element."""
    outs, lses = _parts(parts, 40, 3, 64, dtype, 60 + parts)
    want = oracle.merge_exact(outs, lses)
    outs, lses = [o.cuda() for o in outs], [l.cuda() for l in lses]
    if late:
        flat = torch.empty(outs[-1].numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = outs[-1].flatten()
        outs[-1] = flat[1:].view(40, 3, 64)
    ops.merge_attention(outs, lses)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = ops.merge_attention(outs, lses)
    out.zero_()
    graph.replay()
    within(out, want[0], want[1], "outputs")
    within(lse, want[2], want[3], "log-sum-exps")
