"""Edges of attention over shared prefixes, of joins and of expanded latent prompts, on the kernels: what is reported, and calls at the ends of what is allowed."""
import pytest
import torch

import shared_attn_oracle as oracle
from metrale_inference_alpha_b200 import ops
from metrale_inference_alpha_b200.ops import _native, mla_prompt
from shared_attn_oracle import run_latent, run_shared, within

pytestmark = pytest.mark.gpu


def cuda(c):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}


@pytest.fixture(autouse=True)
def _status():
    yield
    ops.check_status("cuda")


def reported():
    with pytest.raises(_native.KernelError):
        ops.check_status("cuda")


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 2), (256, 4, 1)])
def test_maxima_of_zero_report_what_is_longer(dim, heads, kv_heads):
    """Without a kernel over the prefixes, or over own rows, their lengths and groups are looked at all the same."""
    c = oracle.shared(1, [5, 9, 0], [40], [0, 2], heads, kv_heads, dim, False)
    none = lambda n: torch.zeros(n, dtype=torch.int32)
    for kw, change, seen in ((dict(max_prefix=0), {}, dict(prefix=none(1))), (dict(max_ctx=0), {}, dict(ctx=none(3))),
                             (dict(max_prefix=0, max_ctx=0), {}, dict(prefix=none(1), ctx=none(3))),
                             (dict(max_prefix=0), dict(prefix=none(1), start=torch.tensor([0, 9], dtype=torch.int32)), dict(prefix=none(1))),
                             (dict(max_prefix=0), dict(prefix=none(1), start=torch.tensor([-1, 2], dtype=torch.int32)), dict(prefix=none(1)))):
        out, lse = run_shared(cuda({**c, **change}), **kw)
        reported()
        want = oracle.shared_exact({**c, **seen})
        within(out, want[0], want[1], "outputs")
        within(lse, want[2], want[3], "log-sum-exps")
        # with lengths that the maxima allow nothing is reported
        run_shared(cuda({**c, **seen}), **kw)
        ops.check_status("cuda")


def test_a_cache_without_blocks():
    """It holds nothing, which is all that such a call may ask for."""
    c = cuda(oracle.shared(2, [0, 0], [0], [0, 2], 4, 2, 64, False))
    c.update(k=c["k"][:0], v=c["v"][:0])
    out, lse = run_shared(c)
    assert bool((out == 0).all()) and bool((lse == -float("inf")).all())
    ops.check_status("cuda")
    c["ctx"][1] = 3
    run_shared(c)
    reported()


def test_tables_without_columns():
    """A maximum of 0 needs no table: prefixes of which a step has none, sequences that have nothing of their own."""
    c = oracle.shared(3, [5, 9], [40], [0, 2], 4, 2, 64, False)
    for name, lengths, most in (("prefix_table", "prefix", "max_prefix"), ("table", "ctx", "max_ctx")):
        d = {**c, lengths: torch.zeros_like(c[lengths]), most: 0}
        want = run_shared(cuda(d))
        got = run_shared(cuda({**d, name: c[name][:, :0]}))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("new,ctx,kw", [([5, 1], [5, 9], dict(max_q_len=0)), ([5], [9], dict(total_ctx=0)), ([5], [9], dict(max_ctx=0)), ([0], [9], dict(max_ctx=0, max_q_len=0)),
                                        ([0] * 300, [0] * 299 + [3], dict(max_ctx=2, max_q_len=0))], ids=lambda x: str(x)[:40])
def test_latent_prompts_of_nothing_report_what_is_longer(new, ctx, kw):
    out = run_latent(cuda(oracle.latent(4, new, ctx, 2)), **kw)
    assert bool((out == 0).all())
    reported()


def test_latent_prompts_of_nothing():
    """What the maxima and the sum allow is not reported: portions without rows, sequences without cached tokens, q without rows, no sequences."""
    c = oracle.latent(5, [5, 1], [5, 9], 2)
    none = torch.zeros(2, dtype=torch.int32)
    one = oracle.latent(6, [4], [0], 2)
    for d in ({**c, "q_len": none, "max_q_len": 0}, {**c, "q_len": none, "q": c["q"][:0]}, {**one, "max_ctx": 0}, {**one, "max_ctx": 0, "table": one["table"][:, :0]},
              {**c, "ctx": none, "max_ctx": 0, "total_ctx": 0, "table": c["table"][:, :0], "cache": c["cache"][:0]},
              {**c, **{k: c[k][:0] for k in ("q_start", "q_len", "ctx", "table")}}):
        assert bool((run_latent(cuda(d)) == 0).all())
        ops.check_status("cuda")
    run_latent(cuda({**c, "q": c["q"][:0]}))
    reported()


@pytest.mark.parametrize("scale", [0.0, -0.0, -0.0625, 1e-30, float("nan")])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (10, 2, 128), (8, 1, 256)])
@pytest.mark.parametrize("seqs", [3, 60])
def test_scales_of_an_e4m3_cache_at_their_ends(heads, kv_heads, dim, scale, seqs):
    """A scale of zero makes scores equal, a negative one turns them, one that is no number leaves none; prefixes that end inside a tile, one tile of rows and several."""
    c = oracle.shared(7, [1 + i * 31 % 90 for i in range(seqs)], [300, 129], [0, seqs - 1, seqs], heads, kv_heads, dim, True)
    c["k_scale"] = torch.tensor([scale])
    want = oracle.shared_exact(c)
    out, lse = run_shared(cuda(c))
    within(out, want[0], want[1], "outputs")
    within(lse, want[2], want[3], "log-sum-exps")


@pytest.mark.parametrize("scale", [2.0 ** -126, 2.0 ** -60])
def test_the_smallest_scales(scale):
    """Scores are all but equal; columns that are masked have no weight all the same."""
    for fp8 in (False, True):
        c = {**oracle.shared(9, [5, 90, 1], [300], [0, 3], 10, 2, 128, fp8), "scale": scale}
        want = oracle.shared_exact(c)
        out, lse = run_shared(cuda(c))
        within(out, want[0], want[1], "outputs")
        within(lse, want[2], want[3], "log-sum-exps")
    c = {**oracle.latent(9, [140], [300], 2), "scale": scale}
    want = oracle.latent_exact(c)
    within(run_latent(cuda(c)), want[0], want[1], "outputs")


def test_merge_of_rows_without_dims():
    """The log-sum-exps are those of rows with dims."""
    inf = float("inf")
    lses = [torch.zeros(4, 1, device="cuda"), torch.tensor([[0.0], [inf], [float("nan")], [-inf]], device="cuda")]
    none, some = (ops.merge_attention([torch.zeros(4, 1, d, device="cuda")] * 2, lses) for d in (0, 8))
    assert none[0].shape == (4, 1, 0)
    torch.testing.assert_close(none[1], some[1], rtol=1e-6, atol=1e-6, equal_nan=True)


@pytest.mark.parametrize("start", [[0, 0], [0, 0, 2], [0, 2, 2], [2, 2, 2]], ids=str)
def test_groups_without_sequences_are_not_looked_at(start):
    """Their lengths and tables may be of another step."""
    c = oracle.shared(11, [5, 9], [40, 24], [0, 1, 2], 4, 2, 64, False)
    n = len(start) - 1
    c.update(start=torch.tensor(start, dtype=torch.int32), prefix=c["prefix"][:n].clone(), prefix_table=c["prefix_table"][:n].clone())
    out, tol, lse, ltol = oracle.shared_exact(c)
    for g in range(n):
        if start[g] == start[g + 1]:
            c["prefix"][g], c["prefix_table"][g] = 10 ** 6, -1
    for most in (c["max_prefix"], 0):
        if most or all(a == b for a, b in zip(start, start[1:])):
            a, b = run_shared(cuda(c), max_prefix=most)
            within(a, out, tol, "outputs")
            within(b, lse, ltol, "log-sum-exps")


@pytest.mark.parametrize("heads_at_once", [5, 3, 2, 1])
def test_the_workspace_of_latent_prompts_is_bounded(heads_at_once, monkeypatch):
    c = cuda(oracle.latent(12, [140, 30], [2000, 300], 5))
    want = run_latent(c)
    rows = mla_prompt._cached_rows(2300, 2)
    most = rows * (1153 + 512 * heads_at_once) + 600
    monkeypatch.setattr(mla_prompt, "_WS_BYTES", most)
    assert mla_prompt._heads_at_once(rows, 5) == heads_at_once
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = run_latent(c)
    assert torch.equal(got, want)
    assert torch.cuda.max_memory_allocated() - before <= most + 2048 + got.numel() * 2          # parts begin on 256 bytes, tensors on 512


@pytest.mark.parametrize("heads,kv_heads,dim,n", [(10, 2, 128, 40), (8, 1, 64, 129), (4, 2, 256, 17)])
@pytest.mark.parametrize("fp8", [False, True])
def test_many_new_tokens(heads, kv_heads, dim, n, fp8):
    """More of them than some sequences have rows: the first see the prefix alone, or nothing."""
    c = oracle.shared(14, [n, 3, 2 * n + 5, 0], [200, 0, 70], [0, 1, 2, 3], heads, kv_heads, dim, fp8, n=n)
    want = oracle.shared_exact(c)
    out, lse = run_shared(cuda(c))
    within(out, want[0], want[1], "outputs")
    within(lse, want[2], want[3], "log-sum-exps")


def test_replays_with_other_groups():
    """A captured step whose groups, prefixes and tables are another step's by the time it is replayed, some of them empty."""
    c = cuda(oracle.shared(15, [20, 9, 33, 4, 50, 1], [600, 300, 129], [0, 2, 3, 6], 10, 2, 128, True))
    run_shared(c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = run_shared(c)
    for start, prefix, ctx in (([0, 2, 3, 6], [600, 300, 129], [20, 9, 33, 4, 50, 1]), ([0, 0, 0, 0], [0, 0, 0], [20, 9, 33, 4, 50, 1]), ([1, 1, 4, 5], [600, 299, 0], [0, 9, 1, 4, 0, 1]),
                               ([0, 6, 6, 6], [513, 0, 0], [0, 0, 0, 0, 0, 0])):
        for name, x in (("start", start), ("prefix", prefix), ("ctx", ctx)):
            c[name].copy_(torch.tensor(x, dtype=torch.int32))
        out.zero_()
        graph.replay()
        want = oracle.shared_exact({k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in c.items()})
        within(out, want[0], want[1], f"outputs with groups {start}")
        within(lse, want[2], want[3], f"log-sum-exps with groups {start}")


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 16, 128), (16, 8, 256), (64, 32, 64)])
def test_an_e4m3_cache_beyond_32_bits(heads, kv_heads, dim):
    c = cuda(oracle.shared(16, [20, 90, 3], [300], [0, 3], heads, kv_heads, dim, True))
    want = run_shared(c)
    blocks = 150_000                                             # 16 tokens of 2048 bytes of K: 4.9 GB
    front = blocks - c["k"].shape[0]
    big = {**c, "table": c["table"] + front, "prefix_table": c["prefix_table"] + front}
    for name in ("k", "v"):
        big[name] = torch.empty(blocks, *c[name].shape[1:], dtype=torch.uint8, device="cuda")
        big[name][front:] = c[name]
    got = run_shared(big)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
