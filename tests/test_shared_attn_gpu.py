"""Kernels of attention over shared prefixes, of joined parts and of prompts over an expanded latent cache, against 64 bits: tolerances are the oracle's bounds."""
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


def check_shared(c, **kw):
    want = oracle.shared_exact(c)
    out, lse = run_shared(cuda(c), **kw)
    within(out, want[0], want[1], "outputs")
    within(lse, want[2], want[3], "log-sum-exps")
    return out, lse


# ----------------------------------------------------------------------------- shared prefixes
SHAPES = [(4, 2, 64), (40, 8, 128), (8, 8, 128), (64, 1, 128), (24, 1, 64), (16, 2, 256), (3, 3, 256), (40, 1, 256)]
GROUPS = [([5, 90, 1], [700], [0, 3], 1), ([64, 0, 17, 3, 1, 40, 2], [129, 0, 1, 513], [1, 2, 4, 4, 6], 1), ([9, 20, 5, 33], [300, 127], [0, 1, 4], 4), ([70, 3], [], [0], 1),
          ([0, 0], [128], [0, 1], 1), ([1], [1], [0, 1], 1), ([2, 2, 2], [40], [0, 3], 5)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("ctx,prefix,start,n", GROUPS, ids=str)
def test_shared_prefix(fp8, heads, kv_heads, dim, ctx, prefix, start, n):
    check_shared(oracle.shared(20, ctx, prefix, start, heads, kv_heads, dim, fp8, n=n))


@pytest.mark.parametrize("block,fp8", [(1, False), (7, False), (24, False), (256, False), (2, True), (24, True), (48, True), (100, True)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (10, 2, 128), (6, 2, 256)])
def test_shared_prefix_block_sizes(block, fp8, heads, kv_heads, dim):
    check_shared(oracle.shared(21, [30, 7, 130, 1], [200, 391], [0, 2, 4], heads, kv_heads, dim, fp8, block=block))


@pytest.mark.parametrize("dim,heads,kv_heads,seqs", [(128, 10, 2, 90), (64, 8, 1, 70), (256, 8, 1, 45), (128, 40, 8, 31)])
@pytest.mark.parametrize("fp8", [False, True])
def test_many_rows_behind_one_prefix(dim, heads, kv_heads, seqs, fp8):
    """Several tiles of rows, the last of them ragged."""
    ctx = [1 + i * 7 % 50 for i in range(seqs)]
    check_shared(oracle.shared(22, ctx, [1000], [0, seqs], heads, kv_heads, dim, fp8))


@pytest.mark.parametrize("dim,heads,kv_heads,fp8", [(128, 10, 2, True), (128, 4, 4, False), (64, 8, 2, False), (256, 8, 1, False)])
def test_long_prefix(dim, heads, kv_heads, fp8):
    check_shared(oracle.shared(23, [3, 1200, 40], [40007], [0, 3], heads, kv_heads, dim, fp8))


def test_many_groups():
    n = 300
    check_shared(oracle.shared(24, [1 + i % 9 for i in range(n)], [i * 13 % 260 for i in range(n // 2)], [2 * i for i in range(n // 2 + 1)], 4, 2, 64, False))


def test_large_scores():
    """Scores hundreds of powers of two apart: all but a few weights vanish, and the rest keep their bound."""
    for fp8 in (False, True):
        check_shared(oracle.shared(25, [90, 3, 40], [300], [0, 3], 8, 2, 128, fp8, spread=40.0))


def test_small_queries_over_an_e4m3_cache():
    """Queries far below what f16 holds."""
    c = oracle.shared(26, [90, 3, 40], [300], [0, 3], 8, 2, 128, True)
    c["q"][1] *= 2.0 ** -30
    c["q"][2] *= 2.0 ** 20
    check_shared(c)


def test_queries_of_very_unequal_elements_over_an_e4m3_cache():
    """One element a thousand and a million times the others: these are held to 2^-17 of it."""
    for dim, kv_heads in ((64, 1), (128, 2), (256, 1)):
        c = oracle.shared(34, [40, 3], [300], [0, 2], 8, kv_heads, dim, True)
        c["q"][0, :, 5] *= 2.0 ** 10
        c["q"][1, :, 7] *= 2.0 ** 20
        check_shared(c)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_queries_that_are_no_numbers_over_an_e4m3_cache(dim):
    c = oracle.shared(35, [20, 20, 20], [150], [0, 3], 4, 2, dim, True)
    want = oracle.shared_exact(c)
    c["q"][0, 1, 3], c["q"][2, 0, 0] = float("nan"), float("inf")
    out, lse = run_shared(cuda(c))
    assert bool(out[0, 1].isnan().all()) and bool(out[2, 0].isnan().all())
    for r, h in ((0, 0), (0, 2), (1, 1), (2, 1), (2, 3)):
        within(out[r, h], want[0][r, h], want[1][r, h], f"row {r}, head {h}")


def test_more_sequences_than_a_launch_takes():
    n = 1100
    check_shared(oracle.shared(27, [1 + i % 5 for i in range(n)], [70], [0, n - 3], 4, 2, 64, False))


def test_keys_and_values_that_are_no_numbers():
    """A NaN key or value, or an infinite score, stays with the rows that see it."""
    c = oracle.shared(28, [20, 20, 20, 20], [50, 40], [0, 2, 3], 4, 2, 128, False, n=2)
    at = lambda t, s, j: (int(c[t][s, j // 16]), j % 16)
    c["k"][at("table", 0, 19)][0, 5] = float("nan")                # the last row of sequence 0: seen by its second token alone
    c["v"][at("prefix_table", 1, 39)][1, 7] = float("inf")
    c["v"][at("table", 3, 4)][0, 0] = float("nan")
    want = oracle.shared_exact(c)
    out, lse = run_shared(cuda(c))
    assert bool(out[0].isfinite().all()) and bool(out[1, :2].isnan().all()) and bool(out[1, 2:].isfinite().all()) and bool(lse[1, :2].isnan().all())
    assert bool((out[4:6, 2:, 7] == float("inf")).all()) and bool(out[4:6, :2].isfinite().all()) and bool(lse[4:6].isfinite().all())
    assert bool(out[6:, :2, 0].isnan().all()) and bool(out[6:, :, 1:].isfinite().all())
    for r, heads in ((0, slice(0, 4)), (2, slice(0, 4)), (3, slice(0, 4)), (1, slice(2, 4)), (4, slice(0, 2))):
        within(out[r, heads], want[0][r, heads], want[1][r, heads], f"outputs of row {r}")


def test_scores_of_minus_infinity():
    """A prefix all of whose scores are -inf leaves no weight; with nothing else the row gives zeros."""
    c = oracle.shared(29, [8, 0], [16], [0, 2], 2, 1, 64, False)
    c["q"][:, :, 0] = 1.0
    c["k"].flatten(0, 1)[int(c["prefix_table"][0, 0]) * 16:][:16, 0, 0] = -float("inf")
    want = oracle.shared_exact(c)
    out, lse = run_shared(cuda(c))
    within(out[:1], want[0][:1], want[1][:1], "outputs")
    assert bool((out[1] == 0).all()) and bool((lse[1] == -float("inf")).all())


def test_bad_places_are_reported():
    """Blocks that the cache does not have, lengths beyond the maxima, groups that leave the batch: the status word, and every other row as it should be."""
    base = oracle.shared(30, [20, 9, 33], [50, 70], [0, 1, 2], 4, 2, 128, False)
    want = oracle.shared_exact(base)
    for name, place, value, rows in (("table", (0, 0), 10 ** 6, [1, 2]), ("prefix_table", (1, 2), -5, [0, 2]), ("ctx", (2,), 10 ** 6, [0, 1]), ("prefix", (0,), 71, [1, 2]),
                                     ("start", (2,), 90, [0]), ("start", (0,), -3, [0, 1, 2])):
        c = {**base, name: base[name].clone()}
        c[name][place] = value
        c["k"], c["v"] = c["k"].nan_to_num(), c["v"].nan_to_num()
        out, lse = run_shared(cuda(c))
        with pytest.raises(_native.KernelError):
            ops.check_status("cuda")
        for r in rows:
            within(out[r], want[0][r], want[1][r], f"row {r} with a bad {name}")


def test_shared_prefix_in_a_graph_and_on_another_stream():
    c = cuda(oracle.shared(31, [20, 9, 33, 4], [600], [0, 4], 40, 8, 128, True))
    want = run_shared(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_shared(c)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(run_shared(c))
    # both at once, each over workspaces of its own
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
    # lengths are read by the replay
    c["ctx"].copy_(torch.tensor([1, 9, 2, 0]))
    c["prefix"].copy_(torch.tensor([333]))
    graphs[0].replay()
    again = run_shared(c)
    assert torch.equal(outs[0][0], again[0]) and torch.equal(outs[0][1], again[1])


def test_shared_prefix_agrees_with_attention_over_whole_sequences():
    c = cuda(oracle.shared(32, [40, 9, 100, 64], [640], [0, 4], 40, 8, 128, True))
    c["k"], c["v"] = torch.where(c["k"] == 0x7f, 0, c["k"]), torch.where(c["v"] == 0x7f, 0, c["v"])
    table = torch.cat([c["prefix_table"].expand(4, -1), c["table"]], 1).contiguous()
    one = ops.paged_attention(c["q"], c["k"], c["v"], table, torch.arange(4, dtype=torch.int32, device="cuda"), torch.ones(4, dtype=torch.int32, device="cuda"), c["ctx"] + 640,
                              max_q_len=1, max_ctx=740, scale=c["scale"], k_scale=c["k_scale"], v_scale=c["v_scale"])
    # two results in bf16 of weights in f16
    torch.testing.assert_close(run_shared(c)[0].float(), one.float(), rtol=2 ** -7, atol=2 ** -9)


def test_two_tiers_and_a_join():
    """A prefix of all sequences, one of some, their own rows: three tables, two calls and a join give what one table gives."""
    c = oracle.shared(33, [40, 9, 100, 64], [500, 300, 60], [0, 4, 4, 4], 40, 8, 128, False)
    first = run_shared(cuda({**c, "prefix": c["prefix"][:1], "prefix_table": c["prefix_table"][:1], "start": torch.tensor([0, 4], dtype=torch.int32),
                             "ctx": torch.zeros(4, dtype=torch.int32)}))
    second = run_shared(cuda({**c, "prefix": c["prefix"][1:], "prefix_table": c["prefix_table"][1:], "start": torch.tensor([0, 2, 4], dtype=torch.int32)}))
    out, lse = ops.merge_attention([first[0], second[0]], [first[1], second[1]])
    for s in range(4):
        places = [(c["prefix_table"][0], 500), (c["prefix_table"][1 + s // 2], 300 if s < 2 else 60), (c["table"][s], int(c["ctx"][s]))]
        k, v = (torch.cat([oracle._rows(c[x], t, n) for t, n in places]) for x in ("k", "v"))
        z = torch.einsum("hgd,nhd->hgn", c["q"][s].double().view(8, 5, 128), k) * c["scale"]
        want = torch.einsum("hgn,nhd->hgd", torch.softmax(z, -1), v).reshape(40, 128)
        size = torch.einsum("hgn,nhd->hgd", torch.softmax(z, -1), v.abs()).reshape(40, 128)
        # weights in bf16, two parts rounded to bf16 (each at most `size` in all), the join rounded
        within(out[s], want, 2.0 ** -8 * (2 * size + want.abs()) * 1.01 + 1e-4, f"outputs of sequence {s}")
        within(lse[s], torch.logsumexp(z, -1).reshape(40), torch.full((40,), 1e-4), "log-sum-exps")


# ----------------------------------------------------------------------------- joins
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("parts", [1, 2, 3, 16])
@pytest.mark.parametrize("rows,heads,dim", [(1, 1, 1), (128, 40, 128), (77, 3, 64), (9, 5, 20), (5, 2, 515), (2, 16, 512), (1000, 7, 8)])
def test_merge(dtype, parts, rows, heads, dim):
    g = torch.Generator().manual_seed(40)
    outs = [torch.randn(rows, heads, dim, generator=g).to(dtype) for _ in range(parts)]
    lses = [torch.randn(rows, heads, generator=g) * 5 for _ in range(parts)]
    for o, l in zip(outs, lses):
        none = torch.rand(rows, heads, generator=g) < 0.2
        l[none], o[none] = -float("inf"), float("nan")
    out, tol, lse, ltol = oracle.merge_exact(outs, lses)
    a, b = ops.merge_attention([o.cuda() for o in outs], [l.cuda() for l in lses])
    within(a, out, tol, "outputs")
    within(b, lse, ltol, "log-sum-exps")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_merge_of_rows_off_their_alignment(dtype):
    """Outputs that begin between vectors."""
    flat = torch.randn(4 * 3 * 16 + 1, device="cuda").to(dtype)
    outs = [flat[:-1].view(4, 3, 16), flat[1:].view(4, 3, 16)]
    lses = [torch.zeros(4, 3, device="cuda"), torch.ones(4, 3, device="cuda")]
    want = oracle.merge_exact([o.cpu() for o in outs], [l.cpu() for l in lses])
    within(ops.merge_attention(outs, lses)[0], want[0], want[1], "outputs")


def test_merge_of_what_is_no_number():
    o, l = torch.ones(3, 1, 8, device="cuda"), torch.zeros(3, 1, device="cuda")
    x = l.clone()
    x[0], x[1] = float("nan"), float("inf")
    out, lse = ops.merge_attention([o, o], [l, x])
    assert bool(out[:2].isnan().all()) and bool(lse[:2].isnan().all()) and bool((out[2] == 1).all())


# ----------------------------------------------------------------------------- latent prompts
def check_latent(c, **kw):
    want = oracle.latent_exact(c)
    out = run_latent(cuda(c), **kw)
    within(out, want[0], want[1], "outputs")
    return out


@pytest.mark.parametrize("new,ctx,heads", [([1], [1], 1), ([5, 1], [5, 9], 2), ([333], [333], 16), ([128, 300, 7], [128, 700, 600], 4), ([257], [1000], 3),
                                           ([3, 7, 200, 0], [3, 0, 150, 30], 2), ([129, 64], [129, 65], 128)], ids=str)
@pytest.mark.parametrize("block", [16, 24])
def test_latent_prompt(new, ctx, heads, block):
    check_latent(oracle.latent(50, new, ctx, heads, block=block))


def test_latent_prompt_of_a_long_context():
    check_latent(oracle.latent(51, [140, 3], [9001, 2050], 2))


def test_latent_prompt_without_a_bound_of_the_sum():
    c = oracle.latent(52, [40, 90, 5], [50, 300, 5], 2)
    a = run_latent(cuda(c))
    assert torch.equal(run_latent(cuda(c), total_ctx=None), a)


def test_latent_prompt_in_several_steps_of_heads(monkeypatch):
    c = cuda(oracle.latent(53, [140, 30], [200, 30], 5))
    a = run_latent(c)
    monkeypatch.setattr(mla_prompt, "_WS_BYTES", 2 * 384 * 256 * 2)
    assert torch.equal(run_latent(c), a)


def test_latent_prompt_of_large_scores():
    check_latent(oracle.latent(54, [200], [300], 2, spread=30.0))


def test_latents_that_are_no_numbers():
    """They make the rows that see them NaN, in whatever place of a tile, and no others."""
    c = oracle.latent(55, [300, 20], [400, 20], 3)
    want = oracle.latent_exact(c)
    flat = c["cache"].flatten(0, 1)
    flat[int(c["table"][0, 350 // 16]) * 16 + 350 % 16, 0, 17] = float("inf")
    flat[int(c["table"][1, 0]) * 16 + 3, 0, 575] = float("nan")
    out = run_latent(cuda(c))
    assert bool(out[250:300].isnan().all()) and bool(out[303:].isnan().all())
    for rows in (slice(0, 250), slice(300, 303)):
        within(out[rows], want[0][rows], want[1][rows], "outputs")


def test_latent_prompt_leaves_rows_of_no_sequence():
    c = cuda(oracle.latent(56, [40, 50], [40, 90], 2))
    a = run_latent(c)
    wide = {**c, "q": torch.cat([c["q"][:3], c["q"], c["q"][:9]]).contiguous(), "q_start": c["q_start"] + 3}
    assert torch.equal(run_latent(wide)[3:93], a)


def test_latent_prompt_reports_bad_places():
    base = oracle.latent(57, [40, 50, 10], [40, 90, 30], 2)
    want = oracle.latent_exact(base)
    for name, place, value, rows in (("table", (1, 2), 10 ** 6, slice(0, 40)), ("q_start", (2,), 95, slice(0, 90)), ("ctx", (2,), 10 ** 6, slice(0, 90)),
                                     ("q_len", (2,), 10 ** 6, slice(0, 90))):
        c = {**base, name: base[name].clone(), "cache": base["cache"].nan_to_num()}
        c[name][place] = value
        out = run_latent(cuda(c))
        with pytest.raises(_native.KernelError):
            ops.check_status("cuda")
        within(out[rows], want[0][rows], want[1][rows], f"rows with a bad {name}")


def test_latent_prompt_in_a_graph():
    c = cuda(oracle.latent(58, [140, 30], [200, 60], 16))
    want = run_latent(c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run_latent(c)
    out.zero_()
    g.replay()
    assert torch.equal(out, want)


def test_latent_prompt_agrees_with_the_absorbed_form():
    from metrale_inference_alpha_b200.ops import mla_cuda
    c = cuda(oracle.latent(59, [200, 64], [200, 500], 16))
    uk, uv = c["w"][:, :128], c["w"][:, 128:]
    lat = torch.einsum("thd,hdl->thl", c["q"][..., :128].float(), uk.float())
    qq = torch.cat([lat.bfloat16(), c["q"][..., 128:]], -1).contiguous()
    o = mla_cuda.mla_attention(qq, c["cache"].nan_to_num(), c["table"], c["q_start"], c["q_len"], c["ctx"], max_q_len=200, max_ctx=500, scale=c["scale"])
    want = torch.einsum("thl,hvl->thv", o, uv.float())
    got = run_latent(c).float()
    # roundings of queries, keys, values and weights to bf16 on either side, of values of about one over 64 tokens and more
    assert float((got - want).abs().max()) < 0.05 and float((got - want).square().mean().sqrt()) < 0.004


def test_a_latent_prompt_with_more_cached_tokens_than_stated_is_left_out():
    c = oracle.latent(60, [30, 20], [64, 48], 4)
    want = oracle.latent_exact(c)
    out = run_latent(cuda(c), max_ctx=48, total_ctx=96)
    with pytest.raises(_native.KernelError):
        ops.check_status("cuda")
    within(out[30:], want[0][30:], want[1][30:], "the other sequence")


def test_calls_one_behind_the_other_without_a_pause():
    """Calls of several kinds follow one another on a stream and take up each other's workspace: every one gives what it gives alone."""
    cases = [(run_shared, cuda(oracle.shared(61, [20, 9, 33, 4, 700], [600], [0, 4], 40, 8, 128, True))), (run_shared, cuda(oracle.shared(62, [3], [2000], [0, 1], 8, 1, 64, False))),
             (run_latent, cuda(oracle.latent(63, [140, 30], [200, 60], 16))), (run_shared, cuda(oracle.shared(64, [50, 1], [90, 30], [0, 1, 2], 16, 2, 256, True, n=3))),
             (run_latent, cuda(oracle.latent(65, [5], [1500], 2)))]
    flat = lambda x: x if isinstance(x, tuple) else (x,)
    alone = []
    for run, c in cases:
        alone.append([t.clone() for t in flat(run(c))])
        torch.cuda.synchronize()
    kept = [(i, flat(cases[i][0](cases[i][1]))) for _ in range(8) for i in (0, 1, 2, 3, 4, 3, 1, 0, 2)]
    joined = [ops.merge_attention([o[0], o[0]], [o[1], o[1]]) for i, o in kept if len(o) == 2]
    for i, o in kept:
        assert all(torch.equal(a, b) for a, b in zip(o, alone[i])), i
    for (i, o), (out, lse) in zip([k for k in kept if len(k[1]) == 2], joined):
        assert torch.equal(out, o[0])


def test_calls_on_two_streams_at_once():
    cases = [(run_shared, cuda(oracle.shared(66, [20, 9, 33, 4], [3000], [0, 4], 40, 8, 128, True))), (run_latent, cuda(oracle.latent(67, [300], [900], 8)))]
    alone = [run(c) for run, c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for k, (run, c) in enumerate(cases):
            with torch.cuda.stream(streams[k]):
                got[k].append(run(c))
    torch.cuda.synchronize()
    assert all(torch.equal(o[0], alone[0][0]) and torch.equal(o[1], alone[0][1]) for o in got[0]) and all(torch.equal(o, alone[1]) for o in got[1])


@pytest.mark.parametrize("seed", range(12))
def test_shared_prefixes_of_random_shapes(seed):
    g = torch.Generator().manual_seed(1000 + seed)
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))
    S, n = pick(1, 40), pick(1, 4)
    dim = (64, 128, 256)[pick(0, 2)]
    kv = pick(1, 5)
    heads = kv * pick(1, 12)
    groups = pick(0, 5)
    start = sorted(pick(0, S) for _ in range(groups + 1)) if groups else [0]
    prefix = [pick(0, 900) if pick(0, 3) else pick(0, 3) for _ in range(groups)]
    ctx = [pick(0, 1) if pick(0, 4) == 0 else pick(0, 150) for _ in range(S)]
    check_shared(oracle.shared(2000 + seed, ctx, prefix, start, heads, kv, dim, bool(seed & 1), block=(16, 32, 8, 6)[seed % 4], n=n))


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 8, 128), (8, 4, 256), (32, 16, 64)])
def test_shared_prefixes_in_a_cache_beyond_32_bits(heads, kv_heads, dim):
    c = cuda(oracle.shared(68, [20, 90, 3], [300], [0, 3], heads, kv_heads, dim, False))
    want = run_shared(c)
    blocks = 150_000                                             # 16 tokens of 2048 bytes of K: 4.9 GB
    front = blocks - c["k"].shape[0]
    big = {**c, "table": c["table"] + front, "prefix_table": c["prefix_table"] + front}
    for name in ("k", "v"):
        big[name] = torch.empty(blocks, *c[name].shape[1:], dtype=torch.bfloat16, device="cuda")
        big[name][front:] = c[name]
    got = run_shared(big)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_latent_prompt_in_a_cache_beyond_32_bits():
    c = cuda(oracle.latent(69, [140, 30], [200, 60], 8))
    want = run_latent(c)
    blocks = 250_000                                             # 16 tokens of 1152 bytes: 4.6 GB
    front = blocks - c["cache"].shape[0]
    big = torch.empty(blocks, 16, 1, 576, dtype=torch.bfloat16, device="cuda")
    big[front:] = c["cache"]
    assert torch.equal(run_latent({**c, "cache": big, "table": c["table"] + front}), want)


@pytest.mark.parametrize("new,ctx,heads", [([257], [257], 1), ([100, 300], [129, 641], 3), ([40, 8, 30], [384, 8, 1500], 21), ([64], [1200], 80), ([16] * 9, [130] * 9, 5)])
def test_latent_prompt_rows_of_many_heads(new, ctx, heads):
    """Units of the expansion that begin and end inside a run of heads, odd numbers of 128 rows, more pairs of CTAs than units and fewer."""
    c = oracle.latent(70, new, ctx, heads)
    want = oracle.latent_exact(c)
    within(run_latent(cuda(c)), want[0], want[1], "outputs")
