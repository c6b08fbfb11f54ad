"""Attention over shared prefixes, joined parts and expanded latent prompts on the CPU: restatements against 64 bits, refusals."""
import pytest
import torch

import shared_attn_oracle as oracle
from shared_attn_oracle import run_latent, run_shared, within
from metrale_inference_alpha_b200 import ops
from metrale_inference_alpha_b200.ops import mla_prompt, shared_attn


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("ctx,prefix,start,n", [([3, 20, 1], [50], [0, 3], 1), ([9, 4, 30, 5, 0], [17, 40], [0, 2, 4], 3), ([0, 7, -2], [5, 0], [1, 1, 2], 1), ([6, 2], [], [0], 2)])
def test_shared_prefix(fp8, ctx, prefix, start, n):
    c = oracle.shared(1, ctx, prefix, start, 4, 2, 64, fp8, block=8, n=n)
    out, tol, lse, ltol = oracle.shared_exact(c)
    a, b = run_shared(c)
    within(a, out, tol, "outputs")
    within(b, lse, ltol, "log-sum-exps")
    assert torch.equal(run_shared(c, return_lse=False), a)


def test_shared_prefix_is_attention_over_one_sequence():
    """Prefix blocks in front of a sequence's own give what the operator gives."""
    c = oracle.shared(2, [9, 20, 4], [32], [0, 3], 4, 2, 64, False)
    table = torch.cat([c["prefix_table"][:, :2].expand(3, -1), c["table"]], 1).contiguous()
    one = ops.paged_attention(c["q"], c["k"].nan_to_num(), c["v"].nan_to_num(), table, torch.arange(3, dtype=torch.int32), torch.ones(3, dtype=torch.int32), c["ctx"] + 32,
                              max_q_len=1, max_ctx=52, scale=c["scale"])
    torch.testing.assert_close(run_shared(c)[0].float(), one.float(), rtol=2 ** -7, atol=1e-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("parts", [1, 2, 16])
def test_merge(dtype, parts):
    g = torch.Generator().manual_seed(3)
    outs = [torch.randn(7, 3, 20, generator=g).to(dtype) for _ in range(parts)]
    lses = [torch.randn(7, 3, generator=g) * 5 for _ in range(parts)]
    lses[-1][2], outs[-1][2] = -float("inf"), float("nan")
    out, tol, lse, ltol = oracle.merge_exact(outs, lses)
    a, b = ops.merge_attention(outs, lses)
    within(a, out, tol, "outputs")
    within(b, lse, ltol, "log-sum-exps")


def test_two_tiers_of_prefixes():
    """A prefix of all sequences and one of some: the former attended on its own, joined with the rest."""
    c = oracle.shared(4, [5, 3, 8, 2], [24, 40, 16], [0, 4, 4, 4], 4, 2, 64, False, block=8)
    empty = torch.zeros(4, dtype=torch.int32)
    tier = lambda rows, start, ctx: run_shared({**c, "prefix": c["prefix"][rows], "prefix_table": c["prefix_table"][rows], "start": torch.tensor(start, dtype=torch.int32),
                                                "ctx": ctx})
    first, second = tier(slice(0, 1), [0, 4], empty), tier(slice(1, 3), [0, 2, 4], c["ctx"])
    out, lse = ops.merge_attention([first[0], second[0]], [first[1], second[1]])
    for s in range(4):
        z, v = [], []
        for t, i, n in ((c["prefix_table"], 0, 24), (c["prefix_table"], 1 + s // 2, 40 if s < 2 else 16), (c["table"], s, int(c["ctx"][s]))):
            k = oracle._rows(c["k"], t[i], n)
            z.append(torch.einsum("hgd,nhd->hgn", c["q"][s].double().view(2, 2, 64), k) * c["scale"])
            v.append(oracle._rows(c["v"], t[i], n))
        z = torch.cat(z, -1)
        want = torch.einsum("hgn,nhd->hgd", torch.softmax(z, -1), torch.cat(v)).reshape(4, 64)
        torch.testing.assert_close(out[s].double(), want, rtol=2 ** -6, atol=2 ** -7)      # outputs of two parts and the join in bf16
        torch.testing.assert_close(lse[s].double(), torch.logsumexp(z, -1).reshape(4), rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("new,ctx,heads", [([5, 1], [5, 9], 2), ([12], [40], 1), ([3, 7, 2], [3, 0, 30], 2)])
def test_latent_prompt(new, ctx, heads):
    c = oracle.latent(5, new, ctx, heads, block=8)
    out, tol = oracle.latent_exact(c)
    within(run_latent(c), out, tol, "outputs")


def test_latents_that_are_no_numbers_stay_visible_to_those_who_see_them():
    c = oracle.latent(6, [6], [10], 2, block=8)
    c["cache"].flatten(0, 1)[int(c["table"][0, 0]) * 8 + 7, 0, 5] = float("nan")
    out = run_latent(c)
    assert bool(out[:3].isfinite().all()) and bool(out[3:].isnan().all())


BAD = [dict(q_len=2), dict(max_prefix=1000), dict(max_ctx=1000), dict(scale=0.0), dict(max_prefix=-1), dict(max_ctx=19), dict(max_prefix=49)]


@pytest.mark.parametrize("kw", BAD, ids=str)
def test_shared_prefix_refuses_numbers(kw):
    c = oracle.shared(7, [3, 20, 1], [50], [0, 3], 4, 2, 64, False)
    with pytest.raises(ValueError, match="shared_prefix_attention"):
        run_shared(c, **kw)


@pytest.mark.parametrize("name,change", [
    ("q", lambda x: x.float()), ("q", lambda x: x[:2]), ("q", lambda x: torch.cat([x, x], 1)[:, ::2]), ("k", lambda x: x.float()), ("v", lambda x: x[:-1]),
    ("k", lambda x: x.transpose(1, 2)), ("ctx", lambda x: x.long()), ("ctx", lambda x: x + 100), ("prefix", lambda x: x + 1), ("prefix", lambda x: x[None]),
    ("start", lambda x: x[:1]), ("start", lambda x: x + 1), ("start", lambda x: x.flip(0)), ("prefix_table", lambda x: x + 100), ("table", lambda x: x - 100),
    ("table", lambda x: x.t().contiguous().t() if x.shape[1] > 1 else x.long()), ("prefix_table", lambda x: x.long()), ("table", lambda x: x[:1])])
def test_shared_prefix_refuses_tensors(name, change):
    c = oracle.shared(8, [3, 20, 1], [50], [0, 3], 4, 2, 64, False)
    with pytest.raises(ValueError, match="shared_prefix_attention"):
        run_shared({**c, name: change(c[name])})


def test_shared_prefix_refuses_shapes():
    for heads, kv_heads, dim in ((4, 2, 96), (65, 1, 64)):
        with pytest.raises(ValueError, match="head"):
            run_shared(oracle.shared(9, [3], [5], [0, 1], heads, kv_heads, dim, False))
    c = oracle.shared(9, [3], [5], [0, 1], 4, 2, 64, True)
    with pytest.raises(ValueError, match="scales"):
        run_shared(c, k_scale=None)
    with pytest.raises(ValueError, match="scales"):
        run_shared(c, v_scale=torch.ones(2))
    with pytest.raises(ValueError, match="even"):
        run_shared(oracle.shared(9, [3], [5], [0, 1], 4, 2, 64, True, block=7))
    c = oracle.shared(9, [1] * 1025, [1] * 1025, list(range(1026)), 1, 1, 64, False, block=1)
    with pytest.raises(ValueError, match="groups"):
        run_shared(c)


def test_merge_refuses():
    o, l = torch.zeros(3, 2, 8), torch.zeros(3, 2)
    for outs, lses in (([], []), ([o], [l, l]), ([o] * 17, [l] * 17), ([o, o.bfloat16()], [l, l]), ([o.half()], [l]), ([o, o[:2]], [l, l]), ([o], [l.double()]),
                       ([o], [l.t()]), ([o.transpose(0, 1)], [l]), ([o[0]], [l[0]])):
        with pytest.raises(ValueError, match="merge_attention"):
            ops.merge_attention(outs, lses)


@pytest.mark.parametrize("name,change", [
    ("q", lambda x: x.float()), ("q", lambda x: x[..., :128]), ("cache", lambda x: x[..., :512]), ("cache", lambda x: x.float()), ("w", lambda x: x[:, :128]),
    ("w", lambda x: x.float()), ("w", lambda x: x[:1]), ("w", lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)), ("ctx", lambda x: x + 30), ("q_len", lambda x: x + 9),
    ("q_start", lambda x: x + 2), ("q_start", lambda x: x - 1), ("q_start", lambda x: x[:1]), ("table", lambda x: x + 50), ("table", lambda x: x.long())])
def test_latent_prompt_refuses_tensors(name, change):
    c = oracle.latent(10, [5, 1], [5, 9], 2, block=8)
    with pytest.raises(ValueError, match="mla_prompt_attention"):
        run_latent({**c, name: change(c[name])})


@pytest.mark.parametrize("kw", [dict(max_q_len=4), dict(max_ctx=8), dict(max_ctx=100), dict(total_ctx=13), dict(total_ctx=-1), dict(scale=-1.0), dict(max_q_len=-1)], ids=str)
def test_latent_prompt_refuses_numbers(kw):
    with pytest.raises(ValueError, match="mla_prompt_attention"):
        run_latent(oracle.latent(11, [5, 1], [5, 9], 2, block=8), **kw)


def test_calls_of_nothing():
    c = oracle.shared(12, [], [], [0], 4, 2, 64, False)
    out, lse = run_shared(c)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    out, lse = ops.merge_attention([torch.zeros(0, 2, 8)], [torch.zeros(0, 2)])
    assert out.shape == (0, 2, 8) and lse.shape == (0, 2)


def test_argument_structures():
    """Sizes that the library was built with."""
    lib = pytest.importorskip("ctypes").CDLL(str(shared_attn._native.LIB_PATH)) if shared_attn._native.available() else pytest.skip("not built")
    lib.mb_shared_attn_args.restype = shared_attn.C.c_size_t
    assert [lib.mb_shared_attn_args(i) for i in range(3)] == [shared_attn._SHARED_ARGS.size, shared_attn._MERGE_ARGS.size, mla_prompt._ARGS.size]
