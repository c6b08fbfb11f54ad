"""Edges of attention over shared prefixes, of joins and of expanded latent prompts, on the CPU: what is refused, and what restatements make of it."""
import pytest
import torch

import shared_attn_oracle as oracle
from metrale_inference_alpha_b200 import ops
from metrale_inference_alpha_b200.engine.batch import ForwardBatch
from metrale_inference_alpha_b200.models import mla
from metrale_inference_alpha_b200.ops import mla_prompt, shared_attn
from shared_attn_oracle import run_latent, run_shared, within


@pytest.mark.parametrize("kw,change", [(dict(max_prefix=0), {}), (dict(max_ctx=0), {}), (dict(max_prefix=0), dict(prefix=[0], start=[0, 9])),
                                       (dict(max_prefix=0), dict(prefix=[0], start=[1, 0]))], ids=str)
def test_maxima_of_zero_refuse_what_is_longer(kw, change):
    c = oracle.shared(1, [5, 9], [40], [0, 2], 4, 2, 64, False)
    c.update({k: torch.tensor(x, dtype=torch.int32) for k, x in change.items()})
    with pytest.raises(ValueError, match="shared_prefix_attention"):
        run_shared(c, **kw)


def test_tables_without_columns():
    c = oracle.shared(3, [5, 9], [40], [0, 2], 4, 2, 64, False)
    for name, lengths, most in (("prefix_table", "prefix", "max_prefix"), ("table", "ctx", "max_ctx")):
        d = {**c, lengths: torch.zeros_like(c[lengths]), most: 0}
        want, got = run_shared(d), run_shared({**d, name: c[name][:, :0]})
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("new,ctx,kw", [([5, 1], [5, 9], dict(max_q_len=0)), ([5], [9], dict(total_ctx=0)), ([5], [9], dict(max_ctx=0)), ([0], [9], dict(max_ctx=0, max_q_len=0))], ids=str)
def test_latent_prompts_of_nothing_refuse_what_is_longer(new, ctx, kw):
    with pytest.raises(ValueError, match="mla_prompt_attention"):
        run_latent(oracle.latent(4, new, ctx, 2), **kw)


def test_latent_prompts_without_rows_refuse_portions():
    c = oracle.latent(5, [5, 1], [5, 9], 2)
    with pytest.raises(ValueError, match="rows of q"):
        run_latent({**c, "q": c["q"][:0]})


@pytest.mark.parametrize("scale", [0.0, -1.0, 1e-46, 1e39, float("inf"), float("nan")])
def test_scales_beyond_32_bits_are_refused(scale):
    """The kernels would multiply a mask's -inf by zero, or scores by infinity."""
    with pytest.raises(ValueError, match="scale"):
        run_shared(oracle.shared(8, [5], [9], [0, 1], 4, 2, 64, False), scale=scale)
    with pytest.raises(ValueError, match="scale"):
        run_latent(oracle.latent(8, [5], [9], 2), scale=scale)


@pytest.mark.parametrize("most", [-1, 1 << 31, 10 ** 12])
def test_maxima_are_looked_at_without_groups_and_sequences(most):
    """What no group and no sequence needs goes to the library all the same."""
    c = oracle.shared(10, [5, 9], [40], [0, 2], 4, 2, 64, False)
    alone = {**c, "prefix": c["prefix"][:0], "prefix_table": c["prefix_table"][:0], "start": c["start"][:1]}
    with pytest.raises(ValueError, match="max_prefix"):
        run_shared(alone, max_prefix=most)
    run_shared(alone, max_prefix=1 << 20)
    nobody = {**c, **{k: c[k][:0] for k in ("q", "ctx", "table")}, "start": torch.zeros(2, dtype=torch.int32)}
    with pytest.raises(ValueError, match="max_ctx"):
        run_shared(nobody, max_ctx=most)
    e = oracle.latent(10, [5], [9], 2)
    with pytest.raises(ValueError, match="max_ctx"):
        run_latent({**e, **{k: e[k][:0] for k in ("q_start", "q_len", "ctx", "table")}}, max_ctx=most)


def test_merge_of_rows_without_dims():
    o, inf = torch.zeros(4, 1, 0), float("inf")
    out, lse = ops.merge_attention([o, o], [torch.zeros(4, 1), torch.tensor([[0.0], [inf], [float("nan")], [-inf]])])
    assert out.shape == (4, 1, 0) and lse[0, 0].item() == pytest.approx(0.6931472) and bool(lse[1:3].isnan().all()) and lse[3, 0].item() == 0.0


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
            a, b = run_shared(c, max_prefix=most)
            within(a, out, tol, "outputs")
            within(b, lse, ltol, "log-sum-exps")


@pytest.mark.parametrize("heads", [1, 16, 128])
@pytest.mark.parametrize("total,seqs", [(1, 1), (8192, 1), (12288, 3), (100_000, 64), (600_000, 200), (640_000, 1), (700_000, 1), (3_000_000, 9)])
def test_the_workspace_of_latent_prompts_is_bounded(total, seqs, heads):
    """Gathered rows count as well; with one head at a time nothing can be saved any more."""
    rows = mla_prompt._cached_rows(total, seqs)
    assert rows % 128 == 0 and rows >= total
    each = mla_prompt._heads_at_once(rows, heads)
    assert 1 <= each <= heads and (each == heads or rows * (1153 + 512 * (each + 1)) > 1 << 30)
    if not shared_attn._native.available():
        pytest.skip("not built")
    need = mla_prompt._library().mb_mla_prompt_ws(rows, seqs, each)
    assert mla_prompt.fits(total, seqs) == (rows * (1153 + 512) <= 1 << 30)
    assert not mla_prompt.fits(total, seqs) or need <= (1 << 30) + 1024            # 1024: parts begin on 256 bytes


def test_steps_beyond_the_workspace_stay_absorbed():
    def batch(n, front):
        return ForwardBatch.build([dict(tokens=[1] * n, start_pos=front, blocks=[1] * ((n + front) // 16 + 2))], 16)
    assert mla._expanded_pays(batch(8192, 600_000)) and not mla._expanded_pays(batch(8192, 700_000))


@pytest.mark.parametrize("starts,fine", [([0, 5, 6], True), ([3, 2, 0], True), ([0, 4, 6], False), ([2, 2, 0], False), ([0, 6, 4], False)], ids=str)
def test_latent_portions_that_share_rows_are_refused(starts, fine):
    c = oracle.latent(13, [5, 1, 2], [5, 9, 30], 2)
    c["q_start"] = torch.tensor(starts, dtype=torch.int32)
    if fine:
        run_latent(c)
        return
    with pytest.raises(ValueError, match="in common"):
        run_latent(c)
