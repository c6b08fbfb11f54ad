"""64-bit oracle of attention over shared prefixes, of joined parts and of prompts over an expanded latent cache, with bounds of what kernels may be off by,
and cases for them, shared by the CPU and the GPU tests."""
import math

import torch

from metrale_inference_alpha_b200 import ops


def run_shared(c, **kw):
    a = dict(max_prefix=c["max_prefix"], max_ctx=c["max_ctx"], scale=c["scale"], q_len=c["n"], k_scale=c["k_scale"], v_scale=c["v_scale"], return_lse=True) | kw
    return ops.shared_prefix_attention(c["q"], c["k"], c["v"], c["prefix_table"], c["prefix"], c["start"], c["table"], c["ctx"], **a)


def run_latent(c, **kw):
    a = dict(max_q_len=c["max_q_len"], max_ctx=c["max_ctx"], scale=c["scale"], total_ctx=c["total_ctx"]) | kw
    return ops.mla_prompt_attention(c["q"], c["cache"], c["table"], c["q_start"], c["q_len"], c["ctx"], c["w"], **a)


def within(got, want, tol, what):
    got = got.double().cpu()
    same = (got == want) | (got.isnan() & want.isnan())
    far = torch.where(same, 0.0, (got - want).abs() - tol)
    assert bool((far <= 0).all()), f"{what}: {int((~(far <= 0)).sum())} of {far.numel()} beyond their bound, by up to {float(far.max()):.3g} at {int(far.argmax())}"


class Pool:
    """A paged cache whose rows are handed out block by block in shuffled order; what no sequence holds is NaN."""

    def __init__(self, gen, lengths, block):
        self.block, self.blocks = block, sum((n + block - 1) // block for n in lengths) + 1
        perm = (torch.randperm(self.blocks - 1, generator=gen) + 1).tolist() if self.blocks > 1 else []
        self.dead, self.rows = torch.ones(self.blocks * block, dtype=torch.bool), []
        for n in lengths:
            mine = [perm.pop() for _ in range((n + block - 1) // block)]
            self.rows.append(mine)
            for j in range(n):
                self.dead[mine[j // block] * block + j % block] = False

    def table(self, which):
        per = max([1] + [len(self.rows[i]) for i in which])
        t = torch.zeros(len(which), per, dtype=torch.int32)
        for r, i in enumerate(which):
            t[r, :len(self.rows[i])] = torch.tensor(self.rows[i], dtype=torch.int32)
        return t


def shared(seed, ctx, prefix, start, heads, kv_heads, dim, fp8, block=16, n=1, spread=1.5):
    """Sequences with `ctx` rows of their own in groups `start` behind prefixes of length `prefix`."""
    g = torch.Generator().manual_seed(seed)
    S, P = len(ctx), len(prefix)
    lengths = [max(0, x) for x in ctx] + [max(0, x) for x in prefix]
    pool = Pool(g, lengths, block)
    ints = lambda x: torch.tensor(x, dtype=torch.int32)
    c = dict(table=pool.table(range(S)), prefix_table=pool.table(range(S, S + P)), ctx=ints(ctx), prefix=ints(prefix), start=ints(start), n=n, scale=dim ** -0.5,
             max_ctx=max([0] + ctx), max_prefix=max([0] + prefix), k_scale=None, v_scale=None)
    for name in ("k", "v"):
        x = torch.randn(pool.blocks * block, kv_heads, dim, generator=g)
        x = (x * 16).to(torch.float8_e4m3fn).view(torch.uint8) if fp8 else x.bfloat16()
        x[pool.dead] = 0x7f if fp8 else float("nan")
        c[name] = x.view(pool.blocks, block, kv_heads, dim)
        if fp8:
            c[name + "_scale"] = torch.tensor([0.0625 if name == "k" else 0.05])
    c["q"] = (torch.randn(S * n, heads, dim, generator=g) * spread).bfloat16()
    return c


def _rows(cache, table, n, scale=None):
    bs, j = cache.shape[1], torch.arange(n)
    x = cache.flatten(0, 1)[table.long()[j // bs] * bs + j % bs]
    return x.view(torch.float8_e4m3fn).double() * scale.double() if cache.dtype == torch.uint8 else x.double()


def score_error(q, k, scale, fp8):
    """What scores [h, g, n] may be off by, natural logarithm, at most: a 32-bit sum of exact products, each addition off by up to 2^-23 of the sum of their
    sizes (a matrix unit may cut instead of round); over an e4m3 cache queries are sums of two e4m3 numbers, exact but for elements that are less
    than 2^-9 of the row's largest, which are off by 2^-17 of it or themselves."""
    e = q.shape[-1] * 2.0 ** -23 * torch.einsum("hgd,nhd->hgn", q.abs(), k.abs()).nan_to_num(posinf=0.0).amax()
    if fp8:
        top = q.abs().amax(-1, keepdim=True)
        off = torch.where(q.abs() < 2.0 ** -9 * top, torch.minimum(q.abs(), 2.0 ** -17 * top), 0.0)
        e = e + torch.einsum("hgd,nhd->hgn", off, k.abs()).nan_to_num(posinf=0.0).amax()
    return float(e) * scale


def _softmax(z):
    """Weights over the last dim and their log-sum-exp; a row of nothing but -inf has none."""
    lse = torch.logsumexp(z, -1)
    return torch.where((lse == -math.inf)[..., None], 0.0, torch.exp(z - lse[..., None])), lse


def shared_exact(c):
    """(out, its bound, lse, its bound)."""
    T, Hq, D = c["q"].shape
    H, n = c["k"].shape[2], c["n"]
    G = Hq // H
    out, tol = (torch.zeros(T, Hq, D, dtype=torch.float64) for _ in range(2))
    lse, ltol = torch.full((T, Hq), -math.inf, dtype=torch.float64), torch.zeros(T, Hq, dtype=torch.float64)
    start = c["start"].tolist()
    for s in range(len(c["ctx"])):
        own = max(0, int(c["ctx"][s]))
        k, v = _rows(c["k"], c["table"][s], own, c["k_scale"]), _rows(c["v"], c["table"][s], own, c["v_scale"])
        p = 0
        for g, (a, b) in enumerate(zip(start, start[1:])):
            if a <= s < b:
                p = max(0, int(c["prefix"][g]))
                k = torch.cat([_rows(c["k"], c["prefix_table"][g], p, c["k_scale"]), k])
                v = torch.cat([_rows(c["v"], c["prefix_table"][g], p, c["v_scale"]), v])
        for t in range(n):
            m, r = p + max(0, own - n + t + 1), s * n + t
            if m == 0:
                continue
            q = c["q"][r].double().view(H, G, D)
            z = torch.einsum("hgd,nhd->hgn", q, k[:m]) * c["scale"]
            w, l = _softmax(z)
            e = score_error(q, k[:m], c["scale"], c["k"].dtype == torch.uint8) + 2.0 ** -21          # and exponentials, of a row's own and of a join
            o, a = torch.einsum("hgn,nhd->hgd", w, v[:m]), torch.einsum("hgn,nhd->hgd", w, v[:m].abs())
            out[r], lse[r] = o.reshape(Hq, D), l.reshape(Hq)
            # weights rounded to bf16 (f16 for an e4m3 cache: finer, but what is under 2^-24 of the largest is lost), then the result
            tol[r] = (2.0 ** -8 * o.abs() + (2.0 ** -8 + 4 * e) * a + m * 2.0 ** -24 * v[:m].abs().nan_to_num().amax(0)[:, None]).reshape(Hq, D)
            # the sum of weights in 32 bits, in any order, and the result
            ltol[r] = (e + m * 2.0 ** -24 + 2.0 ** -23 * l.abs() + 2.0 ** -22).reshape(Hq)
    return out, tol, lse, ltol


def merge_exact(outs, lses):
    """(out, its bound, lse, its bound); bounds: a weight's exponential and its argument, one product and one sum a part in 32 bits, the result's type."""
    l = torch.stack(lses).double()
    lse = torch.logsumexp(l, 0)
    w = torch.where(l == -math.inf, 0.0, torch.exp(l - lse))[..., None]
    o = torch.where(w == 0, 0.0, torch.stack(outs).double())
    out, size = (w * o).sum(0), (w * o.abs()).sum(0)
    half = torch.finfo(outs[0].dtype).eps / 2
    n = len(outs)
    spread = torch.where(l == -math.inf, 0.0, (l - l.amax(0)).abs()).amax(0)[..., None]
    e = (spread + 4 + n) * 2.0 ** -23
    return out, half * out.abs() + 2 * e * size + 1e-38, lse, (e[..., 0] + 2.0 ** -23 * lse.abs()).nan_to_num()


def latent(seed, new, ctx, heads, block=16, spread=1.5):
    """Portions of `new` rows, the last of `ctx` cached ones."""
    g = torch.Generator().manual_seed(seed)
    pool = Pool(g, [max(0, x) for x in ctx], block)
    ints = lambda x: torch.tensor(x, dtype=torch.int32)
    c = dict(table=pool.table(range(len(ctx))), ctx=ints(ctx), q_len=ints(new), q_start=ints([sum(new[:i]) for i in range(len(new))]), scale=192 ** -0.5,
             max_q_len=max(new), max_ctx=max(ctx), total_ctx=sum(max(0, x) for x in ctx))
    x = torch.randn(pool.blocks * block, 1, 576, generator=g).bfloat16()
    x[pool.dead] = float("nan")
    c["cache"] = x.view(pool.blocks, block, 1, 576)
    c["q"] = (torch.randn(sum(new), heads, 192, generator=g) * spread).bfloat16()
    c["w"] = (torch.randn(heads, 256, 512, generator=g) * 512 ** -0.5).bfloat16()
    return c


def latent_exact(c):
    """(out, its bound) in 64 bits, keys and values not rounded."""
    T, H, _ = c["q"].shape
    out, tol = (torch.zeros(T, H, 128, dtype=torch.float64) for _ in range(2))
    w = c["w"].double()
    for s in range(len(c["ctx"])):
        n, ql, at = max(0, int(c["ctx"][s])), int(c["q_len"][s]), int(c["q_start"][s])
        x = _rows(c["cache"], c["table"][s], n)[:, 0]
        kv, kva = torch.einsum("nl,hdl->hnd", x[:, :512], w), torch.einsum("nl,hdl->hnd", x[:, :512].abs(), w.abs())
        # a key's or value's element: its 32-bit sum, then bf16
        off = 2.0 ** -8 * kv.abs() + 512 * 2.0 ** -23 * kva
        for h in range(H):
            q = c["q"][at:at + ql, h].double()
            k, v, dk, dv = kv[h, :, :128], kv[h, :, 128:], off[h, :, :128], off[h, :, 128:]
            z = (q[:, :128] @ k.T + q[:, 128:] @ x[:, 512:].T) * c["scale"]
            e = (q[:, :128].abs() @ dk.T + 192 * 2.0 ** -23 * (q[:, :128].abs() @ k.abs().T + q[:, 128:].abs() @ x[:, 512:].abs().T)) * c["scale"] + 2.0 ** -21
            seen = torch.arange(n) < (n - ql + 1 + torch.arange(ql))[:, None]
            p, _ = _softmax(z.masked_fill(~seen, -math.inf))
            pm = p.masked_fill(~seen, 0.0)
            o = pm @ v
            worst = torch.where(seen, e, 0.0).amax(-1, keepdim=True) if n else torch.zeros(ql, 1, dtype=torch.float64)
            a = pm @ v.abs()
            out[at:at + ql, h] = o
            # a weight is off by its score's error and the normaliser's, then rounded to bf16; values; the result
            tol[at:at + ql, h] = (2.0 ** -8 * o.abs() + (torch.expm1(2 * worst) + 2.0 ** -8 + n * 2.0 ** -24) * a + pm @ dv) * (1 + 2.0 ** -7)
    return out, tol
