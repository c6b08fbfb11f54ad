"""64-bit oracle of the operators that hold a cache to a budget by attention weight, and cases for them, shared by the CPU and the GPU tests."""
import math

import torch

LOG2E = 1.4426950408889634


def rows_of(cache, table, s, idx, scale=None):
    bs = cache.shape[1]
    x = cache.flatten(0, 1)[table[s].long()[idx // bs] * bs + idx % bs]
    return x.view(torch.float8_e4m3fn).double() * scale.double() if cache.dtype == torch.uint8 else x.double()


def case(seed, ctx, heads, kv_heads, dim, fp8, block=16, new=None, columns=None, spread=1.5):
    """A paged cache of sequences of lengths `ctx` behind a shuffled table; what lies behind a context in its last block, and block 0, is NaN."""
    g = torch.Generator().manual_seed(seed)
    S, per = len(ctx), max(1, max((n + block - 1) // block for n in ctx))
    used = [(n + block - 1) // block for n in ctx]
    nb = sum(used) + 1
    perm = (torch.randperm(nb - 1, generator=g) + 1).tolist() if nb > 1 else []
    table = torch.zeros(S, per, dtype=torch.int32)
    dead = torch.ones(nb * block, dtype=torch.bool)
    for s, n in enumerate(ctx):
        mine = [perm.pop() for _ in range(used[s])]
        table[s, :used[s]] = torch.tensor(mine, dtype=torch.int32)
        for j in range(n):
            dead[mine[j // block] * block + j % block] = False
    c = dict(table=table, ctx=torch.tensor(ctx, dtype=torch.int32), scale=dim ** -0.5, max_ctx=max(ctx), k_scale=None, v_scale=None)
    for name in ("k", "v"):
        x = torch.randn(nb * block, kv_heads, dim, generator=g)
        x = (x * 16).to(torch.float8_e4m3fn).view(torch.uint8) if fp8 else x.bfloat16()
        x[dead] = 0x7f if fp8 else float("nan")
        c[name] = x.view(nb, block, kv_heads, dim)
        if fp8:
            c[name + "_scale"] = torch.tensor([0.0625 if name == "k" else 0.05])
    new = [1] * S if new is None else new
    c["q"] = (torch.randn(sum(new), heads, dim, generator=g) * spread).bfloat16()
    c["q_len"], c["max_q_len"] = torch.tensor(new, dtype=torch.int32), max(new)
    c["q_start"] = torch.cat([torch.zeros(1, dtype=torch.int32), c["q_len"].cumsum(0).int()[:-1]])
    c["mass"] = torch.rand(S, kv_heads, max(1, columns or max(ctx)), generator=g) * 0.01
    return c


def weights(c, s, h, G, last):
    """Weights [W, G, n] of the observed rows in 64 bits, and the largest sum of |q k| of a logit, in the log2 domain."""
    n, ql = int(c["ctx"][s]), int(c["q_len"][s])
    w = min(last or ql, ql)
    k = rows_of(c["k"], c["table"], s, torch.arange(n, device=c["table"].device), c["k_scale"])[:, h]
    q0 = int(c["q_start"][s]) + ql
    q = c["q"][q0 - w:q0, h * G:(h + 1) * G].double()
    z = torch.einsum("wgd,nd->wgn", q, k) * c["scale"]
    limit = n - w + 1 + torch.arange(w, device=z.device)
    seen = (torch.arange(n, device=z.device) < limit[:, None])[:, None]
    top = z.masked_fill(~seen, -math.inf).amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top)), torch.zeros_like(z))
    total = e.sum(-1, keepdim=True)
    size = float(torch.einsum("wgd,nd->wgn", q.abs(), k.abs()).max()) * c["scale"] * LOG2E if w and n else 0.0
    return e / torch.where(total == 0, torch.ones_like(total), total), size


def weight_error(c, dim, size):
    """Relative error that a weight may have: a logit's 32-bit sum of `dim` exact products, each addition off by up to 2^-23 of the sum of their
    sizes (a matrix unit may cut instead of round), and the queries' f16 of the e4m3 kernels (elements under 2^-14 are off by up to
    2^-25), twice (its own and the normaliser's); an exponential is off by 2^-22."""
    k = 28.0 if c["k"].dtype == torch.uint8 else 0.0                      # the largest e4m3 value times the cases' scale
    z = dim * 2.0 ** -23 * size + dim * 2.0 ** -25 * k * c["scale"] * LOG2E
    return 2 * (math.log(2) * z + 2.0 ** -22)


def decode(c):
    """(out, its bound, mass, its bound) in 64 bits."""
    S, Hq, D = c["q"].shape
    H = c["k"].shape[2]
    G = Hq // H
    out, tol = torch.zeros(S, Hq, D, dtype=torch.float64), torch.zeros(S, Hq, D, dtype=torch.float64)
    mass, mtol = c["mass"].double().clone(), torch.zeros(c["mass"].shape, dtype=torch.float64)
    for s in range(S):
        n = int(c["ctx"][s])
        if n <= 0:
            continue
        v = rows_of(c["v"], c["table"], s, torch.arange(n), c["v_scale"])
        for h in range(H):
            p, size = weights(c, s, h, G, 1)
            r = weight_error(c, D, size)
            o, a = torch.einsum("gn,nd->gd", p[0], v[:, h]), torch.einsum("gn,nd->gd", p[0], v[:, h].abs())
            out[s, h * G:(h + 1) * G] = o
            # weights rounded to bf16 (f16 for an e4m3 cache: finer, but what is under 2^-24 of the largest is lost), then the result
            tol[s, h * G:(h + 1) * G] = 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2 * r) * a + n * 2.0 ** -24 * v[:, h].abs().max()
            add = p[0].sum(0)
            mass[s, h, :n] += add
            mtol[s, h, :n] = (r + G * 2.0 ** -24) * add + 2.0 ** -23 * mass[s, h, :n] + 1e-30
    return out, tol, mass, mtol


def prompt(c, last):
    """(mass, its bound) in 64 bits."""
    Hq, D = c["q"].shape[1:]
    H = c["k"].shape[2]
    G = Hq // H
    mass, mtol = c["mass"].double().clone(), torch.zeros(c["mass"].shape, dtype=torch.float64)
    for s in range(len(c["ctx"])):
        n, ql = int(c["ctx"][s]), int(c["q_len"][s])
        w = min(last or ql, ql)
        if n <= 0 or w <= 0:
            continue
        for h in range(H):
            p, size = weights(c, s, h, G, last)
            add = p.sum((0, 1))
            r = weight_error(c, D, size)
            mass[s, h, :n] += add
            mtol[s, h, :n] = (r + w * G * 2.0 ** -24) * add + 2.0 ** -23 * mass[s, h, :n] + 1e-30
    return mass, mtol


def evict(c, keep, recent, max_ctx, dst=None):
    """(k, v, mass, kept, lengths): what the operator has to give, exactly."""
    S, H = c["mass"].shape[:2]
    bs = c["k"].shape[1]
    k, v = c["k"].clone(), c["v"].clone()
    mass = c["mass"].clone()
    kept = torch.full((S, H, keep), -1, dtype=torch.int32)
    to_table = c["table"] if dst is None else dst
    for s in range(S):
        n = int(c["ctx"][s])
        m = min(n, keep)
        for h in range(H):
            x = [float(t) for t in c["mass"][s, h, :n]]
            x = [-math.inf if t != t else t for t in x]
            old = max(0, n - recent)
            best = sorted(range(old), key=lambda j: (-x[j], j))[:max(0, m - recent)] if n > keep else list(range(old))
            idx = sorted(best) + list(range(old, n))
            assert len(idx) == m
            kept[s, h, :m] = torch.tensor(idx, dtype=torch.int32)
            mass[s, h, :max_ctx] = 0
            for i, j in enumerate(idx):
                a = int(c["table"][s, j // bs]) * bs + j % bs
                b = int(to_table[s, i // bs]) * bs + i % bs
                for new, old_cache in ((k, c["k"]), (v, c["v"])):
                    new.flatten(0, 1)[b, h] = old_cache.flatten(0, 1)[a, h]
                mass[s, h, i] = c["mass"][s, h, j]
    return k, v, mass, kept, torch.tensor([min(int(n), keep) for n in c["ctx"]], dtype=torch.int32)
