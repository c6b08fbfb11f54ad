"""Attention over what requests have in common, as cases to be timed: a decode or verify step of a batch whose sequences share long
prefixes, which are read once for all of them; the joining of attention that was computed in parts; prompts over a latent cache whose
keys and values are expanded per head.

``run`` computes each in its plain form; where ``own`` is true it calls ``ops.shared_prefix_attention``, ``ops.merge_attention`` and
``ops.mla_prompt_attention``. Caches are [blocks, block, kv heads, dim], bf16 or e4m3 bytes with a scale, or [blocks, block, 1, 576]
bf16 latent rows, behind shuffled block tables.
"""
from __future__ import annotations

import math

import torch

own = False

LATENT, ROPE, NOPE, VALUE = 512, 64, 128, 128              # a latent row's two parts, a head's key without and its value


# ----------------------------------------------------------------------------- cases
def _shared(name, seqs, groups, prefix, prefix_min, ctx, ctx_min, heads, kv_heads, dim, cache, block=16, n=1, alone=0):
    """`seqs` sequences of `ctx_min` to `ctx` tokens of their own, `n` of them new, in `groups` groups behind prefixes of `prefix_min` to
    `prefix` tokens; the last `alone` of them in no group."""
    d = dict(kind="shared", seqs=seqs, groups=groups, prefix=prefix, prefix_min=prefix_min, ctx=ctx, ctx_min=ctx_min, heads=heads, kv_heads=kv_heads, dim=dim,
             cache=cache, block=block, n=n, alone=alone)
    return dict(name=name, **d) if name else d


def _merge(name, parts, rows, heads, dim, type):
    d = dict(kind="merge", parts=parts, rows=rows, heads=heads, dim=dim, type=type)
    return dict(name=name, **d) if name else d


def _latent(name, seqs, new, new_min, ctx, ctx_min, heads, block=16):
    d = dict(kind="latent", seqs=seqs, new=new, new_min=new_min, ctx=ctx, ctx_min=ctx_min, heads=heads, block=block)
    return dict(name=name, **d) if name else d


def listed():
    return [
        # a few chats behind one system prompt: the latency of a token
        _shared("shared 8 behind 700 e4m3", 8, 1, 700, 700, 90, 1, 40, 8, 128, "e4m3"),
        # small heads, short prompts, blocks that are no power of two, a sequence without a prefix
        _shared("shared 5 behind 333 d64", 5, 2, 333, 61, 70, 1, 4, 2, 64, "bf16", block=24, alone=1),
        # the headline benchmark's rung of 128 requests, behind a system prompt with its tools
        _shared("shared 128 behind 8192 e4m3", 128, 1, 8192, 8192, 1151, 129, 40, 8, 128, "e4m3"),
        # questions about a few long documents
        _shared("shared 61 behind 5 of 16000 bf16", 61, 5, 16000, 4001, 300, 10, 32, 8, 128, "bf16"),
        # a medium batch of the hybrid's wide heads, two prompts, some requests with none
        _shared("shared 33 behind 2 of 2047 d256", 33, 2, 2047, 1500, 500, 40, 16, 2, 256, "bf16", alone=4),
        # speculation behind a shared prompt: three drafts a sequence checked in one pass
        _shared("shared 16x4 behind 5000 e4m3", 16, 1, 5000, 5000, 700, 50, 40, 8, 128, "e4m3", n=4),
        # a step's rows, attended in two parts
        _merge("merge 2 x 128", 2, 128, 40, 128, "bf16"),
        # a prompt's rows, attended in five parts that were kept in 32 bits
        _merge("merge 5 x 8191 fp32", 5, 8191, 32, 128, "fp32"),
        # a chat turn's prompt on one of eight ranks
        _latent("latent prompt 333", 1, 333, 333, 333, 333, 16),
        # a few prompts, some behind what is cached of them
        _latent("latent prompts 3x1300", 3, 1300, 500, 1700, 900, 16),
        # a document of the whole prefill budget
        _latent("latent prompt 8192", 1, 8192, 8192, 8192, 8192, 16),
        # a portion of a long prompt, all heads on one GPU
        _latent("latent portion 4096 at 8192", 1, 4096, 4096, 8192, 8192, 128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("shared", "shared", "shared", "merge", "latent", "latent"))
    if kind == "shared":
        heads, kv_heads, dim = rng.choice(((40, 8, 128), (40, 8, 128), (32, 8, 128), (16, 2, 256), (16, 1, 128), (12, 12, 128), (4, 2, 64), (24, 2, 128)))
        n = rng.choice((1, 1, 1, 2, 4, 5))
        seqs = _log(rng, 1, 160 // n)
        groups = min(seqs, rng.choice((1, 1, 2, 3, 7)))
        width = kv_heads * max(1, dim // 128)
        prefix = _log(rng, 16, min(32768, 640_000 // (groups * width), 128 * 8192 * 40 * 128 // (seqs * n * heads * dim)))
        ctx = max(n, _log(rng, 1, min(2048, 1_300_000 // (seqs * width))))
        return _shared(None, seqs, groups, prefix, rng.randint(max(1, prefix // 4), prefix), ctx, rng.randint(n, ctx), heads, kv_heads, dim, rng.choice(("e4m3", "bf16")),
                       rng.choice((16, 16, 16, 32, 64, 24)), n, rng.choice((0, 0, min(3, seqs - 1))))
    if kind == "merge":
        heads, dim = rng.choice(((40, 128), (32, 128), (16, 256), (4, 64), (16, 512), (12, 128)))
        parts = rng.randint(2, 8)
        return _merge(None, parts, _log(rng, 1, min(8191, 5 * 8191 * 32 * 128 // (parts * heads * dim))), heads, dim, rng.choice(("bf16", "fp32")))
    heads = rng.choice((16, 16, 16, 32, 128))
    ctx = _log(rng, 24, 8192)
    new = _log(rng, 16, min(ctx, 4096 * 128 // heads))
    seqs = _log(rng, 1, max(1, min(12, 4096 * 8192 * 128 // (2 * ctx * new * heads), 24576 * 16 // (ctx * heads))))
    return _latent(None, seqs, new, rng.randint(max(1, new // 3), new), ctx, rng.randint(new, ctx), heads, rng.choice((16, 16, 32, 64, 24)))


def _spread(lo, hi, n, step, at):
    """n lengths from lo to hi, the same for every seed, hi the first of them."""
    return [hi if i == 0 else round(lo + ((i * step + at) % n) / max(1, n - 1) * (hi - lo)) for i in range(n)]


def _lengths(c):
    """(cached rows of every sequence, new ones of them, rows of every prefix, the groups' first sequences)."""
    ctx = _spread(c["ctx_min"], c["ctx"], c["seqs"], 37, 11)
    if c["kind"] == "latent":
        return ctx, [min(a, b) for a, b in zip(_spread(c["new_min"], c["new"], c["seqs"], 53, 5), ctx)], None, None
    n = c["groups"]
    shared = max(n, c["seqs"] - c["alone"])
    # groups of unequal size, one sequence at least in each
    start = [0] + [max(i, round(shared * (i / n) ** 1.5)) for i in range(1, n)] + [shared]
    return ctx, [c["n"]] * c["seqs"], _spread(c["prefix_min"], c["prefix"], n, 3, 1), start


# ----------------------------------------------------------------------------- inputs
def _tables(rows, block, perm):
    """Block tables of sequences of these lengths that take their blocks from the front of `perm`, and the blocks that are left."""
    used = [(n + block - 1) // block for n in rows]
    at = torch.tensor([0] + used[:-1]).cumsum(0).to("cuda")
    col = torch.arange(max(max(used), 1), device="cuda")
    table = torch.where(col < torch.tensor(used, device="cuda")[:, None], perm[(at[:, None] + col).clamp(max=perm.numel() - 1)], 0).to(torch.int32)
    return table, perm[sum(used):]


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if c["kind"] == "merge":
        dt = torch.bfloat16 if c["type"] == "bf16" else torch.float32
        outs = [randn(c["rows"], c["heads"], c["dim"]).to(dt) for _ in range(c["parts"])]
        lses = [randn(c["rows"], c["heads"]) * 2 + 6 for _ in range(c["parts"])]
        # here and there a part in which a row saw nothing
        for o, l in zip(outs[1:], lses[1:]):
            none = torch.rand(c["rows"], c["heads"], generator=g, device="cuda") < 0.03
            l[none], o[none] = -math.inf, 0.0
        return dict(case=c, outs=outs, lses=lses)
    ctx, new, prefix, start = _lengths(c)
    bs = c["block"]
    nb = 1 + sum((n + bs - 1) // bs for n in ctx + (prefix or []))         # block 0 belongs to nobody
    perm = torch.randperm(nb - 1, generator=g, device="cuda") + 1
    s = dict(case=c, ctx=_ints(ctx), max_ctx=max(ctx))
    s["table"], perm = _tables(ctx, bs, perm) if perm.numel() else (_ints([[0]]), perm)
    if c["kind"] == "latent":
        s["cache"] = randn(nb, bs, 1, LATENT + ROPE).bfloat16()
        s["q"] = (randn(sum(new), c["heads"], NOPE + ROPE) * 1.5).bfloat16()
        s["w"] = (randn(c["heads"], NOPE + VALUE, LATENT) * LATENT ** -0.5).bfloat16()
        s["q_start"], s["q_len"] = _ints([sum(new[:i]) for i in range(len(new))]), _ints(new)
        s.update(max_q_len=max(new), total_ctx=sum(ctx), scale=(NOPE + ROPE) ** -0.5)
        return s
    s["prefix_table"], _ = _tables(prefix, bs, perm)
    H, D = c["kv_heads"], c["dim"]
    s["k_scale"] = s["v_scale"] = None
    for name in ("k", "v"):
        x = randn(nb * bs, H, D)
        s[name] = ((x * 16).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) if c["cache"] == "e4m3" else x.bfloat16()).view(nb, bs, H, D)
    if c["cache"] == "e4m3":
        s["k_scale"], s["v_scale"] = torch.full((1,), 0.0625, device="cuda"), torch.full((1,), 0.0625, device="cuda")
    s["q"] = (randn(c["seqs"] * c["n"], c["heads"], D) * 1.5).bfloat16()
    s.update(prefix=_ints(prefix), start=_ints(start), first=start, max_prefix=max(prefix), scale=D ** -0.5)
    return s


# ----------------------------------------------------------------------------- plain forms
def _rows(s, name, table, cols):
    """Cached rows of sequences, 32 bits: [sequences, cols, ...]."""
    bs = s["case"]["block"]
    j = torch.arange(cols, device="cuda")
    x = s[name].flatten(0, 1)[table[:, j // bs].long() * bs + j % bs]
    return x.view(torch.float8_e4m3fn).float() * s[name + "_scale"] if x.dtype == torch.uint8 else x.float()


def _joined(zs, vs):
    """Softmax over all of `zs` (keys last), and its sums over `vs`; a row that sees nothing gives zeros."""
    top = torch.stack([z.amax(-1) for z in zs]).amax(0)
    base = torch.where(top == -math.inf, 0.0, top)[..., None]
    es = [torch.exp(z - base) for z in zs]
    total = sum(e.sum(-1) for e in es)
    out = sum(e @ v for e, v in zip(es, vs))
    return out / torch.where(total == 0, 1.0, total)[..., None], torch.where(total == 0, -math.inf, base[..., 0] + torch.log(total))


def _plain_shared(s):
    c, n = s["case"], s["case"]["n"]
    S, H, D, Hq = c["seqs"], c["kv_heads"], c["dim"], c["heads"]
    G = Hq // H
    q = s["q"].float().view(S, n, H, G, D).permute(0, 2, 1, 3, 4).reshape(S, H, n * G, D) * s["scale"]
    out, lse = torch.empty(S, H, n * G, D, device="cuda"), torch.empty(S, H, n * G, device="cuda")
    j, step = torch.arange(s["max_ctx"], device="cuda"), torch.arange(n, device="cuda")
    back = (s["ctx"][:, None] - n + 1 + step)                                  # rows of its own that a token sees
    seen = (j < back[:, :, None])[:, None, :, None].expand(-1, -1, -1, G, -1).reshape(S, 1, n * G, -1)
    bounds = [(a, b, i) for i, (a, b) in enumerate(zip(s["first"], s["first"][1:]))] + [(s["first"][-1], S, None)]
    for a, b, i in bounds:
        if a == b:
            continue
        k, v = (torch.where((j < s["ctx"][a:b, None])[:, :, None, None], _rows(s, x, s["table"][a:b], s["max_ctx"]), 0.0).transpose(1, 2) for x in ("k", "v"))
        zs, vs = [(q[a:b] @ k.transpose(2, 3)).masked_fill_(~seen[a:b], -math.inf)], [v]
        if i is not None:
            p = s["max_prefix"]
            live = torch.arange(p, device="cuda") < s["prefix"][i]
            k, v = (torch.where(live[:, None, None], _rows(s, x, s["prefix_table"][i:i + 1], p)[0], 0.0).transpose(0, 1) for x in ("k", "v"))
            zs.append((q[a:b] @ k.transpose(1, 2)).masked_fill_(~live, -math.inf))
            vs.append(v)
        out[a:b], lse[a:b] = _joined(zs, vs)
    turn = lambda x: x.view(S, H, n, G, *x.shape[3:]).transpose(1, 2).reshape(S * n, Hq, *x.shape[3:])
    return turn(out).bfloat16(), turn(lse)


def _plain_merge(s):
    l = torch.stack(s["lses"])
    top = l.amax(0)
    w = torch.exp(l - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(0)
    out = sum(a[..., None] * o.float() for a, o in zip(w, s["outs"])) / torch.where(total == 0, 1.0, total)[..., None]
    return out.to(s["outs"][0].dtype), torch.where(total == 0, -math.inf, top + torch.log(total))


def _plain_latent(s):
    c = s["case"]
    H = c["heads"]
    ctx, new, _, _ = _lengths(c)
    out = torch.empty(s["q"].shape[0], H, VALUE, dtype=torch.bfloat16, device="cuda")
    w, at = s["w"].float(), 0
    for i, (n, b) in enumerate(zip(ctx, new)):
        x = _rows(s, "cache", s["table"][i:i + 1], n)[0, :, 0]
        seen = torch.arange(n, device="cuda") < (n - b + 1 + torch.arange(b, device="cuda"))[:, None]
        for h in range(H):
            kv = x[:, :LATENT] @ w[h].T
            q = s["q"][at:at + b, h].float() * s["scale"]
            z = (q[:, :NOPE] @ kv[:, :NOPE].T).addmm_(q[:, NOPE:], x[:, LATENT:].T).masked_fill_(~seen, -math.inf)
            z = torch.exp(z.sub_(z.amax(-1, keepdim=True)))
            out[at:at + b, h] = ((z @ kv[:, NOPE:]) / z.sum(-1, keepdim=True)).bfloat16()
        at += b
    return out


# ----------------------------------------------------------------------------- one pass
def _call(s):
    from metrale_inference_alpha_b200 import ops
    c = s["case"]
    if c["kind"] == "merge":
        return ops.merge_attention(s["outs"], s["lses"])
    if c["kind"] == "latent":
        return ops.mla_prompt_attention(s["q"], s["cache"], s["table"], s["q_start"], s["q_len"], s["ctx"], s["w"], max_q_len=s["max_q_len"], max_ctx=s["max_ctx"],
                                        total_ctx=s["total_ctx"], scale=s["scale"])
    return ops.shared_prefix_attention(s["q"], s["k"], s["v"], s["prefix_table"], s["prefix"], s["start"], s["table"], s["ctx"], max_prefix=s["max_prefix"],
                                       max_ctx=s["max_ctx"], scale=s["scale"], q_len=c["n"], k_scale=s["k_scale"], v_scale=s["v_scale"], return_lse=True)


def run(state):
    if own:
        return _call(state)
    return {"shared": _plain_shared, "merge": _plain_merge, "latent": _plain_latent}[state["case"]["kind"]](state)


def work(case):
    c = case
    if c["kind"] == "merge":
        n = c["rows"] * c["heads"]
        return {"bytes": n * (c["parts"] + 1) * (c["dim"] * (2 if c["type"] == "bf16" else 4) + 4), "flops": 2 * n * c["parts"] * c["dim"]}
    ctx, new, prefix, start = _lengths(c)
    bs = c["block"]
    tables = 4 * sum((n + bs - 1) // bs for n in ctx + (prefix or []))
    if c["kind"] == "latent":
        H = c["heads"]
        pairs = sum(b * n - b * (b - 1) // 2 for n, b in zip(ctx, new))
        expand = 2 * sum(ctx) * LATENT * (NOPE + VALUE)
        return {"bytes": 2 * sum(ctx) * (LATENT + ROPE) + 2 * H * (NOPE + VALUE) * LATENT + 2 * sum(new) * H * (NOPE + ROPE + VALUE) + tables,
                "flops": H * (2 * pairs * (NOPE + ROPE + VALUE) + expand)}
    H, D, e, n = c["kv_heads"], c["dim"], 1 if c["cache"] == "e4m3" else 2, c["n"]
    pairs = sum(n * x - n * (n - 1) // 2 for x in ctx) + n * sum((b - a) * p for a, b, p in zip(start, start[1:], prefix))
    return {"bytes": 2 * (sum(ctx) + sum(prefix)) * H * D * e + c["seqs"] * n * c["heads"] * (4 * D + 4) + tables, "flops": 4 * c["heads"] * D * pairs}


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "merge":
        l = torch.stack(s["lses"]).double()
        lse = torch.logsumexp(l, 0)
        w = torch.where(l == -math.inf, 0.0, torch.exp(l - lse))
        return torch.einsum("prh,prhd->rhd", w, torch.stack(s["outs"]).double()), lse
    ctx, new, prefix, start = _lengths(c)
    bs = c["block"]

    def rows(name, table, n):
        j = torch.arange(n, device="cuda")
        x = s[name].flatten(0, 1)[table.long()[j // bs] * bs + j % bs]
        return x.view(torch.float8_e4m3fn).double() * s[name + "_scale"].double() if x.dtype == torch.uint8 else x.double()

    if c["kind"] == "latent":
        out = torch.empty(s["q"].shape[0], c["heads"], VALUE, dtype=torch.float64, device="cuda")
        for i, (n, b) in enumerate(zip(ctx, new)):
            x, at = rows("cache", s["table"][i], n)[:, 0], sum(new[:i])
            for h in range(c["heads"]):
                w = s["w"][h].double()
                k = torch.cat([x[:, :LATENT] @ w[:NOPE].T, x[:, LATENT:]], 1)
                v = x[:, :LATENT] @ w[NOPE:].T
                for t in range(0, b, 2048):
                    q = s["q"][at + t:at + min(b, t + 2048), h].double()
                    z = q @ k.T * s["scale"]
                    limit = n - b + 1 + torch.arange(t, t + q.shape[0], device="cuda")
                    z.masked_fill_(torch.arange(n, device="cuda") >= limit[:, None], -math.inf)
                    out[at + t:at + t + q.shape[0], h] = torch.softmax(z, -1) @ v
        return out
    S, n, H, Hq, D = c["seqs"], c["n"], c["kv_heads"], c["heads"], c["dim"]
    out = torch.zeros(S * n, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.empty(S * n, Hq, dtype=torch.float64, device="cuda")
    behind, last = {}, None
    for g, (a, b) in enumerate(zip(start, start[1:])):
        behind.update({i: g for i in range(a, b)})
    for i in range(S):
        k, v = rows("k", s["table"][i], ctx[i]), rows("v", s["table"][i], ctx[i])
        p = 0
        if i in behind:
            if behind[i] != last:
                last = behind[i]
                common = [rows(x, s["prefix_table"][last], prefix[last]) for x in ("k", "v")]
            k, v, p = torch.cat([common[0], k]), torch.cat([common[1], v]), prefix[last]
        for t in range(n):
            m = p + ctx[i] - n + 1 + t
            z = torch.einsum("hgd,mhd->hgm", s["q"][i * n + t].double().view(H, -1, D), k[:m]) * s["scale"]
            lse[i * n + t] = torch.logsumexp(z, -1).view(-1)
            out[i * n + t] = torch.einsum("hgm,mhd->hgd", torch.softmax(z, -1), v[:m]).reshape(Hq, D)
    return out, lse
