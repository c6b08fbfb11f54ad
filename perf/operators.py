"""A paged key-value cache that is held to a budget of tokens by the attention weight that they have gathered, as cases to be
timed: decode attention that adds its weights up per cached token, the weights that a prompt's last tokens give what is cached,
and the eviction of what has gathered least.

``run`` computes each in its plain form; where ``own`` is true it calls ``ops.paged_attention_mass``, ``ops.prompt_mass`` and
``ops.kv_evict``. Caches are [blocks, block, kv heads, dim], bf16 or e4m3 bytes with a scale, behind a shuffled block table; the
gathered weight is fp32 [sequences, kv heads, columns], column j for a sequence's cached row j.
"""
from __future__ import annotations

import math

import torch

own = False



# ----------------------------------------------------------------------------- cases
def _case(name, kind, seqs, ctx, ctx_min, heads, kv_heads, dim, cache, block=16, **more):
    d = dict(kind=kind, seqs=seqs, ctx=ctx, ctx_min=ctx_min, heads=heads, kv_heads=kv_heads, dim=dim, cache=cache, block=block, **more)
    return dict(name=name, **d) if name else d


def listed():
    return [
        # a token of one user mid-generation: latency
        _case("decode 1x700 e4m3", "decode", 1, 700, 700, 40, 8, 128, "e4m3"),
        # small heads, a handful of short sequences, one of a single token
        _case("decode 5x1-333 d64", "decode", 5, 333, 1, 4, 2, 64, "bf16"),
        # the headline benchmark's rung: 128 requests between their first and their last token
        _case("decode 128x129-1151 e4m3", "decode", 128, 1151, 129, 40, 8, 128, "e4m3"),
        # a medium batch of the hybrid's wide heads
        _case("decode 33x100-2047 d256", "decode", 33, 2047, 100, 16, 2, 256, "bf16"),
        # long documents under discussion, before their caches are cut
        _case("decode 16x32749 bf16", "decode", 16, 32749, 8001, 32, 8, 128, "bf16"),
        # a prompt of the whole prefill budget, its last 32 tokens as observers
        _case("observe 32 of 8192 e4m3", "observe", 1, 8192, 8192, 40, 8, 128, "e4m3", new=8192, new_min=8192, last=32),
        # a batch of chat turns, each prompt's last 64 tokens, shorter prompts whole
        _case("observe 64 of 16x17-1151", "observe", 16, 1151, 17, 32, 8, 128, "bf16", new=1151, new_min=17, last=64),
        # every token of a portion of a prompt, wide heads, behind what is cached of it
        _case("observe 1531 at 4431 d256", "observe", 2, 4431, 3501, 16, 2, 256, "bf16", new=1531, new_min=1001, last=0),
        # every token of a long portion
        _case("observe 4096 at 8192 e4m3", "observe", 1, 8192, 8192, 40, 8, 128, "e4m3", new=4096, new_min=4096, last=0),
        # decode went 256 tokens past its budget: cut in place
        _case("evict 1x4352 to 4096", "evict", 1, 4352, 4352, 40, 8, 128, "e4m3", keep=4096, recent=64, place="same"),
        # a few short sequences of small heads, one within its budget
        _case("evict 3x70-500 to 128 d64", "evict", 3, 500, 70, 4, 2, 64, "bf16", keep=128, recent=16, place="same"),
        # long documents behind a shared prefix, cut into blocks of their own
        _case("evict 8x32749 to 4000", "evict", 8, 32749, 9001, 32, 8, 128, "bf16", keep=4000, recent=128, place="own"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("decode", "decode", "observe", "observe", "evict"))
    heads, kv_heads, dim = rng.choice(((40, 8, 128), (40, 8, 128), (32, 8, 128), (16, 2, 256), (16, 1, 128), (12, 12, 128), (4, 2, 64), (24, 2, 128)))
    cache, block = rng.choice(("e4m3", "bf16")), rng.choice((16, 16, 16, 32, 64, 24))
    most = 4_000_000 // (kv_heads * max(1, dim // 128))       # cached rows in all, the longest sequence's length for each
    if kind == "decode":
        seqs = _log(rng, 1, 160)
        ctx = _log(rng, 1, min(65536, most // seqs))
        return _case(None, kind, seqs, ctx, rng.randint(max(1, ctx // 4), ctx), heads, kv_heads, dim, cache, block)
    if kind == "observe":
        seqs = _log(rng, 1, 24)
        ctx = _log(rng, 2, min(16384, most // seqs))
        new = _log(rng, 1, ctx)
        least, ctx_min = rng.randint(max(1, new // 3), new), rng.randint(max(new, ctx // 2), ctx)
        last = rng.choice((0, 16, 32, 64, 257))
        cost = seqs * heads * ctx * dim                       # logits of one observing token, by their size
        if cost * (min(last, new) if last else new) > 8192 * 2800 * 40 * 128:
            last = max(1, 8192 * 2800 * 40 * 128 // cost)
        return _case(None, kind, seqs, ctx, ctx_min, heads, kv_heads, dim, cache, block, new=new, new_min=least, last=last)
    seqs = _log(rng, 1, 32)
    ctx = _log(rng, 32, min(32749, most // seqs // 4))
    keep = _log(rng, 8, max(16, ctx - 1))
    return _case(None, kind, seqs, ctx, rng.randint(max(1, ctx // 4), ctx), heads, kv_heads, dim, cache, block, keep=keep, recent=rng.choice((0, 1, keep // 4, keep)),
                 place=rng.choice(("same", "own")))


def _spread(lo, hi, n, step, at):
    """n lengths from lo to hi, the same for every seed, hi the first of them."""
    return [hi if i == 0 else round(lo + ((i * step + at) % n) / max(1, n - 1) * (hi - lo)) for i in range(n)]


def _lengths(c):
    """(cached, new) rows of every sequence."""
    ctx = _spread(c["ctx_min"], c["ctx"], c["seqs"], 37, 11)
    if c["kind"] != "observe":
        return ctx, [1] * c["seqs"]
    return ctx, [min(a, b) for a, b in zip(_spread(c["new_min"], c["new"], c["seqs"], 53, 5), ctx)]


# ----------------------------------------------------------------------------- inputs
def _cache(c, rows, gen, tilt):
    x = torch.randn(rows, c["kv_heads"], c["dim"], generator=gen, device="cuda")
    if tilt is not None:
        x += tilt
    if c["cache"] == "e4m3":
        return (x * 16).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return x.bfloat16()


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    S, bs, H, D, dev = c["seqs"], c["block"], c["kv_heads"], c["dim"], "cuda"
    ctx, new = _lengths(c)
    most = max(ctx)
    per = (most + bs - 1) // bs
    used = [(n + bs - 1) // bs for n in ctx]
    nb = sum(used) + 1                                        # block 0 belongs to nobody
    at = torch.tensor([0] + used[:-1]).cumsum(0).to(dev)
    perm = torch.randperm(nb - 1, generator=g, device=dev) + 1
    col = torch.arange(per, device=dev)
    table = torch.where(col < torch.tensor(used, device=dev)[:, None], perm[(at[:, None] + col).clamp(max=nb - 2)], 0).to(torch.int32)
    s = dict(case=c, table=table, ctx=torch.tensor(ctx, dtype=torch.int32, device=dev), max_ctx=most, scale=D ** -0.5, k_scale=None, v_scale=None)
    # some tokens draw the queries of a head: a direction that queries share and keys have more or less of
    way = torch.nn.functional.normalize(torch.randn(H, D, generator=g, device=dev), dim=-1)
    pull = torch.empty(nb * bs, H, 1, device=dev).exponential_(1.0, generator=g)
    s["k"] = _cache(c, nb * bs, g, way * pull if c["kind"] != "evict" else None).view(nb, bs, H, D)
    if c["kind"] != "observe":
        s["v"] = _cache(c, nb * bs, g, None).view(nb, bs, H, D)
    if c["cache"] == "e4m3":
        s["k_scale"], s["v_scale"] = torch.full((1,), 0.0625, device=dev), torch.full((1,), 0.0625, device=dev)
    live = torch.arange(most, device=dev) < s["ctx"][:, None, None]
    s["mass"] = torch.where(live, torch.randn(S, H, most, generator=g, device=dev).mul_(2).exp_(), 0.0)
    if c["kind"] != "evict":
        s["mass"] /= most                                     # what a few tokens before this one gave
    if c["kind"] == "evict":
        # tokens that nothing has looked at yet
        s["mass"] *= torch.rand(S, H, most, generator=g, device=dev) > 0.05
        s["mass_out"] = torch.empty_like(s["mass"])
        s["dst"] = None
        if c["place"] == "own":
            kb = (c["keep"] + bs - 1) // bs
            mine = torch.randperm(S * kb, generator=g, device=dev).view(S, kb) + nb
            s["dst"] = mine.to(torch.int32)
            for name in ("k", "v"):
                s[name] = torch.cat([s[name], torch.zeros(S * kb, bs, H, D, dtype=s[name].dtype, device=dev)])
        return s
    T = sum(new)
    q = torch.randn(T, c["heads"], D, generator=g, device=dev) * 1.5
    s["q"] = (q.view(T, H, -1, D) + way[:, None] * math.sqrt(D)).view(T, c["heads"], D).bfloat16()
    if c["kind"] == "observe":
        start = torch.tensor([0] + new[:-1]).cumsum(0)
        s["q_start"], s["q_len"] = start.to(torch.int32).to(dev), torch.tensor(new, dtype=torch.int32, device=dev)
        s["max_q_len"] = max(new)
    return s


# ----------------------------------------------------------------------------- plain forms
def _values(s, cache, scale, slots):
    """Cached rows at flat slots, 32 bits."""
    nb, bs, H, D = cache.shape
    x = cache.view(nb * bs, H, D)[slots]
    return x.view(torch.float8_e4m3fn).float() * scale if cache.dtype == torch.uint8 else x.float()


def _slots(s, bs, table, cols):
    j = torch.arange(cols, device="cuda")
    return table[:, j // bs].long() * bs + j % bs


def _softmax(z, seen):
    z = z.masked_fill(~seen, -math.inf)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _decode(s):
    c, n = s["case"], s["max_ctx"]
    S, H, D = c["seqs"], c["kv_heads"], c["dim"]
    slots = _slots(s, c["block"], s["table"], n)
    seen = torch.arange(n, device="cuda") < s["ctx"][:, None]
    k = _values(s, s["k"], s["k_scale"], slots)
    z = s["q"].float().view(S, H, -1, D) @ k.permute(0, 2, 3, 1) * s["scale"]
    p = _softmax(z, seen[:, None, None])
    v = torch.where(seen[:, :, None, None], _values(s, s["v"], s["v_scale"], slots), 0.0)
    out = p @ v.permute(0, 2, 1, 3)
    s["mass"] += p.sum(2)
    return out.reshape(S, c["heads"], D).bfloat16(), s["mass"]


def _observe(s):
    c, n = s["case"], s["max_ctx"]
    S, H, D = c["seqs"], c["kv_heads"], c["dim"]
    G = c["heads"] // H
    W = min(c["last"] or s["max_q_len"], s["max_q_len"])
    back = torch.arange(W - 1, -1, -1, device="cuda")                     # tokens before the last one
    live = back < s["q_len"][:, None]
    rows = (s["q_start"] + s["q_len"])[:, None] - 1 - back
    q = s["q"][rows.clamp(min=0)].float().view(S, W, H, G, D).permute(0, 2, 3, 1, 4).reshape(S, H, G * W, D)
    seen = (torch.arange(n, device="cuda") < (s["ctx"][:, None] - back)[:, :, None]) & live[:, :, None]
    k = _values(s, s["k"], s["k_scale"], _slots(s, c["block"], s["table"], n))
    z = q @ k.permute(0, 2, 3, 1) * s["scale"]
    p = _softmax(z.view(S, H, G, W, n), seen[:, None, None])
    s["mass"] += p.sum((2, 3))
    return s["mass"]


def _evict(s):
    c, n = s["case"], s["max_ctx"]
    j, ctx = torch.arange(n, device="cuda"), s["ctx"].long()[:, None, None]
    x = torch.where(torch.isnan(s["mass"]), -math.inf, s["mass"])
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    kind = torch.where(j >= ctx, 2, torch.where(j >= ctx - c["recent"], 0, 1)).expand_as(x)
    order = order.gather(-1, torch.sort(kind.gather(-1, order), dim=-1, stable=True).indices)
    rank = torch.empty_like(order).scatter_(-1, order, j.expand_as(order))
    count = ctx.clamp(max=c["keep"])
    held = rank < count
    to = held.cumsum(-1) - 1
    spare = max(n, c["keep"])                                             # column that nothing is read from
    kept = torch.full((*x.shape[:2], spare + 1), -1, dtype=torch.int64, device="cuda")
    kept.scatter_(-1, torch.where(held, to, spare), j.expand_as(to))
    kept = kept[:, :, :c["keep"]]
    live = kept >= 0
    width = min(n, c["keep"])
    s["mass_out"].zero_()
    s["mass_out"][:, :, :width] = torch.where(live, s["mass"].gather(-1, kept.clamp(min=0)), 0.0)[:, :, :width]
    # columns behind a sequence's kept rows write its last one again
    last = (count - 1).expand(-1, x.shape[1], 1)
    place = torch.minimum(torch.arange(c["keep"], device="cuda").expand_as(kept), last)
    source = kept.gather(-1, place)
    bs, seq = c["block"], torch.arange(c["seqs"], device="cuda")[:, None, None]
    head = torch.arange(c["kv_heads"], device="cuda")[None, :, None]
    dst = s["table"] if s["dst"] is None else s["dst"]
    out = []
    for name in ("k", "v"):
        flat = s[name].view(-1, c["kv_heads"], c["dim"])
        flat[dst[seq, place // bs].long() * bs + place % bs, head] = flat[s["table"][seq, source // bs].long() * bs + source % bs, head]
        out.append(s[name].view(torch.float8_e4m3fn) if s[name].dtype == torch.uint8 else s[name])
    return (*out, s["mass_out"], kept.int(), count.view(-1).int())


# ----------------------------------------------------------------------------- one pass
def _call(s):
    from metrale_inference_alpha_b200 import ops
    c = s["case"]
    if c["kind"] == "decode":
        return ops.paged_attention_mass(s["q"], s["k"], s["v"], s["table"], s["ctx"], s["mass"], max_ctx=s["max_ctx"], scale=s["scale"], k_scale=s["k_scale"],
                                        v_scale=s["v_scale"]), s["mass"]
    if c["kind"] == "observe":
        ops.prompt_mass(s["q"], s["k"], s["table"], s["q_start"], s["q_len"], s["ctx"], s["mass"], max_q_len=s["max_q_len"], max_ctx=s["max_ctx"], scale=s["scale"],
                        last=c["last"], k_scale=s["k_scale"])
        return s["mass"]
    kept, length = ops.kv_evict(s["k"], s["v"], s["table"], s["ctx"], s["mass"], keep=c["keep"], recent=c["recent"], max_ctx=s["max_ctx"], mass_out=s["mass_out"],
                                dst_table=s["dst"])
    caches = [s[name].view(torch.float8_e4m3fn) if s[name].dtype == torch.uint8 else s[name] for name in ("k", "v")]
    return (*caches, s["mass_out"], kept, length)


def run(state):
    if own:
        return _call(state)
    return {"decode": _decode, "observe": _observe, "evict": _evict}[state["case"]["kind"]](state)


def work(case):
    c = case
    ctx, new = _lengths(c)
    H, D, e = c["kv_heads"], c["dim"], 1 if c["cache"] == "e4m3" else 2
    tables = 4 * sum((n + c["block"] - 1) // c["block"] for n in ctx)
    if c["kind"] == "decode":
        rows = sum(ctx)
        return {"bytes": rows * H * (2 * D * e + 8) + 4 * c["seqs"] * c["heads"] * D + tables, "flops": 4 * c["heads"] * D * rows}
    if c["kind"] == "observe":
        seen = [min(c["last"] or b, b) for b in new]
        pairs = sum(w * n - w * (w - 1) // 2 for w, n in zip(seen, ctx))
        return {"bytes": sum(ctx) * H * (D * e + 8) + 2 * sum(seen) * c["heads"] * D + tables, "flops": 2 * c["heads"] * D * pairs}
    kept = sum(min(c["keep"], n) for n in ctx)
    columns = 4 * H * c["seqs"] * (max(ctx) + c["keep"])                  # the gathered weight and the list, as written
    return {"bytes": 4 * H * sum(ctx) + columns + 4 * kept * H * D * e + tables, "flops": 0}


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    ctx, new = _lengths(c)
    bs, H, G = c["block"], c["kv_heads"], c["heads"] // c["kv_heads"]

    def rows(name, i, n, scale):
        j = torch.arange(n, device="cuda")
        x = s[name].flatten(0, 1)[s["table"][i].long()[j // bs] * bs + j % bs]
        return x.view(torch.float8_e4m3fn).double() * scale.double() if x.dtype == torch.uint8 else x.double()

    if c["kind"] == "evict":
        kept = torch.full((c["seqs"], H, c["keep"]), -1, dtype=torch.int32, device="cuda")
        mass = torch.zeros_like(s["mass"], dtype=torch.float64)
        caches = [s["k"].clone(), s["v"].clone()]
        dst = s["table"] if s["dst"] is None else s["dst"]
        for i, n in enumerate(ctx):
            m = min(n, c["keep"])
            to = torch.arange(m, device="cuda")
            to = dst[i].long()[to // bs] * bs + to % bs
            for h in range(H):
                x = s["mass"][i, h, :n].double()
                x = torch.where(x.isnan(), -math.inf, x)
                if n > m:
                    old = n - c["recent"]
                    best = torch.sort(x[:old], descending=True, stable=True).indices[:m - c["recent"]]
                    idx = torch.cat([best.sort().values, torch.arange(old, n, device="cuda")])
                else:
                    idx = torch.arange(n, device="cuda")
                kept[i, h, :m] = idx.int()
                mass[i, h, :m] = s["mass"][i, h, idx].double()
                at = s["table"][i].long()[idx // bs] * bs + idx % bs
                for new_cache, name in zip(caches, ("k", "v")):
                    new_cache.flatten(0, 1)[to, h] = s[name].flatten(0, 1)[at, h]
        if c["cache"] == "e4m3":
            caches = [x.view(torch.float8_e4m3fn) for x in caches]
        return (*caches, mass, kept, torch.tensor([min(n, c["keep"]) for n in ctx], dtype=torch.int32, device="cuda"))

    mass = s["mass"].double()
    if c["kind"] == "decode":
        out = torch.zeros(c["seqs"], c["heads"], c["dim"], dtype=torch.float64, device="cuda")
        for i, n in enumerate(ctx):
            k, v = rows("k", i, n, s["k_scale"]), rows("v", i, n, s["v_scale"])
            z = torch.einsum("hgd,nhd->hgn", s["q"][i].double().view(H, G, -1), k) * s["scale"]
            p = torch.softmax(z, -1)
            out[i] = torch.einsum("hgn,nhd->hgd", p, v).reshape(c["heads"], -1)
            mass[i, :, :n] += p.sum(1)
        return out, mass
    start = s["q_start"].tolist()
    for i, (n, b) in enumerate(zip(ctx, new)):
        k = rows("k", i, n, s["k_scale"])
        first = b - min(c["last"] or b, b)
        for h in range(H):
            for t in range(first, b, 1024):
                q = s["q"][start[i] + t:start[i] + min(b, t + 1024), h * G:(h + 1) * G].double()
                z = torch.einsum("tgd,nd->gtn", q, k[:, h]) * s["scale"]
                limit = n - b + 1 + torch.arange(t, t + q.shape[0], device="cuda")
                z.masked_fill_(torch.arange(n, device="cuda") >= limit[:, None], -math.inf)
                mass[i, h, :n] += torch.softmax(z, -1).sum((0, 1))
    return mass
