"""Relative 2-norms of what attention over shared prefixes and expanded latent prompts may be off by: bounds that a wrong mask, a lost tile or a type with fewer bits passes.

Bounds element by element add every rounding up at its worst, which over thousands of keys leaves room for wrong results. Roundings of different numbers are
independent, so that squares add up: a weight in a type of half step h is off by h / sqrt(3) of itself at most in the mean (uniform over a step), an
output by what rounding the 64-bit one is seen to do. Sums over hundreds of rows keep to that within a few per cent."""
import math

import torch

import shared_attn_oracle as oracle

BF16, F16 = 2.0 ** -8, 2.0 ** -11                # half a step
ROOM = 1.25                                      # of the norm: a few hundred rows, whose weights may be one or two keys' each
ROOM_F16 = 1.1                                   # where nearly all of it is the outputs' rounding, which is computed


def _attend(z, v, seen, round_weights=None):
    """Keys last: (out, sum of p^2 v^2). `round_weights`: a type that weights relative to the row's largest are rounded to."""
    p, _ = oracle._softmax(z.masked_fill(~seen, -math.inf))
    p = p.masked_fill(~seen, 0.0)
    if round_weights is not None:
        top = p.amax(-1, keepdim=True).clamp(min=1e-300)
        p = (p / top * 1.37).to(round_weights).double() / 1.37 * top          # the running maximum of a kernel is not the row's
    return p @ v, (p.square() @ v.square()).sum()


def _bound(out, spread, half, more=0.0):
    """Relative 2-norm: the outputs' rounding to bf16, weights of half step `half`, `more`: further squares."""
    o = torch.cat([x.flatten() for x in out])
    r0 = (o.bfloat16().double() - o).square().sum()
    return float(((r0 + half * half / 3 * spread + more) / o.square().sum()).sqrt())


def distance(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


def latent(c, shift=0, without=None, rope=True):
    """(out in 64 bits over keys and values rounded to bf16 as the kernel's are, bound). `shift`: tokens that rows see more, `without`: keys that they do not, `rope`:
    whether scores have their rotated part."""
    T, H, _ = c["q"].shape
    out, spread, slips = torch.zeros(T, H, 128, dtype=torch.float64), 0.0, 0.0
    w = c["w"].double()
    for s in range(len(c["ctx"])):
        n, ql, at = max(0, int(c["ctx"][s])), int(c["q_len"][s]), int(c["q_start"][s])
        x = oracle._rows(c["cache"], c["table"][s], n)[:, 0]
        seen = torch.arange(n) < (n - ql + 1 + shift + torch.arange(ql))[:, None]
        if without is not None:
            seen[:, without] = False
        for h in range(H):
            kv = x[:, :512] @ w[h].T
            r = kv.bfloat16().double()
            # an element whose 32-bit sum (32 steps of 2^-23 of sums of this size) meets the middle between two numbers goes to the other one, a step away
            slip = 2 * 2.0 ** -18 * (x[:, :512].square() @ w[h].square().T).sqrt() * 2.0 ** -7 * kv.abs()
            q = c["q"][at:at + ql, h].double()
            z = (q[:, :128] @ r[:, :128].T + (q[:, 128:] @ x[:, 512:].T if rope else 0.0)) * c["scale"]
            o, p2 = _attend(z, r[:, 128:], seen)
            out[at:at + ql, h] = o
            spread += p2
            zslip = (q[:, :128].square() @ slip[:, :128].T) * c["scale"] ** 2
            p2rows = oracle._softmax(z.masked_fill(~seen, -math.inf))[0].masked_fill(~seen, 0.0).square()
            slips += ((p2rows * zslip) @ (r[:, 128:].square() + o.square().mean(0))).sum() + (p2rows @ slip[:, 128:]).sum()
    return out, ROOM * _bound([out], spread, BF16, slips)


def shared(c, shift=0, without=None, round_weights=None):
    """(out in 64 bits, bound). `shift`: own tokens that rows see more, `without`: keys of a prefix that they do not see."""
    T, Hq, D = c["q"].shape
    H, n = c["k"].shape[2], c["n"]
    fp8 = c["k"].dtype == torch.uint8
    out, spread, start = torch.zeros(T, Hq, D, dtype=torch.float64), 0.0, c["start"].tolist()
    behind = {i: g for g, (a, b) in enumerate(zip(start, start[1:])) for i in range(a, b)}
    for s in range(len(c["ctx"])):
        own = max(0, int(c["ctx"][s]))
        parts, p = [(c["table"][s], own)], 0
        if s in behind:
            p = max(0, int(c["prefix"][behind[s]]))
            parts.insert(0, (c["prefix_table"][behind[s]], p))
        k, v = (torch.cat([oracle._rows(c[x], t, m, c[x + "_scale"]) for t, m in parts]).transpose(0, 1) for x in ("k", "v"))      # [H, keys, D]
        for t in range(n):
            q = c["q"][s * n + t].double().view(H, Hq // H, D)
            seen = torch.arange(p + own) < p + max(0, min(own, own - n + t + 1 + shift))
            if without is not None:
                seen[without] = False
            o, p2 = _attend(q @ k.transpose(1, 2) * c["scale"], v, seen, round_weights)
            out[s * n + t] = o.reshape(Hq, D)
            spread += p2
    return out, (ROOM_F16 if fp8 else ROOM) * _bound([out], spread, F16 if fp8 else BF16)


LATENT = [dict(new=[333], ctx=[333], heads=2), dict(new=[140, 3], ctx=[9001, 2050], heads=2), dict(new=[64], ctx=[1200], heads=3), dict(new=[257], ctx=[1000], heads=3),
          dict(new=[96], ctx=[12000], heads=3), dict(new=[200], ctx=[300], heads=2, spread=30.0), dict(new=[70, 200, 33], ctx=[70, 900, 500], heads=5)]
SHARED = [dict(ctx=[5, 90, 1] * 4, prefix=[700], start=[0, 12], heads=40, kv_heads=8, dim=128), dict(ctx=[40, 9, 200, 3], prefix=[300, 1029], start=[0, 2, 4], heads=24, kv_heads=2, dim=64, n=3),
          dict(ctx=[60] * 5, prefix=[2047, 1500], start=[0, 3, 5], heads=16, kv_heads=2, dim=256), dict(ctx=[3, 1200, 40], prefix=[6007], start=[0, 3], heads=20, kv_heads=2, dim=128),
          dict(ctx=[10 + i for i in range(60)], prefix=[400], start=[0, 60], heads=10, kv_heads=2, dim=128)]
