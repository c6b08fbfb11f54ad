"""A paged cache that is held to a budget of tokens by the attention weight that they gather (``csrc/kv_mass.cu``,
``csrc/kv_observe.cu``):

``paged_attention_mass``  decode attention, one new token a sequence, that adds every cached token's weight to ``mass``
``prompt_mass``           the weights that the last tokens of prompts (or of portions of them) give to what is cached
``kv_evict``              the cached tokens of each kv head that gathered least go, the others move to the front

``mass`` is fp32 [sequences, kv heads, columns]: column j of sequence s belongs to its cached row j, columns behind the
context are zero. It is kept by sequence and not by block, since sequences that share the blocks of a prefix look at them
differently; a batch of lanes may pass a slice of a larger buffer (columns next to each other). A decode loop over a prompt is

    prompt_mass(q, k, ..., mass, last=32)            # per layer, behind the prompt's attention
    kept, ctx_len = kv_evict(k, v, ..., mass, keep=4096, recent=64, dst_table=blocks)
    out = paged_attention_mass(q, k, v, blocks, ctx_len + 1, mass, ...)

with the new token's row written at slot ctx_len and positions counted on as if nothing had gone: a cached key holds its
own rotation, so rows keep the distances that they had. Eviction leaves a head's rows in the order of their positions;
they belong to different tokens in different heads, and all have the same number. CUDA tensors run the kernels, CPU tensors
the fp32 restatements in ``reference.py``.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _native, reference as ref

_p, _i, _ll = C.c_void_p, C.c_int, C.c_longlong

HEAD_DIMS = (64, 128, 256)
MAX_GROUP = 64                   # query heads that share a kv head


class _MassArgs(C.Structure):
    _fields_ = [("q", _p), ("k_cache", _p), ("v_cache", _p), ("block_table", _p), ("table_ld", _ll), ("q_start", _p), ("q_len", _p), ("ctx_len", _p),
                ("mass", _p), ("mass_seq", _ll), ("mass_head", _ll), ("out", _p), ("ws", _p), ("ws_bytes", C.c_size_t), ("k_scale", _p), ("v_scale", _p),
                ("status", _p), ("num_blocks", _ll), ("q_rows", _ll), ("num_seqs", _i), ("Hq", _i), ("Hkv", _i), ("D", _i), ("block_size", _i), ("fp8", _i),
                ("max_ctx", _i), ("max_q_len", _i), ("last", _i), ("sm_count", _i), ("scale", C.c_float)]


class _EvictArgs(C.Structure):
    _fields_ = [("mass", _p), ("mass_seq", _ll), ("mass_head", _ll), ("mass_out", _p), ("out_seq", _ll), ("out_head", _ll), ("ctx_len", _p), ("kept", _p),
                ("new_len", _p), ("first", _p), ("block_table", _p), ("table_ld", _ll), ("dst_table", _p), ("dst_ld", _ll), ("k_cache", _p), ("v_cache", _p),
                ("num_blocks", _ll), ("status", _p), ("slots", _p), ("num_seqs", _i), ("Hkv", _i), ("keep", _i), ("recent", _i), ("max_ctx", _i), ("block_size", _i),
                ("row_bytes", _i), ("in_place", _i), ("block_shift", _i)]


_native.register_optional("mb_attn_mass", [C.POINTER(_MassArgs), _p])
_native.register_optional("mb_prompt_mass", [C.POINTER(_MassArgs), _p])
_native.register_optional("mb_kv_evict", [C.POINTER(_EvictArgs), _p])


def _sizes(name: str):
    fn = getattr(_native.lib(), name)
    fn.restype = C.c_size_t
    return fn


def _refuse(cond: bool, what: str) -> None:
    if cond:
        raise ValueError(what)


def _check_cache(where, k_cache, v_cache, block_table, ctx_len, mass, max_ctx) -> Tuple[int, int, int, int, int]:
    """Shapes, types and places that all three share; (S, blocks, block, Hkv, D)."""
    _refuse(k_cache.dim() != 4 or k_cache.dtype not in (torch.bfloat16, torch.uint8), f"{where}: k_cache is [blocks, block, kv heads, dim], bf16 or e4m3 bytes")
    nb, bs, Hkv, D = k_cache.shape
    _refuse(v_cache is not None and (v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype), f"{where}: v_cache has the shape and type of k_cache")
    _refuse(not k_cache.is_contiguous() or (v_cache is not None and not v_cache.is_contiguous()), f"{where}: caches are contiguous")
    _refuse(D not in HEAD_DIMS, f"{where}: head dim {D}, one of {HEAD_DIMS} is served")
    S = ctx_len.numel()
    _refuse(ctx_len.dtype != torch.int32 or ctx_len.dim() != 1 or not ctx_len.is_contiguous(), f"{where}: ctx_len is int32 [sequences]")
    _refuse(block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != S or (block_table.shape[1] > 1 and block_table.stride(1) != 1),
            f"{where}: block_table is int32 [sequences, blocks of a sequence]")
    _refuse(mass.dtype != torch.float32 or mass.dim() != 3 or mass.shape[:2] != (S, Hkv) or (mass.shape[2] > 1 and mass.stride(2) != 1),
            f"{where}: mass is fp32 [sequences, kv heads, columns], columns next to each other")
    _refuse(max_ctx < 0 or mass.shape[2] < max_ctx or block_table.shape[1] * bs < max_ctx,
            f"{where}: max_ctx {max_ctx} is beyond the columns of mass ({mass.shape[2]}) or the rows of block_table ({block_table.shape[1] * bs})")
    _refuse(max_ctx > 1 << 30, f"{where}: max_ctx is at most 2^30")
    return S, nb, bs, Hkv, D


def _check_places(where, tensors) -> None:
    """CUDA: one device, the current one, whose stream the launches go to; CPU: all there."""
    dev = tensors[0].device
    _refuse(any(t is not None and t.device != dev for t in tensors), f"{where}: tensors lie on different devices")
    _refuse(dev.type == "cuda" and dev.index != torch.cuda.current_device(), f"{where}: tensors lie on {dev}, the current device is another one")


def _check_scales(where, cache, scale, scales) -> None:
    _refuse(not scale > 0, f"{where}: scale is positive")
    _refuse(cache.dtype == torch.uint8 and any(s is None or s.dtype != torch.float32 or s.numel() < 1 for s in scales), f"{where}: an e4m3 cache comes with fp32 scales")


def _rows_apart(mass: torch.Tensor) -> bool:
    """No two rows of [S, H, columns] share memory."""
    S, H, n = mass.shape
    a, b = sorted(((mass.stride(1), H), (mass.stride(0), S)))
    return (a[1] < 2 or a[0] >= n) and (b[1] < 2 or b[0] >= (a[0] * (a[1] - 1) + n))


# most bytes of logits that a decode step has under way; more sequences go in several steps
_WS_BYTES = 1 << 30


def paged_attention_mass(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, ctx_len: torch.Tensor,
                         mass: torch.Tensor, *, max_ctx: int, scale: float, k_scale: Optional[torch.Tensor] = None,
                         v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token a sequence over a paged cache, as ``paged_attention``, whose weights are added up:
    q [S, Hq, D] bf16 -> [S, Hq, D] bf16, and mass[s, h, j] grows by the weights that the query heads of kv head h give to
    cached row j (they sum to Hq / Hkv over j). The new token's own row is one of the ``ctx_len``. A sequence of length 0 (a lane
    that pads the batch) gives zeros and leaves its mass. A length beyond ``max_ctx`` or a block that the cache does not have sets the
    status word (`check_status`)."""
    where = "paged_attention_mass"
    S, nb, bs, Hkv, D = _check_cache(where, k_cache, v_cache, block_table, ctx_len, mass, max_ctx)
    _refuse(q.dtype != torch.bfloat16 or q.dim() != 3 or q.shape[0] != S or q.shape[2] != D or not q.is_contiguous(), f"{where}: q is contiguous bf16 [sequences, heads, {D}]")
    Hq = q.shape[1]
    _refuse(Hq == 0 or Hq % Hkv != 0 or Hq // Hkv > MAX_GROUP, f"{where}: {Hq} query heads over {Hkv} kv heads: whole groups of up to {MAX_GROUP}")
    _refuse(not _rows_apart(mass), f"{where}: rows of mass share memory")
    _check_scales(where, k_cache, scale, (k_scale, v_scale))
    _check_places(where, (q, k_cache, v_cache, block_table, ctx_len, mass, k_scale, v_scale))
    if not q.is_cuda:
        return ref.paged_attention_mass(q, k_cache, v_cache, block_table, ctx_len, mass, scale, k_scale, v_scale)
    from . import _count, _ptr, _stream, runtime
    out = torch.empty_like(q)
    if S == 0:
        return out
    L, rt, sizes = _native.lib(), runtime(q.device), _sizes("mb_attn_mass_ws")
    one = sizes(1, Hq, D, max_ctx)
    step = min(S, max(1, _WS_BYTES // max(1, one)), 1024)
    ws = torch.empty(sizes(step, Hq, D, max_ctx), dtype=torch.uint8, device=q.device)
    for s in range(0, S, step):
        n = min(step, S - s)
        a = _MassArgs(q.data_ptr() + s * Hq * D * 2, _ptr(k_cache), _ptr(v_cache), block_table.data_ptr() + s * block_table.stride(0) * 4, block_table.stride(0), None,
                      None, ctx_len.data_ptr() + s * 4, mass.data_ptr() + s * mass.stride(0) * 4, mass.stride(0), mass.stride(1), out.data_ptr() + s * Hq * D * 2,
                      _ptr(ws), ws.numel(), _ptr(k_scale), _ptr(v_scale), _ptr(rt.status), nb, 0, n, Hq, Hkv, D, bs, int(k_cache.dtype == torch.uint8), max_ctx, 1, 1,
                      rt.sm_count, scale)
        _native.check(L.mb_attn_mass(C.byref(a), _stream()), f"attn_mass[S={n} ctx={max_ctx} D={D}]")
        _count(2)
    return out


def prompt_mass(q: torch.Tensor, k_cache: torch.Tensor, block_table: torch.Tensor, q_start: torch.Tensor, q_len: torch.Tensor, ctx_len: torch.Tensor,
                mass: torch.Tensor, *, max_q_len: int, max_ctx: int, scale: float, last: int = 0, k_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The weights that the last ``last`` tokens of every sequence's portion (0: all of them) give to what is cached, added to
    ``mass``, which is returned. q [rows, Hq, D] bf16 holds the portions one behind the other as for ``paged_attention`` (sequence s: rows
    q_start[s] to q_start[s] + q_len[s], the last q_len[s] of its ctx_len[s] cached tokens; each token sees those up to itself). Rows
    that see nothing give nothing. A length beyond ``max_q_len`` or ``max_ctx``, rows that q does not have and blocks that the cache
    does not have set the status word."""
    where = "prompt_mass"
    S, nb, bs, Hkv, D = _check_cache(where, k_cache, None, block_table, ctx_len, mass, max_ctx)
    _refuse(q.dtype != torch.bfloat16 or q.dim() != 3 or q.shape[2] != D or not q.is_contiguous(), f"{where}: q is contiguous bf16 [rows, heads, {D}]")
    Hq = q.shape[1]
    _refuse(Hq == 0 or Hq % Hkv != 0 or Hq // Hkv > MAX_GROUP, f"{where}: {Hq} query heads over {Hkv} kv heads: whole groups of up to {MAX_GROUP}")
    _refuse(any(x.dtype != torch.int32 or x.shape != ctx_len.shape or not x.is_contiguous() for x in (q_start, q_len)), f"{where}: q_start and q_len are int32 [sequences]")
    _refuse(last < 0 or max_q_len < 0, f"{where}: last and max_q_len are not negative")
    _refuse(not _rows_apart(mass), f"{where}: rows of mass share memory")
    _check_scales(where, k_cache, scale, (k_scale,))
    _check_places(where, (q, k_cache, block_table, q_start, q_len, ctx_len, mass, k_scale))
    if not q.is_cuda:
        return ref.prompt_mass(q, k_cache, block_table, q_start, q_len, ctx_len, mass, scale, last, k_scale)
    if S == 0 or q.shape[0] == 0 or max_q_len == 0 or max_ctx == 0:
        return mass
    from . import _count, _ptr, _stream, runtime
    seen = min(last or max_q_len, max_q_len)
    ws = torch.empty(_sizes("mb_prompt_mass_ws")(S, Hq, Hkv, D, seen, max_ctx, int(k_cache.dtype == torch.uint8)), dtype=torch.uint8, device=q.device)
    rt = runtime(q.device)
    a = _MassArgs(_ptr(q), _ptr(k_cache), None, _ptr(block_table), block_table.stride(0), _ptr(q_start), _ptr(q_len), _ptr(ctx_len), _ptr(mass), mass.stride(0),
                  mass.stride(1), None, _ptr(ws), ws.numel(), _ptr(k_scale), None, _ptr(rt.status), nb, q.shape[0], S, Hq, Hkv, D, bs,
                  int(k_cache.dtype == torch.uint8), max_ctx, max_q_len, seen, rt.sm_count, scale)
    _native.check(_native.lib().mb_prompt_mass(C.byref(a), _stream()), f"prompt_mass[S={S} last={seen} ctx={max_ctx} D={D}]")
    _count(2)
    return mass


def kv_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, ctx_len: torch.Tensor, mass: torch.Tensor, *, keep: int, recent: int,
             max_ctx: int, mass_out: Optional[torch.Tensor] = None, dst_table: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cuts every sequence's cache to ``keep`` rows a kv head: the last ``recent`` rows stay, and of the others those of the largest mass
    (of equal ones the first; a NaN counts as -inf). Sequences of at most ``keep`` rows stay whole. The rows that stay move to the
    front in their order; returns (kept [S, kv heads, keep] int32, their former places, -1 behind the last; new lengths [S] int32).

    ``dst_table`` [S, >= keep rows' blocks]: blocks that take the rows, none of which a sequence of the call reads; the source's stay as
    they were, so that they may be shared with a prefix cache or other sequences. Without it the rows move inside the sequence's own
    blocks, which then no other sequence may hold. ``mass_out`` takes the mass of the rows that stay and zeros behind them up to column
    ``max_ctx``; without it ``mass`` does. A length beyond ``max_ctx`` or a block that the cache does not have sets the status word."""
    where = "kv_evict"
    S, nb, bs, Hkv, D = _check_cache(where, k_cache, v_cache, block_table, ctx_len, mass, max_ctx)
    _refuse(keep < 1 or recent < 0 or recent > keep, f"{where}: keep {keep} is at least 1 and recent {recent} at most keep")
    mo = mass if mass_out is None else mass_out
    _refuse(mo.dtype != torch.float32 or mo.dim() != 3 or mo.shape[:2] != (S, Hkv) or mo.shape[2] < max_ctx or (mo.shape[2] > 1 and mo.stride(2) != 1) or not _rows_apart(mo),
            f"{where}: mass_out is fp32 [sequences, kv heads, at least max_ctx columns] of its own")
    same = mo.data_ptr() == mass.data_ptr() and mo.stride() == mass.stride()
    span = [(t.data_ptr(), t.data_ptr() + 4 * (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride())))) for t in (mass, mo)] if mass.numel() and mo.numel() else None
    _refuse(not same and span is not None and span[0][0] < span[1][1] and span[1][0] < span[0][1], f"{where}: mass_out overlaps mass")
    held = min(keep, max_ctx)
    if dst_table is not None:
        _refuse(dst_table.dtype != torch.int32 or dst_table.dim() != 2 or dst_table.shape[0] != S or dst_table.shape[1] * bs < held or
                (dst_table.shape[1] > 1 and dst_table.stride(1) != 1), f"{where}: dst_table is int32 [sequences, blocks for {held} rows]")
    _check_places(where, (k_cache, v_cache, block_table, ctx_len, mass, mo, dst_table))
    if not k_cache.is_cuda:
        return ref.kv_evict(k_cache, v_cache, block_table, ctx_len, mass, keep, recent, max_ctx, mo, dst_table)
    from . import _count, _ptr, _stream, runtime
    kept = torch.empty(S, Hkv, keep, dtype=torch.int32, device=k_cache.device)
    new_len = torch.empty(S, dtype=torch.int32, device=k_cache.device)
    if S == 0:
        return kept, new_len
    own = torch.empty(S * Hkv * (keep + 1), dtype=torch.int32, device=k_cache.device)   # of a sequence and head: the rows' slots, the first that moves
    dst = block_table if dst_table is None else dst_table
    a = _EvictArgs(_ptr(mass), mass.stride(0), mass.stride(1), _ptr(mo), mo.stride(0), mo.stride(1), _ptr(ctx_len), _ptr(kept), _ptr(new_len), own.data_ptr() + 4 * S * Hkv * keep,
                   _ptr(block_table), block_table.stride(0), _ptr(dst), dst.stride(0), _ptr(k_cache), _ptr(v_cache), nb, _ptr(runtime(k_cache.device).status), _ptr(own), S, Hkv,
                   keep, recent, max_ctx, bs, D * k_cache.element_size(), int(dst_table is None), 0)
    _native.check(_native.lib().mb_kv_evict(C.byref(a), _stream()), f"kv_evict[S={S} ctx={max_ctx} keep={keep}]")
    _count(2)
    return kept, new_len
