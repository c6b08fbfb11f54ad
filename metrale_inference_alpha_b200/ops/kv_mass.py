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
    ctx_len = ctx_len + 1                            # a token, its row written at the former ctx_len
    out = paged_attention_mass(q, k, v, blocks, ctx_len, mass, ...)

with positions counted on as if nothing had gone: a cached key holds its
own rotation, so rows keep the distances that they had. Eviction leaves a head's rows in the order of their positions;
they belong to different tokens in different heads, and all have the same number. CUDA tensors run the kernels, CPU tensors
the fp32 restatements in ``reference.py``.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Tuple

import torch

from . import _count, _native, _stream, reference as ref, runtime

HEAD_DIMS = (64, 128, 256)
MAX_GROUP = 64                   # query heads that share a kv head

# MbMassArgs and MbEvictArgs of csrc/kv_mass.h, field by field. Calls of some ten microseconds pack them at once: a ctypes structure of as many fields takes
# twice as long to fill.
_MASS_ARGS = struct.Struct("@4P q 4P 2q 2P N 3P 2q 10i f 4x")
_EVICT_ARGS = struct.Struct("@P 2q P 2q 5P q P q 2P q 2P 10i")

for _name in ("mb_attn_mass", "mb_prompt_mass", "mb_kv_evict"):
    _native.register_optional(_name, [C.c_char_p, C.c_void_p])


_lib = None


def _library():
    """The kernel library, once its structures have been found to be those that are packed here."""
    global _lib
    if _lib is None:
        L = _native.lib()
        size = L.mb_kv_mass_args
        size.argtypes, size.restype = [C.c_int], C.c_size_t
        if (size(0), size(1)) != (_MASS_ARGS.size, _EVICT_ARGS.size):
            raise RuntimeError(f"{_native.LIB_PATH} has argument structures of other sizes: build it again")
        _lib = L
    return _lib


_ws_bytes: dict = {}


def _workspace(name: str, *sizes) -> int:
    fn = _ws_bytes.get(name)
    if fn is None:
        fn = getattr(_library(), name)
        fn.restype, fn.argtypes = C.c_size_t, [C.c_int] * len(sizes)
        _ws_bytes[name] = fn
    return fn(*sizes)


def _bad(where: str, what: str):
    raise ValueError(f"{where}: {what}")


# Checks stand in front of every call of a step that takes some ten microseconds, so their messages are put together only where they are needed.
def _check_cache(where, k_cache, v_cache, block_table, ctx_len, mass, max_ctx) -> Tuple[int, int, int, int, int]:
    """Shapes and types that all three share; (S, blocks, block, Hkv, D)."""
    shape, dtype = k_cache.shape, k_cache.dtype
    if len(shape) != 4 or (dtype != torch.bfloat16 and dtype != torch.uint8):
        _bad(where, "k_cache is [blocks, block, kv heads, dim], bf16 or e4m3 bytes")
    nb, bs, Hkv, D = shape
    if v_cache is not None and (v_cache.shape != shape or v_cache.dtype != dtype):
        _bad(where, "v_cache has the shape and type of k_cache")
    if not k_cache.is_contiguous() or (v_cache is not None and not v_cache.is_contiguous()):
        _bad(where, "caches are contiguous")
    if bs == 0 or Hkv == 0 or (nb == 0 and max_ctx > 0):
        _bad(where, f"a cache of {nb} blocks of {bs} tokens and {Hkv} kv heads holds nothing")
    if D not in HEAD_DIMS:
        _bad(where, f"head dim {D}, one of {HEAD_DIMS} is served")
    if ctx_len.dtype != torch.int32 or ctx_len.dim() != 1 or not ctx_len.is_contiguous():
        _bad(where, "ctx_len is int32 [sequences]")
    S, table, m = ctx_len.shape[0], block_table.shape, mass.shape
    if block_table.dtype != torch.int32 or len(table) != 2 or table[0] != S or (table[1] > 1 and block_table.stride(1) != 1):
        _bad(where, "block_table is int32 [sequences, blocks of a sequence]")
    if mass.dtype != torch.float32 or len(m) != 3 or m[0] != S or m[1] != Hkv or (m[2] > 1 and mass.stride(2) != 1):
        _bad(where, "mass is fp32 [sequences, kv heads, columns], columns next to each other")
    if max_ctx < 0 or m[2] < max_ctx or table[1] * bs < max_ctx:
        _bad(where, f"max_ctx {max_ctx} is beyond the columns of mass ({m[2]}) or the rows of block_table ({table[1] * bs})")
    if max_ctx > 1 << 30:
        _bad(where, "max_ctx is at most 2^30")
    return S, nb, bs, Hkv, D


def _check_queries(where, q, rows, Hkv, D) -> int:
    shape = q.shape
    if q.dtype != torch.bfloat16 or len(shape) != 3 or shape[2] != D or (rows >= 0 and shape[0] != rows) or not q.is_contiguous():
        _bad(where, f"q is contiguous bf16 [{'rows' if rows < 0 else rows}, heads, {D}]")
    Hq = shape[1]
    if Hq == 0 or Hq % Hkv != 0 or Hq // Hkv > MAX_GROUP:
        _bad(where, f"{Hq} query heads over {Hkv} kv heads: whole groups of up to {MAX_GROUP}")
    return Hq


def _check_places(where, *tensors) -> None:
    """CUDA: one device, the current one, whose stream the launches go to; CPU: all there."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _bad(where, "tensors lie on different devices")
    if dev >= 0 and dev != torch._C._cuda_getDevice():
        _bad(where, f"tensors lie on device {dev}, the current device is another one")


def _check_values(where, nb, bs, ctx_len, max_ctx, *tables) -> None:
    """CPU: what the kernels cut and report is refused. Each of `tables` comes with the rows of every sequence that are looked up in it."""
    if bool((ctx_len > max_ctx).any()):
        _bad(where, f"a length of ctx_len is beyond max_ctx {max_ctx}")
    for table, rows in tables:
        used = torch.arange(table.shape[1]) * bs < rows[:, None]
        if bool((used & ((table < 0) | (table >= nb))).any()):
            _bad(where, f"a table has a block that the cache of {nb} does not have")


def _check_scales(where, cache, scale, *scales) -> None:
    if not scale > 0:
        _bad(where, "scale is positive")
    if cache.dtype == torch.uint8:
        for s in scales:
            if s is None or s.dtype != torch.float32 or s.numel() != 1:
                _bad(where, "an e4m3 cache comes with fp32 scales of one element")


def _check_rows(where, name, mass) -> None:
    """No two rows of [S, H, columns] share memory."""
    S, H, n = mass.shape
    a, b = mass.stride(1), mass.stride(0)
    if a >= n and b >= a * H:
        return
    (a, x), (b, y) = sorted(((a, H), (b, S)))
    if not ((x < 2 or a >= n) and (y < 2 or b >= a * (x - 1) + n)):
        _bad(where, f"rows of {name} share memory")


def _columns_overlap(x, y) -> bool:
    """Whether two fp32 buffers [S, H, columns] of as many rows share memory, or may, and are not the same rows: of those that lie between each other parts of
    one buffer are told apart."""
    (S, H, n), m, (a, b, _), (c, e, _) = x.shape, y.shape[2], x.stride(), y.stride()
    d = (y.data_ptr() - x.data_ptr()) // 4
    if d >= (S - 1) * a + (H - 1) * b + n or -d >= (S - 1) * c + (H - 1) * e + m or not (S and H and n and m):
        return False
    if (a != c and S > 1) or (b != e and H > 1):
        return True
    for step, p, q in ((a, (H - 1) * b + n, (H - 1) * b + m), (b if S == 1 or b and a % b == 0 else 0, n, m)):       # windows of a sequence, of a row
        if step and d % step >= p and step - d % step >= q:
            return False
    return d != 0


def _tables_overlap(a, b) -> bool:
    """Whether two int32 tables of as many rows share memory; columns of a table lie next to each other."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (S, m), n, d = a.shape, b.shape[1], (b.data_ptr() - a.data_ptr()) // 4
    x, y = a.stride(0), b.stride(0)
    if d >= (S - 1) * x + m or -d >= (S - 1) * y + n:
        return False
    # between each other: slices of the rows of one buffer
    return not (S > 1 and x == y and x >= max(m, n) and d % x >= m and x - d % x >= n)


# most bytes of workspace that a call has under way (a decode step's logits, a prompt's queries and the copy of its keys): more sequences go in several steps
_WS_BYTES = 1 << 30


def _step(name: str, S: int, most: int, *sizes) -> Tuple[int, int]:
    """Sequences that are worked on at once, and their workspace."""
    step = min(S, most)
    need = _workspace(name, step, *sizes)
    if need > _WS_BYTES and step > 1:
        step = min(step, max(1, _WS_BYTES // _workspace(name, 1, *sizes)))
        need = _workspace(name, step, *sizes)
    return step, need


def paged_attention_mass(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, ctx_len: torch.Tensor,
                         mass: torch.Tensor, *, max_ctx: int, scale: float, k_scale: Optional[torch.Tensor] = None,
                         v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token a sequence over a paged cache, as ``paged_attention``, whose weights are added up:
    q [S, Hq, D] bf16 -> [S, Hq, D] bf16, and mass[s, h, j] grows by the weights that the query heads of kv head h give to
    cached row j (they sum to Hq / Hkv over j). The new token's own row is one of the ``ctx_len``. A sequence of length 0 (a lane
    that pads the batch) gives zeros and leaves its mass, and so does a row whose scores are all -inf. A length beyond ``max_ctx`` or a block that the cache does not have sets the
    status word (`check_status`); on the CPU it is refused. A CUDA call of no sequences or with a ``max_ctx`` of 0 looks at neither."""
    where = "paged_attention_mass"
    S, nb, bs, Hkv, D = _check_cache(where, k_cache, v_cache, block_table, ctx_len, mass, max_ctx)
    Hq = _check_queries(where, q, S, Hkv, D)
    if D == 64 and bs % 2 and k_cache.dtype == torch.uint8:
        _bad(where, f"an e4m3 cache of head dim 64 has blocks of an even number of tokens, not {bs}")
    _check_rows(where, "mass", mass)
    _check_scales(where, k_cache, scale, k_scale, v_scale)
    _check_places(where, q, k_cache, v_cache, block_table, ctx_len, mass, k_scale, v_scale)
    if not q.is_cuda:
        _check_values(where, nb, bs, ctx_len, max_ctx, (block_table, ctx_len))
        return ref.paged_attention_mass(q, k_cache, v_cache, block_table, ctx_len, mass, scale, k_scale, v_scale)
    if S == 0 or max_ctx == 0:
        return torch.zeros_like(q)
    out = torch.empty_like(q)
    launch, rt = _library().mb_attn_mass, runtime(q.device)
    step, need = _step("mb_attn_mass_ws", S, 1024, Hq, D, max_ctx)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    fp8 = int(k_cache.dtype == torch.uint8)
    ks, vs = (k_scale.data_ptr(), v_scale.data_ptr()) if fp8 else (0, 0)
    qp, op, tp, cp, mp = q.data_ptr(), out.data_ptr(), block_table.data_ptr(), ctx_len.data_ptr(), mass.data_ptr()
    tld, mseq, mhead, row = block_table.stride(0), mass.stride(0), mass.stride(1), Hq * D * 2
    for s in range(0, S, step):
        a = _MASS_ARGS.pack(qp + s * row, k_cache.data_ptr(), v_cache.data_ptr(), tp + 4 * s * tld, tld, 0, 0, cp + 4 * s, mp + 4 * s * mseq, mseq, mhead, op + s * row,
                            ws.data_ptr(), need, ks, vs, rt.status.data_ptr(), nb, 0, min(step, S - s), Hq, Hkv, D, bs, fp8, max_ctx, 1, 1, rt.sm_count, scale)
        _native.check(launch(a, _stream()), "attn_mass")
        _count(2)
    return out


def prompt_mass(q: torch.Tensor, k_cache: torch.Tensor, block_table: torch.Tensor, q_start: torch.Tensor, q_len: torch.Tensor, ctx_len: torch.Tensor,
                mass: torch.Tensor, *, max_q_len: int, max_ctx: int, scale: float, last: int = 0, k_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The weights that the last ``last`` tokens of every sequence's portion (0: all of them) give to what is cached, added to
    ``mass``, which is returned. q [rows, Hq, D] bf16 holds the portions one behind the other as for ``paged_attention`` (sequence s: rows
    q_start[s] to q_start[s] + q_len[s], the last q_len[s] of its ctx_len[s] cached tokens; each token sees those up to itself). Rows
    that see nothing, or nothing but scores of -inf, give nothing. ``k_scale`` is positive (what is not leaves NaN). A length beyond ``max_q_len`` or ``max_ctx``, rows that q does not have and blocks that the cache
    does not have set the status word; on the CPU they are refused. A CUDA call of no sequences, no rows or with a maximum of 0 looks at none of them."""
    where = "prompt_mass"
    S, nb, bs, Hkv, D = _check_cache(where, k_cache, None, block_table, ctx_len, mass, max_ctx)
    Hq = _check_queries(where, q, -1, Hkv, D)
    for x in (q_start, q_len):
        if x.dtype != torch.int32 or x.shape != ctx_len.shape or not x.is_contiguous():
            _bad(where, "q_start and q_len are int32 [sequences]")
    if last < 0 or max_q_len < 0:
        _bad(where, "last and max_q_len are not negative")
    if max_q_len > 1 << 30:
        _bad(where, "max_q_len is at most 2^30")
    _check_rows(where, "mass", mass)
    _check_scales(where, k_cache, scale, k_scale)
    _check_places(where, q, k_cache, block_table, q_start, q_len, ctx_len, mass, k_scale)
    if not q.is_cuda:
        _check_values(where, nb, bs, ctx_len, max_ctx, (block_table, torch.where(q_len > 0, ctx_len, 0)))
        if bool((q_len > max_q_len).any()):
            _bad(where, f"a length of q_len is beyond max_q_len {max_q_len}")
        if bool(((q_len > 0) & ((q_start < 0) | (q_start.long() + q_len > q.shape[0]))).any()):
            _bad(where, f"a portion has rows of q beyond its {q.shape[0]}")
        return ref.prompt_mass(q, k_cache, block_table, q_start, q_len, ctx_len, mass, scale, last, k_scale)
    if S == 0 or q.shape[0] == 0 or max_q_len == 0 or max_ctx == 0:
        return mass
    seen, fp8 = min(last or max_q_len, max_q_len), int(k_cache.dtype == torch.uint8)
    if seen * (Hq // Hkv) > 1 << 25:
        _bad(where, f"{seen} tokens of {Hq // Hkv} heads a group are more than 2^25 rows")
    step, need = _step("mb_prompt_mass_ws", S, 65535, Hq, Hkv, D, bs, seen, max_ctx, fp8)
    ws, rt, launch = torch.empty(need, dtype=torch.uint8, device=q.device), runtime(q.device), _library().mb_prompt_mass
    tp, qs, ql, cp, mp, tld, mseq = (block_table.data_ptr(), q_start.data_ptr(), q_len.data_ptr(), ctx_len.data_ptr(), mass.data_ptr(), block_table.stride(0),
                                     mass.stride(0))
    for s in range(0, S, step):
        a = _MASS_ARGS.pack(q.data_ptr(), k_cache.data_ptr(), 0, tp + 4 * s * tld, tld, qs + 4 * s, ql + 4 * s, cp + 4 * s, mp + 4 * s * mseq, mseq, mass.stride(1), 0,
                            ws.data_ptr(), need, k_scale.data_ptr() if fp8 else 0, 0, rt.status.data_ptr(), nb, q.shape[0], min(step, S - s), Hq, Hkv, D, bs, fp8,
                            max_ctx, max_q_len, seen, rt.sm_count, scale)
        _native.check(launch(a, _stream()), "prompt_mass")
        _count(2)                                                # the two passes; copies and joins, which go by the sizes, are not counted
    return mass


def kv_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, ctx_len: torch.Tensor, mass: torch.Tensor, *, keep: int, recent: int,
             max_ctx: int, mass_out: Optional[torch.Tensor] = None, dst_table: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cuts every sequence's cache to ``keep`` rows a kv head: the last ``recent`` rows stay, and of the others those of the largest mass
    (of equal ones the first; a NaN counts as -inf). Sequences of at most ``keep`` rows stay whole. The rows that stay move to the
    front in their order; returns (kept [S, kv heads, keep] int32, their former places, -1 behind the last; new lengths [S] int32).

    ``dst_table`` [S, >= keep rows' blocks]: blocks that take the rows, none of which a sequence of the call reads; the source's stay as
    they were, so that they may be shared with a prefix cache or other sequences. Without it the rows move inside the sequence's own
    blocks, which then no other sequence may hold. ``mass_out`` takes the mass of the rows that stay and zeros behind them up to column
    ``max_ctx``; without it ``mass`` does. A length beyond ``max_ctx`` or a block that the cache does not have sets the status word; on the CPU it is
    refused. A CUDA call of no sequences or with a ``max_ctx`` of 0 looks at neither."""
    where = "kv_evict"
    S, nb, bs, Hkv, D = _check_cache(where, k_cache, v_cache, block_table, ctx_len, mass, max_ctx)
    if abs(k_cache.data_ptr() - v_cache.data_ptr()) < k_cache.numel() * k_cache.element_size():
        _bad(where, "k_cache and v_cache share memory")     # they move side by side: the one would write rows that the other has not read
    if keep < 1 or keep > 1 << 30 or recent < 0 or recent > keep:
        _bad(where, f"keep {keep} is from 1 to 2^30 and recent {recent} at most keep")
    mo = mass
    if mass_out is not None:
        mo, m = mass_out, mass_out.shape
        if mo.dtype != torch.float32 or len(m) != 3 or m[0] != S or m[1] != Hkv or m[2] < max_ctx or (m[2] > 1 and mo.stride(2) != 1):
            _bad(where, "mass_out is fp32 [sequences, kv heads, at least max_ctx columns]")
        if _columns_overlap(mass, mo):
            _bad(where, "mass_out overlaps mass")
    _check_rows(where, "mass_out", mo)
    dst, moved = block_table, max_ctx if keep < max_ctx else 0                 # and the rows of a sequence that others may not have
    if dst_table is not None:
        dst, m, moved = dst_table, dst_table.shape, min(keep, max_ctx)
        if dst_table.dtype != torch.int32 or len(m) != 2 or m[0] != S or m[1] * bs < moved or (m[1] > 1 and dst_table.stride(1) != 1):
            _bad(where, f"dst_table is int32 [sequences, blocks for {moved} rows]")
        if _tables_overlap(block_table, dst_table):
            _bad(where, "dst_table and block_table share memory; without dst_table rows move in place")
    if S > 1 and dst.stride(0) < (moved + bs - 1) // bs:
        _bad(where, f"sequences share rows of {'block_table, which are moved in place' if dst_table is None else 'dst_table'}")
    _check_places(where, k_cache, v_cache, block_table, ctx_len, mass, mo, dst_table)
    if not k_cache.is_cuda:
        _check_values(where, nb, bs, ctx_len, max_ctx, (block_table, ctx_len), *([] if dst_table is None else [(dst_table, ctx_len.clamp(max=keep))]))
        return ref.kv_evict(k_cache, v_cache, block_table, ctx_len, mass, keep, recent, max_ctx, mo, dst_table)
    dev = k_cache.device
    kept, new_len = torch.empty(S, Hkv, keep, dtype=torch.int32, device=dev), torch.empty(S, dtype=torch.int32, device=dev)
    if S == 0 or max_ctx == 0:
        return kept.fill_(-1), new_len.zero_()
    own = torch.empty(S * Hkv * (keep + 1), dtype=torch.int32, device=dev)     # of a sequence and head: the rows' slots, the first that moves
    launch, status = _library().mb_kv_evict, runtime(dev).status.data_ptr()
    (ma, mb, _), (oa, ob, _), tld, dld, row, slots = mass.stride(), mo.stride(), block_table.stride(0), dst.stride(0), 4 * Hkv * keep, own.data_ptr()
    mp, op, cp, kp, np, tp, dp, first = (mass.data_ptr(), mo.data_ptr(), ctx_len.data_ptr(), kept.data_ptr(), new_len.data_ptr(), block_table.data_ptr(), dst.data_ptr(),
                                         slots + S * row)
    for s in range(0, S, 65535):
        a = _EVICT_ARGS.pack(mp + 4 * s * ma, ma, mb, op + 4 * s * oa, oa, ob, cp + 4 * s, kp + s * row, np + 4 * s, first + 4 * s * Hkv, tp + 4 * s * tld, tld,
                             dp + 4 * s * dld, dld, k_cache.data_ptr(), v_cache.data_ptr(), nb, status, slots + s * row, min(65535, S - s), Hkv, keep, recent, max_ctx, bs,
                             D * k_cache.element_size(), dst_table is None, 0, 0)
        _native.check(launch(a, _stream()), "kv_evict")
        _count(2)
    return kept, new_len
