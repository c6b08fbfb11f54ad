"""Prompts over a latent cache in expanded form (``csrc/mla_prompt.cu``): the keys and values of every head are made from the cached rows, c -> [W_k c | rotated
part] and W_v c, and attended as usual. A pair of query and cached token then costs 192 + 128 multiply-adds a head instead of the 576 + 512 of the absorbed
form (``mla_cuda.mla_attention``), and a cached token 512 x 256 a head in front: the form for portions of a few hundred tokens and more, not for decode."""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional

import torch

from . import _PERSIST_PREFILL, _count, _native, _stream, reference as ref, runtime
from .shared_attn import _bad, _check_ints, _check_places, _check_scale, _check_table

LATENT, ROPE, NOPE, VALUE = 512, 64, 128, 128
ROW, QK, KV = LATENT + ROPE, NOPE + ROPE, NOPE + VALUE

# MbMlaPromptArgs of csrc/shared_attn.h, field by field
_ARGS = struct.Struct("@3P q 6P N P 3q 8i f 4x")

_native.register_optional("mb_mla_prompt", [C.c_char_p, C.c_void_p])

_lib = None
# most bytes of gathered rows and expanded keys and values that a call holds: more heads go in several steps, of one head at the least
_WS_BYTES = 1 << 30
_ROW_BYTES = 2 * ROW + 1             # of a gathered row and what is remembered beside it


def _cached_rows(total_ctx: int, seqs: int) -> int:
    return (total_ctx + 127 * seqs) // 128 * 128             # every sequence begins on a multiple of 128


def _heads_at_once(rows: int, H: int) -> int:
    return max(1, min(H, (_WS_BYTES - rows * _ROW_BYTES) // (rows * KV * 2)))


def fits(total_ctx: int, seqs: int) -> bool:
    """Whether a call over so many cached tokens keeps to the workspace of 1 GB: some 640,000 do."""
    return _cached_rows(total_ctx, seqs) * (_ROW_BYTES + 2 * KV) <= _WS_BYTES


def _library():
    global _lib
    if _lib is None:
        L = _native.lib()
        size = L.mb_shared_attn_args
        size.argtypes, size.restype = [C.c_int], C.c_size_t
        if size(2) != _ARGS.size:
            raise RuntimeError(f"{_native.LIB_PATH} has argument structures of other sizes: build it again")
        L.mb_mla_prompt_ws.argtypes, L.mb_mla_prompt_ws.restype = [C.c_longlong, C.c_int, C.c_int], C.c_size_t
        _lib = L
    return _lib


def mla_prompt_attention(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, q_start: torch.Tensor, q_len: torch.Tensor, ctx_len: torch.Tensor,
                         w_kv: torch.Tensor, *, max_q_len: int, max_ctx: int, scale: float, total_ctx: Optional[int] = None) -> torch.Tensor:
    """Causal attention of prompts, or portions of prompts, over a paged latent cache: q [rows, H, 192] bf16 (128 dims without position, 64 rotated),
    cache [blocks, block, 1, 576] bf16 (512 of the latent, 64 of the rotated key), w_kv [H, 256, 512] bf16 (a head's keys without position, its values)
    -> [rows, H, 128] bf16. Sequence s has rows q_start[s] to q_start[s] + q_len[s], the last q_len[s] of its ctx_len[s] cached tokens; each token sees those
    up to itself, and one that sees none gives zeros. Rows of q that belong to no sequence are not written, and none belongs to two (on CUDA the sequences'
    results would meet in it, 16 bytes from one or the other; on the CPU such portions are refused). ``total_ctx``: the sum of ctx_len, or a bound of it (None:
    ``max_ctx`` a sequence); memory and the making of keys and values go by it. The workspace is 1152 bytes a cached token and 512 for each of the heads that
    are made at once: as many as 1 GB has room for, one at least.

    Keys and values are rounded to bf16, as cached ones would be (what is beyond its range is infinite), and so are the weights in the product with the
    values. A cached latent that is no number makes the rows that see it NaN, and no others. Lengths beyond ``max_q_len``, ``max_ctx`` or ``total_ctx``, rows
    that q does not have and blocks that the cache does not have set the status word (`check_status`), and a sequence with too many rows or cached tokens is
    left out; on the CPU they are refused. A CUDA call of no sequences looks at nothing and gives zeros."""
    where = "mla_prompt_attention"
    if cache.dim() != 4 or cache.shape[2] != 1 or cache.shape[3] != ROW or cache.dtype != torch.bfloat16 or not cache.is_contiguous():
        _bad(where, f"cache is contiguous bf16 [blocks, block, 1, {ROW}]")
    nb, bs = cache.shape[:2]
    if bs == 0 or (nb == 0 and max_ctx > 0):
        _bad(where, f"a cache of {nb} blocks of {bs} tokens holds nothing")
    if q.dim() != 3 or q.shape[2] != QK or q.dtype != torch.bfloat16 or not q.is_contiguous():
        _bad(where, f"q is contiguous bf16 [rows, heads, {QK}]")
    T, H, _ = q.shape
    if w_kv.shape != (H, KV, LATENT) or w_kv.dtype != torch.bfloat16 or not w_kv.is_contiguous() or H == 0:
        _bad(where, f"w_kv is contiguous bf16 [{H}, {KV}, {LATENT}]")
    if ctx_len.dim() != 1:
        _bad(where, "ctx_len is int32 [sequences]")
    S = ctx_len.shape[0]
    for name, x in (("q_start", q_start), ("q_len", q_len), ("ctx_len", ctx_len)):
        _check_ints(where, name, x, S)
    _check_table(where, "block_table", block_table, S, bs, max_ctx, "max_ctx")
    if max_q_len < 0 or max_q_len > 1 << 30:
        _bad(where, "max_q_len is from 0 to 2^30")
    if S > 65535 or H > 65535:
        _bad(where, "at most 65535 sequences and heads")
    total = S * max_ctx if total_ctx is None else min(total_ctx, S * max_ctx)
    rows = _cached_rows(total, S)
    if total < 0 or rows >= 1 << 31:
        _bad(where, f"total_ctx {total} is from 0 to 2^31")
    _check_scale(where, scale)
    _check_places(where, q, cache, block_table, q_start, q_len, ctx_len, w_kv)
    if not q.is_cuda:
        _check_values(where, T, nb, bs, block_table, q_start, q_len, ctx_len, max_q_len, max_ctx, total)
        return ref.mla_prompt_attention(q, cache, block_table, q_start, q_len, ctx_len, w_kv, scale)
    if (q.data_ptr() | cache.data_ptr() | w_kv.data_ptr()) & 15:
        _bad(where, "q, cache and w_kv begin on 16 bytes")
    dev = q.device
    nothing = rows == 0 or max_q_len == 0 or max_ctx == 0 or T == 0         # to be attended: lengths and places are looked at all the same
    out = (torch.zeros if nothing else torch.empty)(T, H, VALUE, dtype=torch.bfloat16, device=dev)
    if S == 0:
        return out
    L, rt = _library(), runtime(dev)
    each = 1 if nothing else _heads_at_once(rows, H)
    need = 0 if nothing else L.mb_mla_prompt_ws(rows, S, each)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    a = _ARGS.pack(q.data_ptr(), cache.data_ptr(), block_table.data_ptr(), block_table.stride(0), q_start.data_ptr(), q_len.data_ptr(), ctx_len.data_ptr(),
                   w_kv.data_ptr(), out.data_ptr(), ws.data_ptr(), need, rt.status.data_ptr(), nb, T, rows, S, H, bs, max_q_len, max_ctx, each, rt.sm_count,
                   _PERSIST_PREFILL, scale)
    _native.check(L.mb_mla_prompt(a, _stream()), "mla_prompt")
    _count(1 if nothing else 1 + 2 * ((H + each - 1) // each))
    return out


def _check_values(where, T, nb, bs, block_table, q_start, q_len, ctx_len, max_q_len, max_ctx, total) -> None:
    """CPU: what the kernels cut and report is refused."""
    if bool((ctx_len > max_ctx).any()) or bool((q_len > max_q_len).any()) or int(ctx_len.clamp(min=0).sum()) > total:
        _bad(where, f"a length is beyond max_q_len {max_q_len} or max_ctx {max_ctx}, or the sum beyond total_ctx {total}")
    if bool(((q_len > 0) & ((q_start < 0) | (q_start.long() + q_len > T))).any()):
        _bad(where, f"a portion has rows of q beyond its {T}")
    some = q_len > 0
    first, order = q_start[some].long().sort()
    if bool((first[1:] < (first + q_len[some].long()[order])[:-1]).any()):
        _bad(where, "two portions have a row of q in common")
    used = torch.arange(block_table.shape[1]) * bs < ctx_len[:, None]
    if bool((used & ((block_table < 0) | (block_table >= nb))).any()):
        _bad(where, f"the table has a block that the cache of {nb} does not have")
