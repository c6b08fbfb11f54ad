"""Attention over what several sequences share (``csrc/shared_attn.cu``) and the joining of attention in parts (``csrc/attn_merge.cu``):

``shared_prefix_attention``  a decode or verify step of a batch in groups, each behind a prefix that is read once for the whole group
``merge_attention``          attention of the same queries over disjoint sets of keys, joined by their log-sum-exps

A group's prefix lies in the cache's blocks once (the blocks that the prefix cache handed to all of its sequences) and has a table of its own;
``block_table`` and ``ctx_len`` are then about what a sequence has behind it:

    out = shared_prefix_attention(q, k, v, prefix_table, prefix_len, group_start, own_table, own_len, max_prefix=..., max_ctx=..., scale=s)

which is ``paged_attention`` over prefix and own rows one behind the other. Prefixes of prefixes, or keys that lie elsewhere: attend each part with
``return_lse`` and join them with ``merge_attention``. CUDA tensors run the kernels, CPU tensors the fp32 restatements in ``reference.py``.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _count, _native, _stream, reference as ref, runtime

HEAD_DIMS = (64, 128, 256)
MAX_GROUP = 64                   # query heads that share a kv head
MAX_GROUPS = 1024                # groups of a call
MAX_PARTS = 16

# MbSharedArgs and MbMergeArgs of csrc/shared_attn.h, field by field
_SHARED_ARGS = struct.Struct("@4P q 3P q 4P N 3P q 11i f")
_MERGE_ARGS = struct.Struct(f"@{2 * MAX_PARTS + 2}P q 4i")

for _name in ("mb_shared_attn", "mb_merge_attn"):
    _native.register_optional(_name, [C.c_char_p, C.c_void_p])

_lib = None


def _library():
    """The kernel library, once its structures have been found to be those that are packed here."""
    global _lib
    if _lib is None:
        L = _native.lib()
        size = L.mb_shared_attn_args
        size.argtypes, size.restype = [C.c_int], C.c_size_t
        if (size(0), size(1)) != (_SHARED_ARGS.size, _MERGE_ARGS.size):
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


def _check_places(where, *tensors) -> None:
    """CUDA: one device, the current one, whose stream the launches go to; CPU: all there."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _bad(where, "tensors lie on different devices")
    if dev >= 0 and dev != torch._C._cuda_getDevice():
        _bad(where, f"tensors lie on device {dev}, the current device is another one")


def _check_scale(where, scale) -> None:
    """The kernels have it in 32 bits, and multiply a mask's -inf by it."""
    if not 2.0 ** -126 <= scale <= 2.0 ** 126:
        _bad(where, f"scale is positive, from 2^-126 to 2^126, not {scale}")


def _check_ints(where, name, x, n: int) -> None:
    if x.dtype != torch.int32 or x.dim() != 1 or x.shape[0] != n or not x.is_contiguous():
        _bad(where, f"{name} is contiguous int32 [{n}]")


def _check_table(where, name, x, rows: int, bs: int, most: int, what: str) -> None:
    if x.dtype != torch.int32 or x.dim() != 2 or x.shape[0] != rows or (x.shape[1] > 1 and x.stride(1) != 1):
        _bad(where, f"{name} is int32 [{rows}, blocks], a row's blocks next to each other")
    if most < 0 or most > 1 << 30 or (rows > 0 and x.shape[1] * bs < most):
        _bad(where, f"{what} {most} is beyond the rows of {name} ({x.shape[1] * bs}), or not from 0 to 2^30")


def shared_prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, prefix_table: torch.Tensor, prefix_len: torch.Tensor,
                            group_start: torch.Tensor, block_table: torch.Tensor, ctx_len: torch.Tensor, *, max_prefix: int, max_ctx: int, scale: float,
                            q_len: int = 1, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                            return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of ``q_len`` new tokens a sequence (one, or a draft's): q [S * q_len, Hq, D] bf16 -> bf16 of that shape, with ``return_lse`` also the rows'
    log-sum-exps fp32 [S * q_len, Hq] (natural logarithm, -inf for a row that sees nothing, whose output is zero).

    Sequences group_start[g] to group_start[g + 1] (int32 [groups + 1], rising) stand behind the prefix of group g: the first prefix_len[g] rows of
    prefix_table[g]. Every one of their tokens sees the whole of it, and of the sequence's own ctx_len[s] rows in block_table[s], whose last ``q_len`` belong
    to the new tokens, those up to its own. Sequences in front of the first group and behind the last have no prefix; the length and table of a group
    without sequences are not looked at. Lengths of zero and less hold nothing: a lane that pads the batch stands behind the last group and has length 0.
    Caches [blocks, block, kv heads, D] bf16, or e4m3 bytes with scales (behind a prefix of these an infinite query gives NaN). Lengths beyond ``max_prefix`` or ``max_ctx``, blocks that the cache does not have and
    groups that fall or leave the batch set the status word (`check_status`); on the CPU they are refused. A CUDA call of no sequences looks at none of them.
    How a prefix is shared out over the GPU, and with it the order of sums, follows from the whole call: unlike with ``paged_attention``, the last bits of a
    sequence's result may depend on its batch."""
    where = "shared_prefix_attention"
    shape, dtype = k_cache.shape, k_cache.dtype
    if len(shape) != 4 or (dtype != torch.bfloat16 and dtype != torch.uint8):
        _bad(where, "k_cache is [blocks, block, kv heads, dim], bf16 or e4m3 bytes")
    nb, bs, Hkv, D = shape
    if v_cache.shape != shape or v_cache.dtype != dtype:
        _bad(where, "v_cache has the shape and type of k_cache")
    if not k_cache.is_contiguous() or not v_cache.is_contiguous():
        _bad(where, "caches are contiguous")
    if bs == 0 or Hkv == 0 or (nb == 0 and (max_ctx > 0 or max_prefix > 0)):
        _bad(where, f"a cache of {nb} blocks of {bs} tokens and {Hkv} kv heads holds nothing")
    if D not in HEAD_DIMS:
        _bad(where, f"head dim {D}, one of {HEAD_DIMS} is served")
    if ctx_len.dim() != 1 or prefix_len.dim() != 1:
        _bad(where, "ctx_len and prefix_len are int32 of one dimension")
    S, groups = ctx_len.shape[0], prefix_len.shape[0]
    _check_ints(where, "ctx_len", ctx_len, S)
    _check_ints(where, "prefix_len", prefix_len, groups)
    _check_ints(where, "group_start", group_start, groups + 1)
    if groups > MAX_GROUPS:
        _bad(where, f"{groups} groups, at most {MAX_GROUPS} are served")
    _check_table(where, "prefix_table", prefix_table, groups, bs, max_prefix, "max_prefix")
    _check_table(where, "block_table", block_table, S, bs, max_ctx, "max_ctx")
    if q_len < 1 or q_len > 1 << 16:
        _bad(where, "q_len is from 1 to 65536")
    T = S * q_len
    if q.dtype != torch.bfloat16 or q.dim() != 3 or q.shape[0] != T or q.shape[2] != D or not q.is_contiguous():
        _bad(where, f"q is contiguous bf16 [{T}, heads, {D}]")
    Hq = q.shape[1]
    if Hq == 0 or Hq % Hkv != 0 or Hq // Hkv > MAX_GROUP:
        _bad(where, f"{Hq} query heads over {Hkv} kv heads: whole groups of up to {MAX_GROUP}")
    if T * Hq * D > 1 << 29:
        _bad(where, f"{T} tokens of {Hq} heads of {D} dims are more than 2^29 elements: a step of a batch is meant, not its prompts")
    _check_scale(where, scale)
    fp8 = dtype == torch.uint8
    if fp8:
        if D == 64 and bs % 2:
            _bad(where, f"an e4m3 cache of head dim 64 has blocks of an even number of tokens, not {bs}")
        for x in (k_scale, v_scale):
            if x is None or x.dtype != torch.float32 or x.numel() != 1:
                _bad(where, "an e4m3 cache comes with fp32 scales of one element")
    else:
        k_scale = v_scale = None
    _check_places(where, q, k_cache, v_cache, prefix_table, prefix_len, group_start, block_table, ctx_len, k_scale, v_scale)
    if not q.is_cuda:
        _check_values(where, nb, bs, max_prefix, max_ctx, prefix_table, prefix_len, group_start, block_table, ctx_len)
        out, lse = ref.shared_prefix_attention(q, k_cache, v_cache, prefix_table, prefix_len, group_start, block_table, ctx_len, q_len, scale, k_scale, v_scale)
        return (out, lse) if return_lse else out
    qp, kp, vp = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    if (qp | kp | vp) & 15:
        _bad(where, "q and the caches begin on 16 bytes")
    if nb * bs >= 1 << 31:
        _bad(where, f"a cache of {nb} blocks of {bs} has 2^31 rows or more")
    out = torch.empty_like(q)
    lse = torch.empty(T, Hq, dtype=torch.float32, device=q.device) if return_lse else None
    if T == 0:
        return (out, lse) if return_lse else out
    rt = runtime(q.device)
    need = _workspace("mb_shared_attn_ws", S, q_len, groups, Hq, Hkv, D, max_prefix, max_ctx, rt.sm_count)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    a = _SHARED_ARGS.pack(qp, kp, vp, prefix_table.data_ptr(), prefix_table.stride(0), prefix_len.data_ptr(), group_start.data_ptr(), block_table.data_ptr(),
                          block_table.stride(0), ctx_len.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), ws.data_ptr(), need, k_scale.data_ptr() if fp8 else 0,
                          v_scale.data_ptr() if fp8 else 0, rt.status.data_ptr(), nb, S, q_len, groups, Hq, Hkv, D, bs, int(fp8), max_prefix, max_ctx, rt.sm_count, scale)
    _native.check(_library().mb_shared_attn(a, _stream()), "shared_attn")
    _count(1 + (groups > 0 and max_prefix > 0) + (max_ctx > 0))          # the join, prefixes, own rows; further steps, which go by the sizes, are not counted
    return (out, lse) if return_lse else out


def _check_values(where, nb, bs, max_prefix, max_ctx, prefix_table, prefix_len, group_start, block_table, ctx_len) -> None:
    """CPU: what the kernels cut and report is refused."""
    S = ctx_len.shape[0]
    if prefix_len.shape[0] and (bool((group_start.diff() < 0).any()) or int(group_start[0]) < 0 or int(group_start[-1]) > S):
        _bad(where, f"group_start falls, or leaves the batch of {S}")
    held = group_start.diff() > 0
    if bool((ctx_len > max_ctx).any()) or bool((held & (prefix_len > max_prefix)).any()):
        _bad(where, f"a length is beyond max_prefix {max_prefix} or max_ctx {max_ctx}")
    for table, rows in ((prefix_table, torch.where(held, prefix_len, 0)), (block_table, ctx_len)):
        used = torch.arange(table.shape[1]) * bs < rows[:, None]
        if bool((used & ((table < 0) | (table >= nb))).any()):
            _bad(where, f"a table has a block that the cache of {nb} does not have")


def merge_attention(outs: Sequence[torch.Tensor], lses: Sequence[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of the same queries over disjoint sets of keys, as one: outs[i] [rows, heads, dim] (all bf16 or all fp32) with the log-sum-exps lses[i] fp32
    [rows, heads] -> (out of that type, lse). A part with lse -inf has no weight and its values are not looked at; a row without any weight gives zeros
    and -inf; one that has a part with +inf or NaN gives NaN. From 1 to 16 parts. Outputs are new tensors."""
    where = "merge_attention"
    n = len(outs)
    if n == 0 or n > MAX_PARTS or len(lses) != n:
        _bad(where, f"{n} outputs and {len(lses)} log-sum-exps: as many of each, from 1 to {MAX_PARTS}")
    shape, dtype = outs[0].shape, outs[0].dtype
    if len(shape) != 3 or (dtype != torch.bfloat16 and dtype != torch.float32):
        _bad(where, "outputs are [rows, heads, dim], bf16 or fp32")
    for o, l in zip(outs, lses):
        if o.shape != shape or o.dtype != dtype or not o.is_contiguous():
            _bad(where, "outputs are contiguous and have one shape and type")
        if l.dtype != torch.float32 or l.shape != shape[:2] or not l.is_contiguous():
            _bad(where, f"log-sum-exps are contiguous fp32 {list(shape[:2])}")
    if shape[2] > 1 << 20:
        _bad(where, "dim is at most 2^20")
    _check_places(where, *outs, *lses)
    if not outs[0].is_cuda:
        return ref.merge_attention(outs, lses)
    out, lse = torch.empty_like(outs[0]), torch.empty_like(lses[0])
    rows = shape[0] * shape[1]
    if rows == 0 or shape[2] == 0:
        return (out, lse) if rows == 0 else (out, ref.merged_lse(torch.stack(list(lses))))
    pad = [0] * (MAX_PARTS - n)
    a = _MERGE_ARGS.pack(*[o.data_ptr() for o in outs], *pad, *[l.data_ptr() for l in lses], *pad, out.data_ptr(), lse.data_ptr(), rows, n, shape[2],
                         int(dtype == torch.float32), runtime(out.device).sm_count)
    _native.check(_library().mb_merge_attn(a, _stream()), "merge_attn")
    _count()
    return out, lse
