"""A paged K/V cache held in 8 bits, and attention over it: what a serving program runs each
step. The reference has no counterpart.

The cache is a pool of blocks of 16, 32, 64 or 128 tokens: ``k_cache`` and ``v_cache`` are
float8_e4m3fn ``[num_blocks, H_kv, block_size, D]`` (``[num_blocks, block_size, H_kv, D]``
storage goes in as ``.transpose(1, 2)``, without a copy), ``k_scale`` and ``v_scale`` float32
``[num_blocks, H_kv]``; a value is code * scale. ``block_table`` int32 ``[batch, width]`` names
each request's blocks in order; the token at position t sits in slot
``block_table[b, t // block_size] * block_size + t % block_size``.

A step is

    lens, free_count = kv_cache_release(block_table, lens, finished, free_blocks, free_count, block_size)
    plan = kv_cache_plan(block_table, lens, new_lens, free_blocks, free_count, block_size, max_new_tokens)
    for each layer:
        kv_cache_append(k, v, k_cache, v_cache, k_scale, v_scale, plan.slots)
        o = custom_attention_paged_forward(q, k_cache, v_cache, k_scale, v_scale, block_table,
                                           plan.seq_lens, plan.cu_seqlens, max_seqlen_q)

No call reads a length on the host or synchronises. Errors are as for the other operators:
ValueError / TypeError / KeyError (head dim) for arguments, RuntimeError with the library's
status text otherwise.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from . import _lib
from .ops import _DTYPES

_E4M3 = torch.float8_e4m3fn
_HEAD_DIMS = (64, 128, 256)
_BLOCK_SIZES = (16, 32, 64, 128)


class KVCachePlan(NamedTuple):
    """What kv_cache_plan returns; see there."""
    slots: torch.Tensor
    cu_seqlens: torch.Tensor
    seq_lens: torch.Tensor
    free_count: torch.Tensor
    placed: torch.Tensor


def _int32(t, name, numel, device):
    if t.dtype != torch.int32 or t.dim() != 1 or t.numel() != numel or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {numel} values on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")


def _table(block_table):
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1:
        raise ValueError(f"block_table must be int32 [batch, width] with unit stride along a row, got "
                         f"{block_table.dtype} {tuple(block_table.shape)}")
    if not block_table.is_cuda:
        raise ValueError("block_table must be a CUDA tensor")
    batch, width = block_table.shape
    return batch, width, max(block_table.stride(0), width) if batch > 1 else width


def _bookkeeping(block_table, seq_lens, free_blocks, free_count, block_size):
    batch, width, stride = _table(block_table)
    device = block_table.device
    _int32(seq_lens, "seq_lens", batch, device)
    _int32(free_count, "free_count", 1, device)
    _int32(free_blocks, "free_blocks", free_blocks.numel(), device)
    if block_size not in _BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {_BLOCK_SIZES}, got {block_size}")
    out = torch.empty(batch + 1, dtype=torch.int32, device=device)  # lengths, then the count
    args = _lib.KVPlanArgs(block_table=block_table.data_ptr(), seq_lens=seq_lens.data_ptr(),
                           free_blocks=free_blocks.data_ptr(), free_count=free_count.data_ptr(),
                           seq_lens_out=out.data_ptr(), free_count_out=out.data_ptr() + 4 * batch,
                           table_stride=stride, batch=batch, table_width=width,
                           free_capacity=free_blocks.numel(), block_size=block_size)
    return args, out, batch, device


def kv_cache_plan(block_table, seq_lens, new_lens, free_blocks, free_count, block_size,
                  max_new_tokens) -> KVCachePlan:
    """Places the new tokens of a step: request b holds ``seq_lens[b]`` tokens and brings
    ``new_lens[b]`` more (int32 ``[batch]``). Blocks come off the top of the stack
    ``free_blocks[: free_count]`` (int32; ``free_count`` an int32 tensor of one value) in
    request order, and their ids are written into ``block_table`` behind the ones that the
    request holds. Returns

    * ``slots`` int64 ``[max_new_tokens]``: the slot of each new token, requests one after
      another, -1 past the last (``max_new_tokens``: an upper bound that the host knows);
    * ``cu_seqlens`` int32 ``[batch + 1]``: where each request's new tokens begin;
    * ``seq_lens`` and ``free_count``: their values after the step (new tensors; the inputs
      and ``free_blocks`` keep theirs);
    * ``placed`` int32 ``[batch]``: 0 for a request that the stack, the table row or the slot
      array had no room for. It takes no block, keeps its length, and its slots are -1.

    At most 8192 requests. Asynchronous on the current CUDA stream of the table's device."""
    args, out, batch, device = _bookkeeping(block_table, seq_lens, free_blocks, free_count, block_size)
    _int32(new_lens, "new_lens", batch, device)
    if max_new_tokens < 1:
        raise ValueError("max_new_tokens must be positive")
    slots = torch.empty(max_new_tokens, dtype=torch.int64, device=device)
    more = torch.empty(2 * batch + 1, dtype=torch.int32, device=device)
    args.new_lens = new_lens.data_ptr()
    args.slots = slots.data_ptr()
    args.cu_seqlens = more.data_ptr()
    args.placed = more.data_ptr() + 4 * (batch + 1)
    args.max_new_tokens = max_new_tokens
    stream = torch.cuda.current_stream(device).cuda_stream
    _lib.check(_lib.load().apex_attn_kv_plan(ctypes.byref(args), stream), "kv_cache_plan")
    return KVCachePlan(slots, more[:batch + 1], out[:batch], out[batch:], more[batch + 1:])


def kv_cache_release(block_table, seq_lens, finished, free_blocks, free_count,
                     block_size) -> tuple[torch.Tensor, torch.Tensor]:
    """Pushes the blocks of the requests with a non-zero entry in ``finished`` (int32
    ``[batch]``) back on the stack ``free_blocks`` (behind its first ``free_count`` entries, in
    request order). Returns the lengths (0 for those requests) and the count after it, as
    new tensors; the table rows stay as they are. Arguments as for kv_cache_plan."""
    args, out, batch, device = _bookkeeping(block_table, seq_lens, free_blocks, free_count, block_size)
    _int32(finished, "finished", batch, device)
    args.finished = finished.data_ptr()
    stream = torch.cuda.current_stream(device).cuda_stream
    _lib.check(_lib.load().apex_attn_kv_release(ctypes.byref(args), stream), "kv_cache_release")
    return out[:batch], out[batch:]


def _cache(k_cache, v_cache, k_scale, v_scale, device):
    """Checks the cache and returns its (block, head, token) byte strides, K's then V's."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError(f"k_cache and v_cache must be [num_blocks, H_kv, block_size, D] alike, got "
                         f"{tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    if k_cache.dtype != _E4M3 or v_cache.dtype != _E4M3:
        raise TypeError(f"k_cache and v_cache must be float8_e4m3fn, got {k_cache.dtype}, {v_cache.dtype}")
    blocks, heads, block_size, headdim = k_cache.shape
    if headdim not in _HEAD_DIMS:
        raise KeyError(headdim)
    if block_size not in _BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {_BLOCK_SIZES}, got {block_size}")
    for s in (k_scale, v_scale):
        if s.dtype != torch.float32 or s.shape != (blocks, heads) or not s.is_contiguous() or s.device != device:
            raise ValueError(f"k_scale and v_scale must be contiguous float32 {(blocks, heads)} on {device}, got "
                             f"{s.dtype} {tuple(s.shape)} on {s.device}")
    if blocks == 0 or heads == 0:
        raise ValueError("the cache has no blocks or no heads")
    strides = []
    for c in (k_cache, v_cache):
        sb, sh, st, sd = c.stride()
        sh = sh if heads > 1 else block_size * headdim
        sb = sb if blocks > 1 else heads * block_size * headdim
        # The cache is written and kept by its owner, so a layout that the kernels cannot
        # take is refused instead of copied.
        if sd != 1 or st < headdim or (sb | sh | st | c.data_ptr()) & 15 or c.device != device:
            raise ValueError("k_cache and v_cache need unit stride along D, other strides multiples of 16, 16-byte "
                             f"aligned storage, and the device {device}")
        strides += (sb, sh, st)
    return strides


def _rows(t, name):
    """[rows, H, D] as the kernels read it: unit stride along D, others multiples of 8."""
    st, sh, sd = t.stride()
    if sd != 1 or (st | sh) & 7 or sh < t.shape[2] or t.data_ptr() & 15:
        return t.contiguous()
    return t


def kv_cache_append(k, v, k_cache, v_cache, k_scale, v_scale, slots) -> None:
    """Quantises new tokens ``k``, ``v`` ``[total, H_kv, D]`` (bf16 or fp16) into the cache, in
    place: token t goes to slot ``slots[t]`` (int64 ``[total]``, as kv_cache_plan gives them;
    slots outside the cache, -1 among them, are skipped).

    Tokens with consecutive slots inside one block form a run; its scale (per head) is the
    smallest power of two, at least 2^-100, that holds the run's largest magnitude in e4m3. A
    run that starts inside a block keeps the tokens before it: the scale is at least the
    block's old one, and where it grows their codes are divided by the growth. Values that are
    not finite are stored as NaN and leave the scale alone. In one call at most one run may go
    to a block, and a block must belong to one request. ``slots`` may be longer than ``k``
    (then its first ``total`` entries count)."""
    if k.dim() != 3 or k.shape != v.shape:
        raise ValueError(f"k and v must be [total, H_kv, D] alike, got {tuple(k.shape)}, {tuple(v.shape)}")
    total, heads, headdim = k.shape
    device = k.device
    if k.dtype not in _DTYPES or v.dtype != k.dtype:
        raise TypeError(f"k and v must both be float16 or bfloat16, got {k.dtype}, {v.dtype}")
    if not k.is_cuda or v.device != device:
        raise ValueError("k and v must be CUDA tensors on one device")
    cache_strides = _cache(k_cache, v_cache, k_scale, v_scale, device)
    blocks, cache_heads, block_size, cache_dim = k_cache.shape
    if (cache_heads, cache_dim) != (heads, headdim):
        raise ValueError(f"k {tuple(k.shape)} does not match the cache {tuple(k_cache.shape)}")
    if slots.dtype != torch.int64 or slots.dim() != 1 or slots.numel() < total or slots.device != device \
            or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int64 tensor of at least {total} values on {device}")
    if total == 0:
        return
    k, v = _rows(k, "k"), _rows(v, "v")
    args = _lib.KVAppendArgs(k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                             k_scale.data_ptr(), v_scale.data_ptr(), slots.data_ptr(), total, heads, headdim,
                             _DTYPES[k.dtype], blocks, block_size,
                             (k.stride(0), k.stride(1), v.stride(0), v.stride(1), *cache_strides))
    stream = torch.cuda.current_stream(device).cuda_stream
    _lib.check(_lib.load().apex_attn_kv_append(ctypes.byref(args), stream), "kv_cache_append")


def custom_attention_paged_forward(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens,
                                   cu_seqlens_q=None, max_seqlen_q=None, causal=True, sm_scale=None,
                                   return_lse=False, window_left=None, out=None):
    """Attention of new query tokens over the cached tokens of their requests.

    ``q`` is ``[total_q, H, D]`` (bf16 or fp16; H a multiple of the cache's heads), requests one
    after another at the offsets ``cu_seqlens_q`` (int32 ``[batch + 1]``) with at most
    ``max_seqlen_q`` tokens each; without offsets every request has ``total_q / batch`` (one
    for a decode step). ``seq_lens`` int32 ``[batch]`` counts each request's cached tokens, the
    query tokens' own among them: append first. Causal (default): query token i of n sees the
    positions up to ``seq_len - n + i``, from ``window_left`` before it on if a window is given;
    otherwise all. Returns o like q (rows outside every request are zeros) and, with
    ``return_lse``, the fp32 natural logsumexp ``[H, total_q]``. A row that sees nothing gives 0
    and -inf. ``out``: a tensor like q to write o into; its rows outside every request keep what
    they hold.

    Head dims 64, 128, 256 (others: KeyError). Asynchronous on the current CUDA stream."""
    if q.dim() != 3:
        raise ValueError(f"q must be [total_q, H, D], got {tuple(q.shape)}")
    total, nheads, headdim = q.shape
    device = q.device
    if q.dtype not in _DTYPES:
        raise TypeError(f"q must be float16 or bfloat16, got {q.dtype}")
    if not q.is_cuda:
        raise ValueError("q must be a CUDA tensor")
    cache_strides = _cache(k_cache, v_cache, k_scale, v_scale, device)
    blocks, kv_heads, block_size, cache_dim = k_cache.shape
    if cache_dim != headdim or nheads == 0 or nheads % kv_heads != 0:
        raise ValueError(f"q {tuple(q.shape)} does not match the cache {tuple(k_cache.shape)}: D alike, and H_kv "
                         "dividing q's heads")
    batch, width, table_stride = _table(block_table)
    if block_table.device != device:
        raise ValueError("all tensors must be CUDA tensors on one device")
    _int32(seq_lens, "seq_lens", batch, device)
    if cu_seqlens_q is not None:
        _int32(cu_seqlens_q, "cu_seqlens_q", batch + 1, device)
        if max_seqlen_q is None or max_seqlen_q < 1:
            raise ValueError("cu_seqlens_q needs a positive max_seqlen_q")
    elif batch == 0 or total % batch != 0 or (max_seqlen_q is not None and max_seqlen_q * batch != total):
        raise ValueError(f"without cu_seqlens_q, q's {total} rows must be max_seqlen_q for each of {batch} requests")
    else:
        max_seqlen_q = total // batch
    if window_left is not None and (window_left < 0 or not causal):
        raise ValueError("window_left must be >= 0 and needs causal=True")
    if out is None:
        o = torch.empty(q.shape, dtype=q.dtype, device=device)
    else:
        o = out
        if o.shape != q.shape or o.dtype != q.dtype or o.device != device or _rows(o, "out") is not o:
            raise ValueError("out must be like q, with unit stride along D and other strides multiples of 8")
    lse = torch.empty((nheads, total), dtype=torch.float32, device=device) if return_lse else None
    if total == 0 or batch == 0 or width == 0:
        if out is None:
            o.zero_()
        return (o, lse.zero_()) if return_lse else o
    q = _rows(q, "q")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(headdim)
    lib = _lib.load()
    ws_bytes = lib.apex_attn_fwd_paged_workspace_bytes(nheads, kv_heads, max_seqlen_q, headdim)
    workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    args = _lib.PagedArgs(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
                          v_scale.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
                          None if cu_seqlens_q is None else cu_seqlens_q.data_ptr(), o.data_ptr(),
                          None if lse is None else lse.data_ptr(), table_stride,
                          (q.stride(0), q.stride(1), o.stride(0), o.stride(1), *cache_strides), batch, nheads,
                          kv_heads, total, max_seqlen_q, headdim, _DTYPES[q.dtype], blocks, block_size, width,
                          1 if causal else 0, -1 if window_left is None else window_left, 1 if out is None else 0,
                          sm_scale)
    stream = torch.cuda.current_stream(device).cuda_stream
    rc = lib.apex_attn_fwd_paged(ctypes.byref(args), workspace.data_ptr(), ws_bytes, stream)
    _lib.check(rc, "custom_attention_paged_forward")
    return (o, lse) if return_lse else o
