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
import functools
import importlib.util
import math
import sysconfig
import warnings
from typing import NamedTuple

import torch

from . import _lib
from .ops import _DTYPES

_E4M3 = torch.float8_e4m3fn
_INT32 = torch.int32
_HEAD_DIMS = (64, 128, 256)
_BLOCK_SIZES = (16, 32, 64, 128)
_INT_MAX = 2 ** 31 - 1

# A decode step's kernels are short, so the host's share counts. Well-formed calls go through the
# native module _calls, which checks, allocates and calls the library in one step; it returns
# None for anything else, and then the Python here copies what can be copied, raises what has
# to be raised, and makes the same call. It asks each tensor for a property once, too.
_calls = None


def _import_calls():
    """The native module, or False where it was not built. One that was built for another torch or
    Python knows their objects by another layout: False too, with a warning."""
    if importlib.util.find_spec("._calls", __package__) is None:
        return False
    here = f"torch {torch.__version__} {sysconfig.get_config_var('SOABI')}"
    try:
        from . import _calls as module
        built_for = getattr(module, "built_for", "an unknown version")
    except ImportError as e:
        built_for = f"another version ({e})"
    if built_for == here:
        return module
    warnings.warn(f"apex_attn._calls was built for {built_for} and is left out with {here}: build it again")
    return False


def _load_calls():
    """The native module with the library's addresses set, or False."""
    global _calls
    lib = _lib.load()
    module = _import_calls()
    if module:
        module.init(*(ctypes.cast(getattr(lib, "apex_attn_" + name), ctypes.c_void_p).value for name in (
            "kv_plan", "kv_release", "kv_append", "fwd_paged_workspace_bytes", "fwd_paged")))
    _calls = module
    return module


try:
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:  # a build of torch without CUDA, or one that names it otherwise
    def _raw_stream(device):
        return torch.cuda.current_stream(device).cuda_stream


class KVCachePlan(NamedTuple):
    """What kv_cache_plan returns; see there."""
    slots: torch.Tensor
    cu_seqlens: torch.Tensor
    seq_lens: torch.Tensor
    free_count: torch.Tensor
    placed: torch.Tensor


def _int32(t, name, numel, device):
    """The address of a contiguous int32 vector."""
    if t.dtype is not _INT32 or t.shape != (numel,) or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {numel} values on the CUDA device {device}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _table(block_table):
    """(batch, width, row stride) of a block table."""
    if block_table.dtype is not _INT32 or block_table.dim() != 2:
        raise ValueError(f"block_table must be int32 [batch, width], got {block_table.dtype} "
                         f"{tuple(block_table.shape)}")
    batch, width = block_table.shape
    row, unit = block_table.stride()
    if width > 1 and unit != 1 or batch > 1 and row < width:
        raise ValueError("block_table needs unit stride along its rows, and rows that do not overlap")
    return batch, width, row if batch > 1 else width


def _bookkeeping(call, name, block_table, seq_lens, new_lens, finished, free_blocks, free_count, block_size,
                 slots, cu_at, lens_at, count_at, placed_at, max_new):
    """Checks what plan and release share and runs `call`, writing to the given addresses."""
    device = block_table.get_device()
    if device < 0:
        raise ValueError("block_table must be a CUDA tensor")
    batch, width, stride = _table(block_table)
    if batch == 0 or width == 0:
        raise ValueError(f"block_table has no entries: {tuple(block_table.shape)}")
    if block_size not in _BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {_BLOCK_SIZES}, got {block_size}")
    capacity = free_blocks.numel()
    args = _lib.KV_PLAN_ARGS.pack(
        block_table.data_ptr(), _int32(seq_lens, "seq_lens", batch, device),
        0 if new_lens is None else _int32(new_lens, "new_lens", batch, device),
        0 if finished is None else _int32(finished, "finished", batch, device),
        _int32(free_blocks, "free_blocks", capacity, device), _int32(free_count, "free_count", 1, device), slots,
        cu_at, lens_at, count_at, placed_at, stride, batch, width, capacity, block_size, max_new, device + 1)
    rc = call(args, _raw_stream(device))
    if rc:
        _lib.check(rc, name)


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
    calls = _load_calls() if _calls is None else _calls
    if calls:
        done = calls.plan(block_table, seq_lens, new_lens, free_blocks, free_count, block_size, max_new_tokens)
        if done is not None:
            return KVCachePlan._make(done)
    if not 1 <= max_new_tokens <= 2 ** 30:
        raise ValueError(f"max_new_tokens must lie in [1, 2^30], got {max_new_tokens}")
    batch = seq_lens.numel()
    where = block_table.device
    slots = torch.empty(max_new_tokens, dtype=torch.int64, device=where)
    out = torch.empty(3 * batch + 2, dtype=_INT32, device=where)
    at = out.data_ptr()
    _bookkeeping(_lib.load().apex_attn_kv_plan, "kv_cache_plan", block_table, seq_lens, new_lens, None, free_blocks,
                 free_count, block_size, slots.data_ptr(), at, at + 4 * batch + 4, at + 12 * batch + 4,
                 at + 8 * batch + 4, max_new_tokens)
    cu, lens, placed, count = out.split_with_sizes((batch + 1, batch, batch, 1))
    return KVCachePlan(slots, cu, lens, count, placed)


def kv_cache_release(block_table, seq_lens, finished, free_blocks, free_count,
                     block_size) -> tuple[torch.Tensor, torch.Tensor]:
    """Pushes the blocks of the requests with a non-zero entry in ``finished`` (int32
    ``[batch]``) back on the stack ``free_blocks`` (behind its first ``free_count`` entries, in
    request order). Returns the lengths (0 for those requests) and the count after it, as
    new tensors; the table rows stay as they are. Arguments as for kv_cache_plan."""
    calls = _load_calls() if _calls is None else _calls
    if calls:
        done = calls.release(block_table, seq_lens, finished, free_blocks, free_count, block_size)
        if done is not None:
            return done
    lens, count = torch.empty_like(seq_lens), torch.empty_like(free_count)
    _bookkeeping(_lib.load().apex_attn_kv_release, "kv_cache_release", block_table, seq_lens, None, finished,
                 free_blocks, free_count, block_size, 0, 0, lens.data_ptr(), count.data_ptr(), 0, 0)
    return lens, count


def _cache(k_cache, v_cache, k_scale, v_scale, device):
    """Checks the cache; returns its shape, the four addresses, and the (block, head, token) byte
    strides of K, then V."""
    shape = k_cache.shape
    if len(shape) != 4 or shape != v_cache.shape:
        raise ValueError(f"k_cache and v_cache must be [num_blocks, H_kv, block_size, D] alike, got "
                         f"{tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    if k_cache.dtype is not _E4M3 or v_cache.dtype is not _E4M3:
        raise TypeError(f"k_cache and v_cache must be float8_e4m3fn, got {k_cache.dtype}, {v_cache.dtype}")
    blocks, heads, block_size, headdim = shape
    if headdim not in _HEAD_DIMS:
        raise KeyError(headdim)
    if block_size not in _BLOCK_SIZES:
        raise ValueError(f"block_size must be one of {_BLOCK_SIZES}, got {block_size}")
    if blocks == 0 or heads == 0:
        raise ValueError("the cache has no blocks or no heads")
    k_at, v_at = k_cache.data_ptr(), v_cache.data_ptr()
    strides = []
    for c, ptr in ((k_cache, k_at), (v_cache, v_at)):
        sb, sh, st, sd = c.stride()
        if heads == 1:
            sh = block_size * headdim
        if blocks == 1:
            sb = heads * block_size * headdim
        # The cache is written and kept by its owner, so a layout that the kernels cannot
        # take is refused instead of copied.
        if sd != 1 or st < headdim or (sb | sh | st | ptr) & 15 or c.get_device() != device:
            raise ValueError("k_cache and v_cache need unit stride along D, other strides multiples of 16, 16-byte "
                             f"aligned storage, and the CUDA device {device}")
        strides += (sb, sh, st)
    for s in (k_scale, v_scale):
        if s.dtype is not torch.float32 or s.shape != (blocks, heads) or not s.is_contiguous() \
                or s.get_device() != device:
            raise ValueError(f"k_scale and v_scale must be contiguous float32 {(blocks, heads)} on the CUDA device "
                             f"{device}, got {s.dtype} {tuple(s.shape)} on {s.device}")
    return shape, (k_at, v_at, k_scale.data_ptr(), v_scale.data_ptr()), strides


def _rows(t):
    """[rows, H, D] as the kernels read it (unit stride along D, others multiples of 8), copied if
    need be, with its token and head strides."""
    st, sh, sd = t.stride()
    if sd != 1 or (st | sh) & 7 or sh < t.shape[2] or t.data_ptr() & 15:
        t = t.contiguous()
        st, sh, sd = t.stride()
    return t, st, sh


def _distinct_rows(t, st, sh):
    """Whether the (token, head) rows of an output do not overlap."""
    total, heads, headdim = t.shape
    return (total <= 1 or st >= headdim) and (heads <= 1 or sh >= headdim) and (
        total <= 1 or heads <= 1 or st >= (heads - 1) * sh + headdim or sh >= (total - 1) * st + headdim)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(nheads, kv_heads, max_seqlen_q, headdim):
    return _lib.load().apex_attn_fwd_paged_workspace_bytes(nheads, kv_heads, max_seqlen_q, headdim)


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
    calls = _load_calls() if _calls is None else _calls
    if calls and calls.append(k, v, k_cache, v_cache, k_scale, v_scale, slots) is not None:
        return
    shape = k.shape
    if len(shape) != 3 or shape != v.shape:
        raise ValueError(f"k and v must be [total, H_kv, D] alike, got {tuple(k.shape)}, {tuple(v.shape)}")
    total, heads, headdim = shape
    dtype = _DTYPES.get(k.dtype)
    if dtype is None or v.dtype is not k.dtype:
        raise TypeError(f"k and v must both be float16 or bfloat16, got {k.dtype}, {v.dtype}")
    device = k.get_device()
    if device < 0 or v.get_device() != device:
        raise ValueError("k and v must be CUDA tensors on one device")
    (blocks, cache_heads, block_size, cache_dim), at, cache_strides = _cache(k_cache, v_cache, k_scale, v_scale, device)
    if cache_heads != heads or cache_dim != headdim:
        raise ValueError(f"k {tuple(shape)} does not match the cache {tuple(k_cache.shape)}")
    if slots.dtype is not torch.int64 or slots.dim() != 1 or slots.numel() < total or slots.get_device() != device \
            or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int64 tensor of at least {total} values on the CUDA device {device}")
    if total == 0:
        return
    k, k_st, k_sh = _rows(k)
    v, v_st, v_sh = _rows(v)
    args = _lib.KV_APPEND_ARGS.pack(k.data_ptr(), v.data_ptr(), *at, slots.data_ptr(), total, heads, headdim, dtype,
                                    blocks, block_size, k_st, k_sh, v_st, v_sh, *cache_strides, device + 1)
    rc = _lib.load().apex_attn_kv_append(args, _raw_stream(device))
    if rc:
        _lib.check(rc, "kv_cache_append")


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
    ``return_lse``, the fp32 natural logsumexp ``[H, total_q]`` (0 outside every request). A row that
    sees nothing gives 0 and -inf. ``out``: a tensor like q to write o into, whose rows do not
    overlap; those outside every request keep what they hold.

    Precision: scores, maxima and sums are fp32. A softmax weight (times its block's V scale) is held
    to 2^-11 of itself, or to 2^-30 of the row's largest; a value of q exactly, or to 2^-17 (bf16) or
    2^-24 (fp16) of its row's largest. Long sums of one sign come out low, by 2.6e-4 for 131072 tokens.

    Scales are not negative; V scales below 2^-100 count as 2^-100. A code or scale of NaN, or an
    infinite or NaN value of q, makes the rows that see it NaN and no others. Table entries
    outside the cache read as blocks of zeros.

    Head dims 64, 128, 256 (others: KeyError). Asynchronous on the current CUDA stream."""
    calls = _load_calls() if _calls is None else _calls
    if calls:
        done = calls.attend(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_seqlens_q, max_seqlen_q,
                            causal, sm_scale, return_lse, window_left, out)
        if done is not None:
            return done
    shape = q.shape
    if len(shape) != 3:
        raise ValueError(f"q must be [total_q, H, D], got {tuple(shape)}")
    total, nheads, headdim = shape
    dtype = _DTYPES.get(q.dtype)
    if dtype is None:
        raise TypeError(f"q must be float16 or bfloat16, got {q.dtype}")
    device = q.get_device()
    if device < 0:
        raise ValueError("q must be a CUDA tensor")
    (blocks, kv_heads, block_size, cache_dim), at, cache_strides = _cache(k_cache, v_cache, k_scale, v_scale, device)
    if cache_dim != headdim or nheads == 0 or nheads % kv_heads != 0:
        raise ValueError(f"q {tuple(shape)} does not match the cache {tuple(k_cache.shape)}: D alike, and H_kv "
                         "dividing q's heads")
    batch, width, table_stride = _table(block_table)
    if block_table.get_device() != device:
        raise ValueError("all tensors must be CUDA tensors on one device")
    if batch == 0 or width == 0:
        raise ValueError(f"block_table has no entries: {tuple(block_table.shape)}")
    lens_at = _int32(seq_lens, "seq_lens", batch, device)
    cu_at = 0
    if cu_seqlens_q is not None:
        cu_at = _int32(cu_seqlens_q, "cu_seqlens_q", batch + 1, device)
        if max_seqlen_q is None or max_seqlen_q < 1:
            raise ValueError("cu_seqlens_q needs a positive max_seqlen_q")
        max_seqlen_q = min(max_seqlen_q, max(total, 1))
    elif total % batch != 0 or (max_seqlen_q is not None and max_seqlen_q * batch != total):
        raise ValueError(f"without cu_seqlens_q, q's {total} rows must be max_seqlen_q for each of {batch} requests")
    else:
        max_seqlen_q = total // batch
    if window_left is not None and (window_left < 0 or not causal):
        raise ValueError("window_left must be >= 0 and needs causal=True")
    where = q.device
    if out is None:
        o = torch.empty_like(q) if q.is_contiguous() else torch.empty(shape, dtype=q.dtype, device=where)
        o_st, o_sh = nheads * headdim, headdim
    else:
        o, o_st, o_sh = _rows(out)
        if o is not out or o.shape != shape or o.dtype is not q.dtype or o.get_device() != device \
                or not _distinct_rows(o, o_st, o_sh):
            raise ValueError("out must be like q, with unit stride along D, other strides multiples of 8, and rows "
                             "that do not overlap")
    lse = None
    if return_lse:  # the kernel clears the rows outside every request unless `out` keeps its own
        new = torch.empty if out is None or cu_seqlens_q is None else torch.zeros
        lse = new(nheads, total, dtype=torch.float32, device=where)
    if total == 0:
        return (o, lse) if return_lse else o
    q, q_st, q_sh = _rows(q)
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(headdim)
    ws_bytes = _workspace_bytes(nheads, kv_heads, max_seqlen_q, headdim)
    workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=where)
    args = _lib.PAGED_ARGS.pack(
        q.data_ptr(), *at, block_table.data_ptr(), lens_at, cu_at, o.data_ptr(), 0 if lse is None else lse.data_ptr(),
        table_stride, q_st, q_sh, o_st, o_sh, *cache_strides, batch, nheads, kv_heads, total, max_seqlen_q, headdim,
        dtype, blocks, block_size, width, 1 if causal else 0, -1 if window_left is None else min(window_left, _INT_MAX),
        1 if out is None else 0, sm_scale, device + 1)
    rc = _lib.load().apex_attn_fwd_paged(args, workspace.data_ptr(), ws_bytes, _raw_stream(device))
    if rc:
        _lib.check(rc, "custom_attention_paged_forward")
    return (o, lse) if return_lse else o
