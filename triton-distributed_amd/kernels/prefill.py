"""Attention of many query rows: whole prompts, chunks of prompts, drafted tokens, and decode steps of sequences that
share a prefix.

``gqa_fwd_batch_prefill`` is what the reference's attention block does for more than one new token
(``python/triton_dist/layers/amd/tp_attn.py:262-269``), over packed keys or over the paged cache that
``rope_kv_append`` writes and ``gqa_fwd_batch_decode`` reads.  ``gqa_fwd_batch_decode_shared_prefix`` is
``gqa_fwd_batch_decode`` for sequences that have long prefixes in common: a prefix is read once for all of them.

Every function enqueues hand-written HIP kernels through the C ABI in ``include/flash_decode.h`` (``fd_prefill``,
``fd_decode_shared``); nothing synchronises with the host, lengths are never read on it, and there is no CPU path.  Forward
only: a query, key, value or fp8 scale that requires a gradient is refused while autograd records, one with a forward-mode
tangent always.

``stream=`` enqueues a call's kernels there instead of on the current stream.  The caller orders it behind what the arguments
need and what uses the result behind it, and keeps the arguments alive; what the call allocates needs no ordering.
"""
from __future__ import annotations

from ctypes import byref
from typing import Optional

import torch
from torch.autograd import forward_ad

from .._lib import (FD_COMBINE_SPLIT, FdParams, FdPrefillArgs, FdSharedArgs, check, fd_dtype_of, load_library,
                    stream_handle)
from .flash_decode import _on, _require_cuda


def _need(condition, message):
    if not condition:
        raise RuntimeError(message)


def _check_devices(name, first, *tensors):
    """All tensors on one GPU."""
    _require_cuda(first, *tensors)
    for t in tensors:
        _need(t is None or t.device == first.device, f"{name}: tensors on {first.device} and {t.device if t is not None else ''}")


def _check_int32(name, what, t, shape):
    _need(t.dtype == torch.int32 and tuple(t.shape) == shape and t.is_contiguous(),
          f"{name}: {what} must be a contiguous int32 tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")


def _check_scales(name, k_scale, v_scale, kv_heads):
    _need((k_scale is None) == (v_scale is None), f"{name}: k_scale and v_scale must be given together")
    for s in (k_scale, v_scale):
        _need(s is None or (s.dtype == torch.float32 and s.is_contiguous() and s.numel() == kv_heads),
              f"{name}: fp8 scales are contiguous float32 tensors of {kv_heads} values")


def _check_no_grad(name, q, k, v, k_scale, v_scale):
    """No argument that a derivative goes through, in either mode."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or k_scale is not None and k_scale.requires_grad
                                    or v_scale is not None and v_scale.requires_grad):
        raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad() or inference_mode()")
    if getattr(forward_ad, "_current_level", 0) >= 0:      # (outside every dual level nothing carries a tangent)
        for t in (q, k, v, k_scale, v_scale):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name} has no forward-mode derivative: an argument carries a tangent")


def _check_pool(name, q, k_cache, v_cache):
    _need(k_cache.dim() == 4 and v_cache.dim() == 4 and k_cache.shape == v_cache.shape,
          f"{name}: k_cache and v_cache are pools [pages, P, Hkv, D] of one shape")
    _need(k_cache.dtype == v_cache.dtype, f"{name}: K and V caches of different types")
    _need(k_cache.shape[3] == q.shape[2], f"{name}: head dims {q.shape[2]} (query) and {k_cache.shape[3]} (cache)")
    k_st, v_st = k_cache.stride(), v_cache.stride()
    _need(k_st[3] == 1 and v_st[3] == 1, f"{name}: the last dim of the caches must be contiguous")
    # a token's row is found at page * P + slot: the pool must be linear in it
    P = k_cache.shape[1]
    _need(k_st[0] == P * k_st[1] and v_st[0] == P * v_st[1], f"{name}: pages must follow each other in the pool")


def _check_table(name, what, table, rows):
    _need(table.dtype == torch.int32 and table.dim() == 2 and table.shape[0] == rows
          and (table.shape[1] <= 1 or table.stride(1) == 1),
          f"{name}: {what} must be int32 [{rows}, max_pages] with contiguous rows, got {table.dtype} {tuple(table.shape)}")


def _launch(fn, device, *args):
    """Calls the library on the tensors' device, whatever the current one is, and raises what it reports."""
    if device.index == torch.cuda.current_device():
        rc = fn(stream_handle(None, device.index), *args)
    else:
        with torch.cuda.device(device):
            rc = fn(stream_handle(None, device.index), *args)
    if rc:
        check(rc)


def _sig(t):
    """What the checks of an argument look at: a call whose arguments have all been seen before skips them."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _workspace(workspace, need, device):
    """The caller's workspace if it is large enough and aligned, else a new one."""
    if not need:
        return None
    if (isinstance(workspace, torch.Tensor) and workspace.device == device and workspace.is_contiguous()
            and workspace.data_ptr() % 256 == 0 and workspace.numel() * workspace.element_size() >= need):
        return workspace
    return torch.empty(need, dtype=torch.uint8, device=device)


_PREFILL_CACHE = {}   # fd_prefill_args images of calls by everything but the pointers
_SHARED_CACHE = {}


def _remember(cache, key, value):
    if len(cache) > 4096:
        cache.clear()
    cache[key] = value
    return value


def gqa_fwd_batch_prefill(q, k, v, cu_seqlens_q, kv_lens, block_table, scale, soft_cap=0.0, *, causal=True,
                          cu_seqlens_k: Optional[torch.Tensor] = None, q_lens: Optional[torch.Tensor] = None,
                          output: Optional[torch.Tensor] = None, lse_out: Optional[torch.Tensor] = None,
                          k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                          workspace: Optional[torch.Tensor] = None, max_kv_len: Optional[int] = None, kv_split: int = 0,
                          stream=None):
    """Attention of packed query rows ``q [total_q, Hq, D]`` -> ``output [total_q, Hq, D]`` in the query's type.

    Sequence ``b`` has the rows ``cu_seqlens_q[b] .. cu_seqlens_q[b + 1] - 1`` (int32 ``[B + 1]``), of which only the first
    ``q_lens[b]`` count if ``q_lens`` (int32 ``[B]``: a padded batch) is given.  Its keys are

    * in the paged pools ``k``, ``v`` ``[pages, P, Hkv, D]`` (the query's type, or fp8-e4m3 with ``k_scale`` / ``v_scale``
      ``[Hkv]``): ``kv_lens[b]`` tokens of row ``b`` of ``block_table`` (int32 ``[B, max_pages]``), the new ones included
      -- append first; a length beyond the table's room means the keys that there are, with the causal limits of the full
      length; or
    * with ``block_table=None`` and ``kv_lens=None`` packed in ``k``, ``v`` ``[total_k, Hkv, D]``: rows
      ``cu_seqlens_k[b] .. cu_seqlens_k[b + 1] - 1`` (default: ``cu_seqlens_q``).

    ``causal``: row ``i`` of ``n_q`` sees the keys ``j <= i + n_k - n_q`` -- the last row sees the last key; otherwise all
    rows see all keys of their sequence.  A row that sees nothing gets 0 (LSE ``-inf``); rows that belong to no sequence
    are left as they are in ``output`` and ``lse_out`` (fp32 ``[total_q, Hq]``, natural log).  A row that meets a NaN -- its
    own, a key's that it sees, a scale's -- is NaN, however its keys are split.  ``soft_cap``: 0 is off; a capped score is good
    to ``soft_cap * 2**-22``.  Head dims 64, 128, 256, fp16 / bf16, any number of query heads per KV head.

    ``workspace``: a contiguous GPU tensor on a 256-byte boundary that is used for partials if it is large enough
    (``prefill_workspace_bytes``).  ``max_kv_len``: an upper bound of the key counts, a hint.  ``kv_split``: 0 lets the
    library choose how many key ranges a row tile is cut into (more than one where there are few rows), else exactly that
    many, up to 64.  It chooses for caches of about equal length; for a few long ones among many short ones 8 is better (five
    drafted tokens on 24 caches of 17 - 16384 tokens: 98 us against 214).
    """
    if stream is not None:
        return _on(stream, gqa_fwd_batch_prefill, q, k, v, cu_seqlens_q, kv_lens, block_table, scale, soft_cap, causal=causal,
                   cu_seqlens_k=cu_seqlens_k, q_lens=q_lens, output=output, lse_out=lse_out, k_scale=k_scale, v_scale=v_scale,
                   workspace=workspace, max_kv_len=max_kv_len, kv_split=kv_split)
    _check_no_grad("gqa_fwd_batch_prefill", q, k, v, k_scale, v_scale)
    # (values: a tensor could change under the key)
    scale, soft_cap, causal = float(scale), float(soft_cap or 0.0), bool(causal)
    max_kv_len, kv_split = int(max_kv_len or 0), int(kv_split)
    key = (_sig(q), _sig(k), _sig(v), _sig(cu_seqlens_q), _sig(kv_lens), _sig(block_table), _sig(cu_seqlens_k), _sig(q_lens),
           _sig(output), _sig(lse_out), _sig(k_scale), _sig(v_scale), scale, soft_cap, causal, max_kv_len, kv_split)
    cached = _PREFILL_CACHE.get(key)
    if cached is None:
        cached = _remember(_PREFILL_CACHE, key, _prefill_image(
            "gqa_fwd_batch_prefill", q, k, v, cu_seqlens_q, kv_lens, block_table, scale, soft_cap, causal, cu_seqlens_k,
            q_lens, output, lse_out, k_scale, v_scale, max_kv_len, kv_split))
    image, need = cached
    if output is None:
        output = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if image is None:      # no rows, or no sequence
        return output
    a = FdPrefillArgs.from_buffer_copy(image)
    a.q = q_ptr = q.data_ptr()
    # (an empty tensor has no address: nothing is read through the stand-in)
    a.k, a.v = k.data_ptr() or q_ptr, v.data_ptr() or q_ptr
    a.cu_seqlens_q, a.out = cu_seqlens_q.data_ptr(), output.data_ptr()
    if lse_out is not None:
        a.lse_out = lse_out.data_ptr()
    if q_lens is not None:
        a.q_lens = q_lens.data_ptr()
    if block_table is not None:
        a.block_table, a.kv_lens = block_table.data_ptr(), kv_lens.data_ptr()
    else:
        a.cu_seqlens_k = (cu_seqlens_q if cu_seqlens_k is None else cu_seqlens_k).data_ptr()
    if k_scale is not None:
        a.params.k_scale, a.params.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
    if need:
        hold = _workspace(workspace, need, q.device)
        a.workspace, a.workspace_bytes = hold.data_ptr(), need
    _launch(load_library().fd_prefill, q.device, byref(a))
    return output


def prefill_workspace_bytes(q, k, v, cu_seqlens_q, kv_lens, block_table, *, cu_seqlens_k=None, k_scale=None, v_scale=None,
                            max_kv_len=None, kv_split=0) -> int:
    """Bytes of workspace that ``gqa_fwd_batch_prefill`` uses for tensors of these shapes (0: none)."""
    return _prefill_image("prefill_workspace_bytes", q, k, v, cu_seqlens_q, kv_lens, block_table, 1.0, 0.0, True,
                          cu_seqlens_k, None, None, None, k_scale, v_scale, int(max_kv_len or 0), int(kv_split))[1]


def _prefill_image(name, q, k, v, cu_q, kv_lens, block_table, scale, soft_cap, causal, cu_k, q_lens, output, lse_out,
                   k_scale, v_scale, max_kv_len, kv_split):
    """Checks a call and returns (the fd_prefill_args image without its pointers, bytes of workspace)."""
    _need(q.dim() == 3 and q.stride(2) == 1, f"{name}: q must be [total_q, Hq, D] with a contiguous last dim")
    _check_devices(name, q, k, v, cu_q, kv_lens, block_table, cu_k, q_lens, output, lse_out, k_scale, v_scale)
    _need(cu_q.dim() == 1 and cu_q.numel() >= 1, f"{name}: cu_seqlens_q must be int32 [batch + 1]")
    batch = cu_q.numel() - 1
    _check_int32(name, "cu_seqlens_q", cu_q, (batch + 1,))
    total_q, q_heads, head_dim = q.shape
    paged = block_table is not None
    if paged:
        _need(cu_k is None, f"{name}: cu_seqlens_k goes with packed keys, not with a block table")
        _need(kv_lens is not None, f"{name}: paged keys need kv_lens")
        _check_pool(name, q, k, v)
        _check_table(name, "block_table", block_table, batch)
        _check_int32(name, "kv_lens", kv_lens, (batch,))
        kv_heads, page_size, num_pages, max_pages = k.shape[2], k.shape[1], k.shape[0], block_table.shape[1]
        k_st, v_st, table_st = k.stride()[1:3], v.stride()[1:3], block_table.stride(0)
        total_k = 0
    else:
        _need(kv_lens is None, f"{name}: kv_lens goes with a block table; packed keys have cu_seqlens_k")
        _need(k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype and k.shape[2] == head_dim and k.stride(2) == 1
              and v.stride(2) == 1, f"{name}: packed k and v must be [total_k, Hkv, D] with a contiguous last dim")
        if cu_k is None:
            cu_k = cu_q
        _check_int32(name, "cu_seqlens_k", cu_k, (batch + 1,))
        kv_heads, page_size, num_pages, max_pages = k.shape[1], 0, 0, 0
        k_st, v_st, table_st = k.stride()[:2], v.stride()[:2], 0
        total_k = k.shape[0]
    _need(kv_heads > 0 and q_heads % kv_heads == 0, f"{name}: {q_heads} query heads on {kv_heads} KV heads")
    _check_scales(name, k_scale, v_scale, kv_heads)
    if q_lens is not None:
        _check_int32(name, "q_lens", q_lens, (batch,))
    _need(output is None or (output.shape == q.shape and output.dtype == q.dtype and output.stride(2) == 1),
          f"{name}: output must have the query's shape and type and a contiguous last dim")
    _need(lse_out is None or (lse_out.dtype == torch.float32 and tuple(lse_out.shape) == (total_q, q_heads)
                              and lse_out.is_contiguous()),
          f"{name}: lse_out must be a contiguous float32 tensor [{total_q}, {q_heads}]")
    a = FdPrefillArgs()
    a.stride_q_t, a.stride_q_h = q.stride()[:2]
    a.stride_ot, a.stride_oh = output.stride()[:2] if output is not None else (q_heads * head_dim, head_dim)
    (a.stride_k_tok, a.stride_k_h), (a.stride_v_tok, a.stride_v_h) = k_st, v_st
    a.stride_table_bs, a.sm_scale, a.batch, a.total_q, a.total_k = table_st, float(scale), batch, total_q, total_k
    a.causal = 1 if causal else 0
    p = a.params
    p.q_heads, p.kv_heads, p.head_dim, p.page_size, p.num_pages = q_heads, kv_heads, head_dim, page_size, num_pages
    p.max_pages_per_seq, p.q_dtype, p.kv_dtype = max_pages, fd_dtype_of(q), fd_dtype_of(k, fp8_bytes=k_scale is not None)
    p.out_dtype, p.soft_cap = p.q_dtype, float(soft_cap or 0.0)
    p.max_kv_len, p.num_splits = max_kv_len, kv_split
    probe = FdPrefillArgs.from_buffer_copy(a)
    probe.block_table = 256 if paged else None    # whether there is a table is all that the size asks of it
    need = load_library().fd_prefill_workspace_bytes(byref(probe))
    if need < 0:
        check(int(need))
    return (bytes(a) if total_q and batch else None), need


def gqa_fwd_batch_decode_shared_prefix(q, k_cache, v_cache, workspace, q_lens, kv_lens, block_table, prefix_lens,
                                       prefix_table, scale, soft_cap=0.0, *, group_starts: Optional[torch.Tensor] = None,
                                       output_combine: Optional[torch.Tensor] = None,
                                       lse_out: Optional[torch.Tensor] = None, k_scale: Optional[torch.Tensor] = None,
                                       v_scale: Optional[torch.Tensor] = None, max_kv_len: Optional[int] = None,
                                       max_prefix_len: Optional[int] = None, stream=None):
    """One decode step ``q [B, Hq, D]`` -> ``output_combine [B, Hq, D]`` of sequences that share prefixes.

    Group ``g`` -- the sequences ``group_starts[g] .. group_starts[g + 1] - 1`` (int32 ``[groups + 1]``; default: all
    sequences in one group) -- attends to the ``prefix_lens[g]`` tokens of row ``g`` of ``prefix_table`` (int32
    ``[groups, max_prefix_pages]``), and each sequence behind that to its own ``kv_lens[b]`` tokens of ``block_table``, as in
    ``gqa_fwd_batch_decode`` (``kv_lens`` does not count the prefix; 0 is allowed).  All pages are of the same pools; a
    sequence outside every group attends to its own tokens only.  The result is that of ``gqa_fwd_batch_decode`` over the
    concatenated tables, but a group's prefix is read from memory once: its part of the step is one matrix product of all the
    group's query heads.  ``q_lens`` is accepted and ignored, ``workspace`` used if it is large enough, as there; 16-bit
    queries with a cache of the same type or fp8-e4m3.  ``max_kv_len`` / ``max_prefix_len``: host-side hints.
    """
    if stream is not None:
        return _on(stream, gqa_fwd_batch_decode_shared_prefix, q, k_cache, v_cache, workspace, q_lens, kv_lens, block_table,
                   prefix_lens, prefix_table, scale, soft_cap, group_starts=group_starts, output_combine=output_combine,
                   lse_out=lse_out, k_scale=k_scale, v_scale=v_scale, max_kv_len=max_kv_len, max_prefix_len=max_prefix_len)
    _check_no_grad("gqa_fwd_batch_decode_shared_prefix", q, k_cache, v_cache, k_scale, v_scale)
    scale, soft_cap = float(scale), float(soft_cap or 0.0)
    # (the length hints count in steps of 1024 tokens, so that a growing batch keeps its prepared step)
    hints = (-(-int(max_kv_len or 0) // 1024) * 1024, -(-int(max_prefix_len or 0) // 1024) * 1024)
    key = (_sig(q), _sig(k_cache), _sig(v_cache), _sig(kv_lens), _sig(block_table), _sig(prefix_lens), _sig(prefix_table),
           _sig(group_starts), _sig(output_combine), _sig(lse_out), _sig(k_scale), _sig(v_scale), scale, soft_cap, hints)
    cached = _SHARED_CACHE.get(key)
    if cached is None:
        cached = _remember(_SHARED_CACHE, key, _shared_image(
            "gqa_fwd_batch_decode_shared_prefix", q, k_cache, v_cache, kv_lens, block_table, prefix_lens, prefix_table, scale,
            soft_cap, group_starts, output_combine, lse_out, k_scale, v_scale, hints))
    image, need = cached
    if output_combine is None:
        output_combine = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if image is None:      # no sequence
        return output_combine
    a = FdSharedArgs.from_buffer_copy(image)
    s = a.step
    hold = _workspace(workspace, need, q.device)
    s.workspace, s.workspace_bytes = hold.data_ptr(), need
    s.q, s.k_cache, s.v_cache, s.out = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), output_combine.data_ptr()
    s.block_table, s.kv_lens = block_table.data_ptr(), kv_lens.data_ptr()
    a.prefix_table, a.prefix_lens = prefix_table.data_ptr(), prefix_lens.data_ptr()
    if group_starts is not None:
        a.group_starts = group_starts.data_ptr()
    if lse_out is not None:
        s.lse_out = lse_out.data_ptr()
    if k_scale is not None:
        s.params.k_scale, s.params.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
    _launch(load_library().fd_decode_shared, q.device, byref(a))
    return output_combine


def _shared_image(name, q, k_cache, v_cache, kv_lens, block_table, prefix_lens, prefix_table, scale, soft_cap, group_starts,
                  output_combine, lse_out, k_scale, v_scale, hints):
    """Checks a call and returns (the fd_shared_args image without its pointers, bytes of workspace)."""
    _need(q.dim() == 3 and q.stride(2) == 1, f"{name}: q must be [B, Hq, D] with a contiguous last dim")
    _check_devices(name, q, k_cache, v_cache, kv_lens, block_table, prefix_lens, prefix_table, group_starts, output_combine,
                   lse_out, k_scale, v_scale)
    _check_pool(name, q, k_cache, v_cache)
    batch, q_heads, head_dim = q.shape
    kv_heads = k_cache.shape[2]
    _need(kv_heads > 0 and q_heads % kv_heads == 0, f"{name}: {q_heads} query heads on {kv_heads} KV heads")
    groups = prefix_table.shape[0]
    _check_table(name, "block_table", block_table, batch)
    _check_table(name, "prefix_table", prefix_table, groups)
    _check_int32(name, "kv_lens", kv_lens, (batch,))
    _check_int32(name, "prefix_lens", prefix_lens, (groups,))
    _check_scales(name, k_scale, v_scale, kv_heads)
    if group_starts is None:
        _need(groups == 1, f"{name}: {groups} prefixes need group_starts")
    else:
        _check_int32(name, "group_starts", group_starts, (groups + 1,))
    _need(output_combine is None or (output_combine.shape == q.shape and output_combine.dtype == q.dtype
                                     and output_combine.stride(2) == 1),
          f"{name}: output_combine must have the query's shape and type and a contiguous last dim")
    _need(lse_out is None or (lse_out.dtype == torch.float32 and lse_out.numel() == batch * q_heads
                              and lse_out.is_contiguous()), f"{name}: lse_out must be contiguous float32 [{batch}, {q_heads}]")
    if batch == 0:
        return None, 0
    q_st, k_st, v_st = q.stride(), k_cache.stride(), v_cache.stride()
    o_st = output_combine.stride() if output_combine is not None else (q_heads * head_dim, head_dim)
    a = FdSharedArgs()
    s = a.step
    s.stride_q_bs, s.stride_q_h, s.stride_obs, s.stride_oh = q_st[0], q_st[1], o_st[0], o_st[1]
    s.stride_k_tok, s.stride_k_h, s.stride_v_tok, s.stride_v_h = k_st[1], k_st[2], v_st[1], v_st[2]
    s.stride_table_bs, s.sm_scale, s.batch, s.combine_mode = block_table.stride(0), float(scale), batch, FD_COMBINE_SPLIT
    p: FdParams = s.params
    p.q_heads, p.kv_heads, p.head_dim, p.page_size = q_heads, kv_heads, head_dim, k_cache.shape[1]
    p.num_splits, p.num_pages, p.max_pages_per_seq = -1, k_cache.shape[0], block_table.shape[1]
    p.q_dtype, p.kv_dtype = fd_dtype_of(q), fd_dtype_of(k_cache, fp8_bytes=k_scale is not None)
    p.out_dtype, p.soft_cap, p.max_kv_len = p.q_dtype, float(soft_cap or 0.0), hints[0]
    a.stride_prefix_bs, a.groups, a.prefix_max_pages = prefix_table.stride(0), groups, prefix_table.shape[1]
    a.max_prefix_len = hints[1]
    need = load_library().fd_decode_shared_workspace_bytes(byref(a))
    if need < 0:
        check(int(need))
    return bytes(a), need
