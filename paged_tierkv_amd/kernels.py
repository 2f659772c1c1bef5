"""Python entry points of the demotion, promotion, block-score and label
kernels, and of a serving step's slot map, norm and rotation of rows, K/V row
writes (HOT and quantized), rows read back and token choice (C ABI in
include/tierkv_hip.h).

All tensors are GPU tensors; index arrays are int32.  Launches are
asynchronous on the current stream.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

WARM_FORMATS = {"ref_u8": _lib.WARM_REF_U8, "absmax_i8": _lib.WARM_ABSMAX_I8}
LABEL_MODES = {"hot_only": 0, "hot_warm": 1, "hot_warm_cold": 2}


def _i32(x, device) -> torch.Tensor:
    t = torch.as_tensor(x, dtype=torch.int32)
    return t.to(device).contiguous()


def _table_positions(table_pos, block_table, block_states, n, device):
    """Validate (on the host, where the positions usually come from) and
    upload the flat table positions of a migration batch."""
    if table_pos is None:
        return None
    if block_table is None or block_states is None:
        raise ValueError("table_pos needs block_table and block_states.")
    host = torch.as_tensor(table_pos, dtype=torch.int32)
    if host.numel() != n:
        raise ValueError("table_pos needs one entry per job.")
    if host.device.type == "cpu" and host.numel():
        hi = int(host.max())
        if hi >= min(block_table.numel(), block_states.numel()):
            raise ValueError("table_pos entry outside the block table.")
    return host.to(device).contiguous()


def _check_tiles(t: torch.Tensor, name: str, dtype) -> None:
    _lib.require_gpu_tensor(t, name)
    if t.dtype != dtype or t.ndim != 4 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} [tiles, kv_heads, block_size, head_dim] tensor.")


def demote_to_warm(src_k, src_v, src_index, dst_slot, lengths, warm_k, warm_v, k_scale, k_zero,
                   v_scale, v_zero, warm_format: str = "ref_u8", pad_tail: bool = False,
                   block_table=None, block_states=None, table_pos=None):
    """Quantize fp16 tiles ``src_k/src_v[src_index[i]]`` (first ``lengths[i]``
    tokens) into WARM slots ``dst_slot[i]``; optionally rewrite
    ``block_table/block_states`` at flat positions ``table_pos`` to
    (dst_slot, WARM).  Batched CompactTieredKVTensorPool.demote_to_warm
    (tierkv_policy.py:1042-1068) / write_warm_block (969-1002)."""
    lib = _lib.lib()
    fmt = WARM_FORMATS[warm_format]
    _check_tiles(src_k, "src_k", torch.float16)
    _check_tiles(src_v, "src_v", torch.float16)
    _check_tiles(warm_k, "warm_k", torch.uint8 if fmt == _lib.WARM_REF_U8 else torch.int8)
    _check_tiles(warm_v, "warm_v", warm_k.dtype)
    kv_heads, bs, dim = (int(x) for x in src_k.shape[1:])
    if tuple(warm_k.shape[1:]) != (kv_heads, bs, dim) or src_v.shape != src_k.shape or warm_v.shape != warm_k.shape:
        raise ValueError("source and WARM pool geometry differ.")
    device = src_k.device
    src_index = _i32(src_index, device)
    dst_slot = _i32(dst_slot, device)
    lengths = _i32(lengths, device)
    n = int(src_index.numel())
    if dst_slot.numel() != n or lengths.numel() != n:
        raise ValueError("src_index, dst_slot and lengths must have the same length.")
    tp = _table_positions(table_pos, block_table, block_states, n, device)
    rc = lib.tierkv_demote_to_warm(
        _lib.ptr(src_k), _lib.ptr(src_v), int(src_k.shape[0]),
        _lib.ptr(src_index), _lib.ptr(dst_slot), _lib.ptr(lengths), n,
        _lib.ptr(warm_k), _lib.ptr(warm_v), int(warm_k.shape[0]),
        _lib.ptr(k_scale), _lib.ptr(k_zero), _lib.ptr(v_scale), _lib.ptr(v_zero),
        fmt, int(bool(pad_tail)),
        _lib.ptr(block_table), _lib.ptr(block_states), _lib.ptr(tp),
        kv_heads, bs, dim, _lib.stream_of(device))
    _lib.check(rc, "tierkv_demote_to_warm")


def promote_to_hot(warm_k, warm_v, k_scale, k_zero, v_scale, v_zero, src_slot, dst_slot, lengths,
                   hot_k, hot_v, warm_format: str = "ref_u8",
                   block_table=None, block_states=None, table_pos=None):
    """Dequantize WARM slots into HOT slots (promote_to_hot,
    tierkv_policy.py:1087-1115, with dequantize_int8_to_fp16, 39-44)."""
    lib = _lib.lib()
    fmt = WARM_FORMATS[warm_format]
    _check_tiles(hot_k, "hot_k", torch.float16)
    _check_tiles(hot_v, "hot_v", torch.float16)
    _check_tiles(warm_k, "warm_k", torch.uint8 if fmt == _lib.WARM_REF_U8 else torch.int8)
    kv_heads, bs, dim = (int(x) for x in hot_k.shape[1:])
    device = hot_k.device
    src_slot = _i32(src_slot, device)
    dst_slot = _i32(dst_slot, device)
    lengths = _i32(lengths, device)
    n = int(src_slot.numel())
    tp = _table_positions(table_pos, block_table, block_states, n, device)
    rc = lib.tierkv_promote_to_hot(
        _lib.ptr(warm_k), _lib.ptr(warm_v), int(warm_k.shape[0]),
        _lib.ptr(k_scale), _lib.ptr(k_zero), _lib.ptr(v_scale), _lib.ptr(v_zero),
        _lib.ptr(src_slot), _lib.ptr(dst_slot), _lib.ptr(lengths), n,
        _lib.ptr(hot_k), _lib.ptr(hot_v), int(hot_k.shape[0]), fmt,
        _lib.ptr(block_table), _lib.ptr(block_states), _lib.ptr(tp),
        kv_heads, bs, dim, _lib.stream_of(device))
    _lib.check(rc, "tierkv_promote_to_hot")


def block_mass_from_probs(probs: torch.Tensor, block_size: int, lengths: torch.Tensor | None = None,
                          out: torch.Tensor | None = None):
    """fp32 probabilities [B, H, T] -> per-block mass [B, T / block_size]
    (written into ``out`` when given: contiguous fp32 of that shape)."""
    lib = _lib.lib()
    _lib.require_gpu_tensor(probs, "probs")
    if probs.dtype != torch.float32 or probs.ndim != 3:
        raise ValueError("probs must be fp32 [batch, heads, tokens].")
    probs = probs.contiguous()
    batch, heads, tokens = (int(x) for x in probs.shape)
    if tokens % int(block_size):
        raise ValueError("tokens must be a multiple of block_size.")
    nblk = tokens // int(block_size)
    if out is None:
        out = torch.empty((batch, nblk), dtype=torch.float32, device=probs.device)
    elif (out.dtype != torch.float32 or tuple(out.shape) != (batch, nblk) or not out.is_contiguous()
          or out.device != probs.device):
        raise ValueError("out must be a contiguous fp32 [batch, tokens / block_size] tensor on the probs' device.")
    if lengths is not None:
        lengths = _i32(lengths, probs.device)
        if tuple(lengths.shape) != (batch, nblk):
            raise ValueError("lengths must be [batch, tokens / block_size].")
    rc = lib.tierkv_block_mass_from_probs(_lib.ptr(probs), _lib.ptr(lengths), _lib.ptr(out),
                                          batch, heads, tokens, int(block_size), _lib.stream_of(probs.device))
    _lib.check(rc, "tierkv_block_mass_from_probs")
    return out


def block_scores_from_sums(score_sums: torch.Tensor, lengths: torch.Tensor, num_blocks: int):
    """block_scores_from_probability_sums (tierkv_policy.py:1905-1912):
    score_sums [H, maxB] / [B, H, maxB], lengths [maxB] / [B, maxB] ->
    [n] / [B, n] fp32."""
    lib = _lib.lib()
    squeeze = score_sums.ndim == 2
    s = score_sums.unsqueeze(0) if squeeze else score_sums
    ln = lengths.unsqueeze(0) if lengths.ndim == 1 else lengths
    s = s.contiguous()
    ln = ln.to(torch.int32).contiguous()
    batch, heads, stride = (int(x) for x in s.shape)
    n = int(num_blocks)
    out = torch.empty((batch, n), dtype=torch.float32, device=s.device)
    rc = lib.tierkv_block_scores_from_sums(_lib.ptr(s), stride, _lib.ptr(ln), int(ln.shape[-1]), _lib.ptr(out),
                                           batch, heads, n, _lib.stream_of(s.device))
    _lib.check(rc, "tierkv_block_scores_from_sums")
    return out[0] if squeeze else out


def tier_labels(scores: torch.Tensor, cur_states: torch.Tensor, hot_budget: int, warm_budget: int = 0,
                mode: str = "hot_warm_cold", demoted_state: int = 1, out: torch.Tensor | None = None):
    """enforce_tiered_budget / enforce_budget for a batch of sequences.
    scores fp32 [B, n] (or [n]); cur_states int32 [B, >= n] -> new states
    int32 of cur_states' shape (entries >= n copied unchanged)."""
    lib = _lib.lib()
    squeeze = scores.ndim == 1
    sc = (scores.unsqueeze(0) if squeeze else scores).to(torch.float32).contiguous()
    cur = (cur_states.unsqueeze(0) if cur_states.ndim == 1 else cur_states).to(torch.int32).contiguous()
    batch, n = (int(x) for x in sc.shape)
    if out is None:
        # The kernel writes every entry below n: only a wider or taller table
        # needs its other entries copied first (a device copy, about 5 us of a
        # 17 us scoring call).
        out = torch.empty_like(cur) if tuple(cur.shape) == (batch, n) else cur.clone()
    else:
        out = out.unsqueeze(0) if out.ndim == 1 else out
    rc = lib.tierkv_tier_labels(_lib.ptr(sc), _lib.ptr(cur), _lib.ptr(out), int(cur.shape[-1]), batch, n,
                                int(hot_budget), int(warm_budget), LABEL_MODES[mode], int(demoted_state),
                                _lib.stream_of(sc.device))
    _lib.check(rc, "tierkv_tier_labels")
    return out[0] if squeeze else out


_prefill_ws: dict = {}


def prefill_block_mass(query_states: torch.Tensor, key_states: torch.Tensor, block_size: int, scaling: float):
    """Per-sequence prefill block scores without materialised probabilities
    (``tierkv_prefill_block_mass``): query [B, H, T, D] and key [B, H_kv, T, D]
    (fp16 / bf16, any layout with head_dim contiguous, e.g. HF's transposed
    projections) -> fp32 [B, ceil(T / block_size)], the mean causal attention
    probability of each block over heads and queries (compute_block_scores,
    tierkv_policy.py:1380-1389, per sequence)."""
    lib = _lib.lib()
    _lib.require_gpu_tensor(query_states, "query_states")
    _lib.require_gpu_tensor(key_states, "key_states")
    if query_states.ndim != 4 or key_states.ndim != 4:
        raise ValueError("query and key states must be [batch, heads, tokens, head_dim].")
    if query_states.dtype not in (torch.float16, torch.bfloat16) or key_states.dtype != query_states.dtype:
        raise ValueError("query and key states must share an fp16 / bf16 dtype.")
    q, k = query_states, key_states
    if q.stride(-1) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.stride(2) % 8 or q.data_ptr() % 16:
        q = q.contiguous()
    if k.stride(-1) != 1 or k.stride(0) % 8 or k.stride(1) % 8 or k.stride(2) % 8 or k.data_ptr() % 16:
        k = k.contiguous()
    batch, heads, tokens, dim = (int(x) for x in q.shape)
    if k.shape[0] != batch or k.shape[2] != tokens or k.shape[3] != dim:
        raise ValueError("key states do not match the query geometry.")
    kv_heads = int(k.shape[1])
    need = int(lib.tierkv_prefill_block_mass_full_workspace_bytes(batch, heads, kv_heads, tokens))
    # One scratch buffer per (device, stream): calls on one stream are enqueued
    # whole, one after another (_lib.call_lock); launches on different streams
    # may overlap and never share it.  The call passes what this shape needs,
    # not what the buffer holds, so its summation order does not depend on
    # earlier calls.
    nblk = (tokens + int(block_size) - 1) // int(block_size)
    out = torch.empty((batch, nblk), dtype=torch.float32, device=q.device)
    key = (q.device.index, _lib.stream_of(q.device))
    with _lib.call_lock:
        ws = _prefill_ws.get(key)
        if ws is None or ws.numel() < need:
            ws = torch.empty(max(need, 256), dtype=torch.uint8, device=q.device)
            _prefill_ws[key] = ws
        rc = lib.tierkv_prefill_block_mass(
            _lib.ptr(q), q.stride(0), q.stride(1), q.stride(2), _lib.ptr(k), k.stride(0), k.stride(1), k.stride(2),
            _lib.DTYPE_BF16 if q.dtype == torch.bfloat16 else _lib.DTYPE_F16, _lib.ptr(out), batch, heads, kv_heads,
            tokens, dim, int(block_size), float(scaling), _lib.ptr(ws), need, _lib.stream_of(q.device))
    _lib.check(rc, "tierkv_prefill_block_mass")
    return out


# One scratch buffer per (operator, device, stream), as the prefill scores':
# calls on one stream are enqueued whole, one after another (_lib.call_lock);
# launches on different streams may overlap and never share it.  A captured
# call takes scratch of its own from
# its graph's memory, so that graphs replayed on different streams, and eager
# calls beside them, share none.
_scratch_ws: dict = {}


def _scratch(name: str, device, need: int, zeros: int = 0) -> torch.Tensor:
    """At least ``need`` bytes whose first ``zeros`` are zero when new."""
    capturing = torch.cuda.is_current_stream_capturing()   # (a capture is the current device's)
    key = (name, device.index, _lib.stream_of(device))
    ws = None if capturing else _scratch_ws.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.empty(max(need, 256), dtype=torch.uint8, device=device)
        if zeros:
            ws[:zeros].zero_()
        if not capturing:
            _scratch_ws[key] = ws
    return ws


def _on_device(device, call, *args) -> int:
    """``call(*args, stream)`` with ``device`` current and its current stream."""
    if torch.cuda.current_device() == device.index:
        return call(*args, _lib.stream_of(device))
    with torch.cuda.device(device):
        return call(*args, _lib.stream_of(device))


class SlotMap(NamedTuple):
    """``build_slot_map``'s outputs (all int32, on the tables' device)."""

    slots: torch.Tensor       # [num_tokens] slot * block_size + position of each packed row, -1 behind the last request
    positions: torch.Tensor   # [num_tokens] the row's position in its request, or -1
    cu_tokens: torch.Tensor   # [B + 1] first packed row of each request
    context: torch.Tensor     # [B] tokens each request holds after the step


def _require_i32(t, name: str, shape=None) -> None:
    _lib.require_gpu_tensor(t, name)
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor.")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}.")


def build_slot_map(new_tokens: torch.Tensor, block_table: torch.Tensor, block_states: torch.Tensor,
                   block_lengths: torch.Tensor, seq_num_blocks: torch.Tensor, open_blocks: torch.Tensor,
                   hot_free: torch.Tensor, ctl: torch.Tensor, block_size: int, num_tokens: int) -> SlotMap:
    """Table entries and slot map of a step in which request b brings
    ``new_tokens[b]`` tokens (``tierkv_build_slot_map``): its open block is
    filled first, then new HOT blocks are popped from ``hot_free``; the tables
    ``[B, max_blocks]``, ``seq_num_blocks``, ``open_blocks`` ``[B]`` and ``ctl``
    ``[4]`` are updated in place, as ``BatchedTieredKVRuntime`` holds them.
    ``num_tokens`` is the number of packed rows (at least the lengths' sum;
    rows behind the last request get slot -1).  All or nothing: a step that
    does not fit changes no table, sets an error bit in ``ctl[2]`` and gives
    every row slot -1."""
    lib = _lib.lib()
    _lib.require_gpu_tensor(block_table, "block_table")
    if block_table.ndim != 2:
        raise ValueError("block_table must be [batch, max_blocks].")
    shape = block_table.shape
    batch, stride = shape
    index = block_table.get_device()
    for name, t, want in (("block_table", block_table, shape), ("block_states", block_states, shape),
                          ("block_lengths", block_lengths, shape), ("new_tokens", new_tokens, shape[:1]),
                          ("seq_num_blocks", seq_num_blocks, shape[:1]), ("open_blocks", open_blocks, shape[:1]),
                          ("hot_free", hot_free, None), ("ctl", ctl, (4,))):
        _require_i32(t, name, want)
        if t.get_device() != index:
            raise ValueError("the slot map's tensors must be on one device.")
    device = block_table.device
    rows = int(num_tokens)
    if rows < 0:
        raise ValueError("num_tokens must not be negative.")
    # One allocation: slots and positions start at multiples of 16 bytes.
    pad = -rows % 4
    slots, _, positions, _, cu, context = torch.empty(2 * (rows + pad) + 2 * batch + 1, dtype=torch.int32,
                                                      device=device).split([rows, pad, rows, pad, batch + 1, batch])
    need = lib.tierkv_slot_map_workspace_bytes(batch)
    ptr = _lib.ptr
    with _lib.call_lock:
        ws = _scratch("slot_map", device, need)
        rc = _on_device(device, lib.tierkv_build_slot_map, ptr(new_tokens), batch, rows, ptr(block_table),
                        ptr(block_states), ptr(block_lengths), stride, ptr(seq_num_blocks), ptr(open_blocks),
                        ptr(hot_free), hot_free.numel(), ptr(ctl), int(block_size), ptr(slots), ptr(positions), ptr(cu),
                        ptr(context), ptr(ws), ws.numel())
    _lib.check(rc, "tierkv_build_slot_map")
    return SlotMap(slots, positions, cu, context)


def write_slots(key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor, hot_k: torch.Tensor,
                hot_v: torch.Tensor) -> None:
    """Copy packed K/V rows ``[N, kv_heads, head_dim]`` (fp16 / bf16, any
    strides with head_dim contiguous, e.g. columns of a fused projection) into
    the HOT pool rows ``slots`` (``build_slot_map``; negative: skipped)."""
    lib = _lib.lib()
    _check_tiles(hot_k, "hot_k", torch.float16)
    _check_tiles(hot_v, "hot_v", torch.float16)
    kv_heads, bs, dim = (int(x) for x in hot_k.shape[1:])
    if hot_v.shape != hot_k.shape:
        raise ValueError("K and V pools must have identical shapes.")
    _lib.require_gpu_tensor(key, "key")
    _lib.require_gpu_tensor(value, "value")
    if key.dtype not in (torch.float16, torch.bfloat16) or value.dtype != key.dtype:
        raise ValueError("key and value must share an fp16 / bf16 dtype.")
    if key.ndim != 3 or value.shape != key.shape or tuple(key.shape[1:]) != (kv_heads, dim):
        raise ValueError("key and value must be [tokens, kv_heads, head_dim] of the pools' geometry.")
    rows = int(key.shape[0])
    _require_i32(slots, "slots", (rows,))
    index = hot_k.get_device()
    if any(t.get_device() != index for t in (key, value, slots, hot_v)):
        raise ValueError("rows, slots and pools must be on one device.")
    if rows == 0:
        return
    k = key if key.stride(2) == 1 or dim == 1 else key.contiguous()
    v = value if value.stride(2) == 1 or dim == 1 else value.contiguous()
    kt, kh, _ = k.stride()
    vt, vh, _ = v.stride()
    ptr = _lib.ptr
    rc = _on_device(hot_k.device, lib.tierkv_write_slots, ptr(k), kt, kh, ptr(v), vt, vh,
                    _lib.DTYPE_BF16 if k.dtype == torch.bfloat16 else _lib.DTYPE_F16, ptr(slots), rows, ptr(hot_k),
                    ptr(hot_v), hot_k.shape[0], kv_heads, bs, dim)
    _lib.check(rc, "tierkv_write_slots")


_HALVES = (torch.float16, torch.bfloat16)


def _is(t, dtype, shape, index: int) -> bool:
    """Whether t is a contiguous tensor of this dtype, shape and device."""
    return (isinstance(t, torch.Tensor) and t.dtype == dtype and t.get_device() == index and t.shape == shape
            and t.is_contiguous())


def _packed_rows(t, name: str, shape, dtype, index: int):
    """Packed rows [rows, heads, dim] with the last dim contiguous (copied
    where it is not)."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name} must be [tokens, heads, head_dim] of the step's geometry and the rows' dtype.")
    if t.get_device() != index:
        raise ValueError("rows, tables and pools must be on one device.")
    return t if t.stride(2) == 1 or shape[2] == 1 else t.contiguous()


def _out_rows(t, name: str, shape, dtype, device, index: int):
    if t is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if not _is(t, dtype, shape, index):
        raise ValueError(f"{name} must be a contiguous tensor of the rows' shape, dtype and device.")
    return t


def _step_i32(t, name: str, shape, index: int) -> None:
    if not _is(t, torch.int32, shape, index):
        _require_i32(t, name, shape)
        raise ValueError("rows, tables and pools must be on one device.")


def _hot_pools(hot_k, hot_v, index: int) -> None:
    if not (isinstance(hot_k, torch.Tensor) and hot_k.ndim == 4 and _is(hot_k, torch.float16, hot_k.shape, index)
            and _is(hot_v, torch.float16, hot_k.shape, index)):
        _check_tiles(hot_k, "hot_k", torch.float16)
        _check_tiles(hot_v, "hot_v", torch.float16)
        if hot_v.shape != hot_k.shape:
            raise ValueError("K and V pools must have identical shapes.")
        raise ValueError("rows, tables and pools must be on one device.")


def _warm_pools(warm_k, warm_v, k_scale, k_zero, v_scale, v_zero, fmt: int, index: int) -> None:
    """Check WARM pools and their metadata (``fmt``: WARM_FORMATS' value)."""
    ref = fmt == _lib.WARM_REF_U8
    dtype = torch.uint8 if ref else torch.int8
    if not (isinstance(warm_k, torch.Tensor) and warm_k.ndim == 4 and _is(warm_k, dtype, warm_k.shape, index)
            and _is(warm_v, dtype, warm_k.shape, index)):
        _check_tiles(warm_k, "warm_k", dtype)
        _check_tiles(warm_v, "warm_v", dtype)
        if warm_v.shape != warm_k.shape:
            raise ValueError("K and V pools must have identical shapes.")
        raise ValueError("rows, tables and pools must be on one device.")
    slots, kv_heads, bs, _ = warm_k.shape
    entries, kind = (slots * kv_heads * bs, torch.float16) if ref else (slots * kv_heads, torch.float32)
    for t in (k_scale, k_zero, v_scale, v_zero) if ref else (k_scale, v_scale):
        if t is None:
            raise ValueError("WARM pools need their scales, reference-format ones their zero points.")
        _lib.require_gpu_tensor(t, "warm metadata")
        if t.dtype != kind or t.numel() != entries or not t.is_contiguous():
            raise ValueError("WARM metadata must be contiguous: fp16 per token and head (ref_u8), fp32 per slot and "
                             "head (absmax_i8).")
        if t.get_device() != index:
            raise ValueError("rows, tables and pools must be on one device.")


def rotate_rows(query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *,
                q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                attention_scaling: float = 1.0, interleaved: bool = False, value: torch.Tensor | None = None,
                slots: torch.Tensor | None = None, hot_k: torch.Tensor | None = None,
                hot_v: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
                k_out: torch.Tensor | None = None):
    """Per-head norms and rotation by position of a step's packed rows
    (``tierkv_rotate_rows``): ``query`` ``[N, H, D]``, ``key`` ``[N, kv_heads,
    D]`` (fp16 / bf16, any strides with head_dim contiguous, e.g. columns of a
    fused projection), ``positions`` int32 ``[N]`` (``build_slot_map``; rows of
    negative ones are left out), ``inv_freq`` fp32 ``[rotary_dim / 2]``.  Where a
    weight ``[head_dim]`` is given (the rows' dtype or fp32), the heads become
    ``x * rsqrt(mean(x^2) + eps) * weight`` first; the first ``rotary_dim`` dims
    turn in pairs ``(i, i + rotary_dim / 2)``, ``interleaved``: ``(2 i, 2 i + 1)``,
    by angles formed in 64 bits, and are scaled by ``attention_scaling``.  With
    ``value``, ``slots`` and the HOT pools, keys and values go there as
    ``write_slots`` puts them.  Returns ``(q_out, k_out)``: contiguous rows (the
    tensors given, which must not overlap the inputs, or new ones), ``k_out``
    None where the keys go to pools and none is given.  Rows that are left out
    are not written."""
    lib = _lib.lib()
    _lib.require_gpu_tensor(query, "query")
    _lib.require_gpu_tensor(key, "key")
    if query.ndim != 3 or key.ndim != 3 or query.dtype not in _HALVES:
        raise ValueError("query and key must be fp16 / bf16 [tokens, heads, head_dim].")
    shape = query.shape
    rows, heads, dim = shape
    kv_heads = key.shape[1]
    kv_shape = (rows, kv_heads, dim)
    index, device, dtype = query.get_device(), query.device, query.dtype
    q = _packed_rows(query, "query", shape, dtype, index)
    k = _packed_rows(key, "key", kv_shape, dtype, index)
    _step_i32(positions, "positions", (rows,), index)
    half = inv_freq.numel() if isinstance(inv_freq, torch.Tensor) else 0
    if not _is(inv_freq, torch.float32, (half,), index) or 2 * half > dim:
        raise ValueError("inv_freq must be contiguous fp32 [rotary_dim / 2] on the rows' device, rotary_dim at most head_dim.")
    of = q_weight if q_weight is not None else k_weight
    for w in (q_weight, k_weight):
        if w is not None and (w.dtype not in (dtype, torch.float32) or not _is(w, of.dtype, (dim,), index)):
            raise ValueError("norm weights must be contiguous [head_dim] tensors of the rows' dtype or fp32, both alike.")
    bs, pool, v, vt, vh = 1, 0, None, 0, 0
    if slots is None:
        if value is not None or hot_k is not None or hot_v is not None:
            raise ValueError("value, slots, hot_k and hot_v go together.")
    else:
        if value is None or hot_k is None or hot_v is None:
            raise ValueError("value, slots, hot_k and hot_v go together.")
        _hot_pools(hot_k, hot_v, index)
        pool, pool_heads, bs, pool_dim = hot_k.shape
        if pool_heads != kv_heads or pool_dim != dim:
            raise ValueError("the pools must have the rows' geometry.")
        _step_i32(slots, "slots", (rows,), index)
        v = _packed_rows(value, "value", kv_shape, dtype, index)
        vt, vh, _ = v.stride()
    q_out = _out_rows(q_out, "q_out", shape, dtype, device, index)
    if k_out is not None or slots is None:
        k_out = _out_rows(k_out, "k_out", kv_shape, dtype, device, index)
    qt, qh, _ = q.stride()
    kt, kh, _ = k.stride()
    code = _lib.DTYPE_BF16 if dtype == torch.bfloat16 else _lib.DTYPE_F16
    ptr = _lib.ptr
    rc = _on_device(device, lib.tierkv_rotate_rows, ptr(q), qt, qh, ptr(q_out), ptr(k), kt, kh, ptr(k_out), ptr(v), vt,
                    vh, code, ptr(positions), rows, ptr(inv_freq), 2 * half, 1 if interleaved else 0, attention_scaling,
                    ptr(q_weight), ptr(k_weight), _lib.DTYPE_F32 if of is not None and of.dtype == torch.float32 else code,
                    eps, ptr(slots), ptr(hot_k), ptr(hot_v), pool, heads, kv_heads, bs, dim)
    _lib.check(rc, "tierkv_rotate_rows")
    return q_out, k_out


def quantize_rows(key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor, warm_k: torch.Tensor,
                  warm_v: torch.Tensor, k_scale: torch.Tensor, k_zero: torch.Tensor | None, v_scale: torch.Tensor,
                  v_zero: torch.Tensor | None, warm_format: str = "ref_u8") -> None:
    """Quantize packed K/V rows ``[N, kv_heads, head_dim]`` (as ``write_slots``
    takes them) into the WARM pool rows ``slots`` (slot * block_size +
    position; negative: skipped), as a step writes them
    (``tierkv_quantize_rows``).  ``ref_u8``: each row and head by itself, as
    ``demote_to_warm`` does.  ``absmax_i8``: a block's rows are consecutive in
    the call, with no skipped row among them; the block's scale grows where
    they ask for it, and the rows that it holds before them are brought to the
    new scale, rounded once more: in a block of b tokens filled one by one, the
    values of position p end within (b - p) / 2 steps of the last scale."""
    lib = _lib.lib()
    if warm_format not in WARM_FORMATS:
        raise ValueError('warm_format must be "absmax_i8" or "ref_u8".')
    fmt = WARM_FORMATS[warm_format]
    _lib.require_gpu_tensor(key, "key")
    _lib.require_gpu_tensor(value, "value")
    _lib.require_gpu_tensor(slots, "slots")
    index = key.get_device()
    _warm_pools(warm_k, warm_v, k_scale, k_zero, v_scale, v_zero, fmt, index)
    pool, kv_heads, bs, dim = warm_k.shape
    if key.ndim != 3 or key.dtype not in _HALVES:
        raise ValueError("key and value must be fp16 / bf16 [tokens, kv_heads, head_dim].")
    rows, dtype = key.shape[0], key.dtype
    k = _packed_rows(key, "key", (rows, kv_heads, dim), dtype, index)
    v = _packed_rows(value, "value", (rows, kv_heads, dim), dtype, index)
    _step_i32(slots, "slots", (rows,), index)
    if rows == 0:
        return
    kt, kh, _ = k.stride()
    vt, vh, _ = v.stride()
    ptr, ref = _lib.ptr, fmt == _lib.WARM_REF_U8
    rc = _on_device(key.device, lib.tierkv_quantize_rows, ptr(k), kt, kh, ptr(v), vt, vh,
                    _lib.DTYPE_BF16 if dtype == torch.bfloat16 else _lib.DTYPE_F16, ptr(slots), rows,
                    ptr(warm_k), ptr(warm_v), pool, ptr(k_scale), ptr(k_zero) if ref else None, ptr(v_scale),
                    ptr(v_zero) if ref else None, fmt, kv_heads, bs, dim)
    _lib.check(rc, "tierkv_quantize_rows")


def read_rows(start: torch.Tensor, cu_tokens: torch.Tensor, num_tokens: int, block_table: torch.Tensor,
              block_states: torch.Tensor, block_lengths: torch.Tensor, seq_num_blocks: torch.Tensor | None,
              hot_k: torch.Tensor, hot_v: torch.Tensor, warm_k: torch.Tensor, warm_v: torch.Tensor,
              k_scale: torch.Tensor, k_zero: torch.Tensor | None, v_scale: torch.Tensor, v_zero: torch.Tensor | None,
              dtype: torch.dtype = torch.float16, out=None):
    """Tokens of a tiered cache as packed rows (``tierkv_read_rows``): rows
    ``cu_tokens[b]`` to ``cu_tokens[b + 1]`` (int32 ``[B + 1]``) are request b's
    tokens from ordinal ``start[b]`` (int32 ``[B]``) on, in order; evicted ones
    and those past what the request holds are 0.  Tables are ``[B,
    max_blocks]``, pools and metadata those of ``tierkv_extend_attention``.
    Returns K and V ``[num_tokens, kv_heads, head_dim]`` of ``dtype`` (fp16, bf16
    or fp32; ``out``: a pair to write into).  Rows of no request are not
    written."""
    lib = _lib.lib()
    _lib.require_gpu_tensor(block_table, "block_table")
    if block_table.ndim != 2:
        raise ValueError("block_table must be [batch, max_blocks].")
    shape = block_table.shape
    batch, stride = shape
    index, device = block_table.get_device(), block_table.device
    _step_i32(block_table, "block_table", shape, index)
    _step_i32(block_states, "block_states", shape, index)
    _step_i32(block_lengths, "block_lengths", shape, index)
    _step_i32(start, "start", (batch,), index)
    _step_i32(cu_tokens, "cu_tokens", (batch + 1,), index)
    if seq_num_blocks is not None:
        _step_i32(seq_num_blocks, "seq_num_blocks", (batch,), index)
    if dtype not in _LOGIT_DTYPES:
        raise ValueError("dtype must be fp16, bf16 or fp32.")
    rows = int(num_tokens)
    if not 0 <= rows < 1 << 31:
        raise ValueError("num_tokens must not be negative or pass 2^31.")
    _hot_pools(hot_k, hot_v, index)
    _lib.require_gpu_tensor(warm_k, "warm_k")
    fmt = _lib.WARM_ABSMAX_I8 if warm_k.dtype == torch.int8 else _lib.WARM_REF_U8
    _warm_pools(warm_k, warm_v, k_scale, k_zero, v_scale, v_zero, fmt, index)
    hot, kv_heads, bs, dim = hot_k.shape
    warm, *geometry = warm_k.shape
    if geometry != [kv_heads, bs, dim]:
        raise ValueError("HOT and WARM pools must have one geometry.")
    want = (rows, kv_heads, dim)
    k_rows, v_rows = (None, None) if out is None else out
    k_rows = _out_rows(k_rows, "out", want, dtype, device, index)
    v_rows = _out_rows(v_rows, "out", want, dtype, device, index)
    ptr, ref = _lib.ptr, fmt == _lib.WARM_REF_U8
    rc = _on_device(device, lib.tierkv_read_rows, ptr(start), ptr(cu_tokens), rows, ptr(block_table), ptr(block_states),
                    ptr(block_lengths), stride, ptr(seq_num_blocks), stride, ptr(hot_k), ptr(hot_v), hot,
                    ptr(warm_k), ptr(warm_v), warm, ptr(k_scale), ptr(k_zero) if ref else None, ptr(v_scale),
                    ptr(v_zero) if ref else None, fmt, ptr(k_rows), ptr(v_rows), _LOGIT_DTYPES[dtype], batch, kv_heads,
                    bs, dim)
    _lib.check(rc, "tierkv_read_rows")
    return k_rows, v_rows


SAMPLE_MAX_VOCAB = 1 << 20   # tierkv_sample_tokens
_LOGIT_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}


def _limit(x, name: str, batch: int, device, dtype, low=None, high=None):
    """A sampling limit: (device tensor or None, value for all rows)."""
    if isinstance(x, torch.Tensor):
        if x.device != device or tuple(x.shape) != (batch,):
            raise ValueError(f"{name} must be a number or one value per row on the logits' device.")
        if dtype == torch.int32 and x.dtype != dtype:
            # To a type that holds the bound, and bounded before it becomes 32 bits; NaN is off.
            x = x.double().nan_to_num(nan=0.0) if x.is_floating_point() else x.long()
            x = x.clamp(0, SAMPLE_MAX_VOCAB)
        return x.to(dtype).contiguous(), 0
    if x != x or (low is not None and x < low) or (high is not None and x > high):
        raise ValueError(f"{name} is out of range.")
    return None, x


def _sampling_limits(uniforms, temperature, top_k, top_p, min_p, batch: int, device):
    """What ``sample_tokens`` asks of its arguments beside the logits: the four
    limits as ``_limit`` gives them."""
    _lib.require_gpu_tensor(uniforms, "uniforms")
    if uniforms.dtype != torch.float32 or tuple(uniforms.shape) != (batch,) or uniforms.device != device:
        raise ValueError("uniforms must be one fp32 number per row on the logits' device.")
    return (_limit(temperature, "temperature", batch, device, torch.float32, low=0.0),
            _limit(top_k, "top_k", batch, device, torch.int32),
            _limit(top_p, "top_p", batch, device, torch.float32, low=0.0),
            _limit(min_p, "min_p", batch, device, torch.float32, low=0.0, high=1.0))


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Next tokens of logits ``[B, vocab]`` (fp16 / bf16 / fp32) with one random
    number in [0, 1) per row (``tierkv_sample_tokens``): temperature, then the
    first ``top_k`` tokens (0: all), of these the smallest set of the likeliest
    that holds ``top_p`` of their probability, of these those at least
    ``min_p`` times as likely as the likeliest; equal logits rank by index.
    The token is the first, in index order, whose running sum of what is left
    exceeds the random number's share.  Each limit is a number or a tensor
    ``[B]``; temperature 0 takes the likeliest token.  Returns (int64 tokens
    [B], fp32 probabilities [B] the tokens were drawn with); a row without a
    logit above -inf gives token -1."""
    lib = _lib.lib()
    _lib.require_gpu_tensor(logits, "logits")
    if logits.ndim != 2 or logits.dtype not in _LOGIT_DTYPES or not logits.numel():
        raise ValueError("logits must be fp16, bf16 or fp32 [batch, vocab].")
    batch, vocab = (int(x) for x in logits.shape)
    device = logits.device
    (t, t_all), (k, k_all), (p, p_all), (m, m_all) = _sampling_limits(uniforms, temperature, top_k, top_p, min_p, batch,
                                                                      device)
    x = logits if logits.stride(1) == 1 and (batch == 1 or logits.stride(0) >= vocab) else logits.contiguous()
    u = uniforms.contiguous()
    tokens = torch.empty(batch, dtype=torch.int64, device=device)
    probs = torch.empty(batch, dtype=torch.float32, device=device)
    need = lib.tierkv_sample_workspace_bytes(batch, vocab)
    ptr = _lib.ptr
    with _lib.call_lock:
        ws = _scratch("sample", device, need, _lib.SAMPLE_COUNTER_BYTES)
        rc = _on_device(device, lib.tierkv_sample_tokens, ptr(x), _LOGIT_DTYPES[x.dtype], x.stride(0), batch, vocab,
                        ptr(u), ptr(t), float(t_all), ptr(k), int(min(max(k_all, 0), SAMPLE_MAX_VOCAB)), ptr(p),
                        float(p_all), ptr(m), float(m_all), ptr(tokens), ptr(probs), ptr(ws), ws.numel())
    _lib.check(rc, "tierkv_sample_tokens")
    return tokens, probs
