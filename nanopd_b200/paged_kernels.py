"""Drop-in for the reference's ``paged_kernels`` extension module, on top of the C ABI.

``paged_attention_forward`` and ``paged_kv_store`` keep the positional signatures the
reference binds (nanoPD/paged_attention/csrc/attention/paged_attention_bindings.cpp:6-14,
nanoPD/paged_attention/csrc/kvstore/paged_kv_store_bindings.cpp:4-11), so
``ModelRunner.paged_forward`` (nanoPD/engine/model_runner.py:94,146,189,270) can import this
module unchanged.  ``paged_prefill_attention`` and ``paged_kv_migrate`` are additions.

Everything launches asynchronously on the current stream of the tensors' device and
returns ``None``; argument errors raise ``RuntimeError`` like the reference's TORCH_CHECKs.
Device-side anomalies (an out-of-range block id, a length beyond the table) never fault:
the kernels skip the access and set a status word that :func:`check_status` reads.
"""
from __future__ import annotations

import ctypes
import math
import struct
import threading
from array import array
from typing import Dict, Optional, Sequence, Tuple

import torch

from . import _lib

_DTYPE_CODE = {torch.float16: _lib.NPD_DTYPE_F16, torch.bfloat16: _lib.NPD_DTYPE_BF16,
               torch.float32: _lib.NPD_DTYPE_F32}

_C = _lib.load()   # raises ImportError when the CUDA library is missing: no fallback path


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


# ---------------------------------------------------------------------------
# Per-(device, stream) workspace.  The reference's split-K op allocates three temporaries
# and syncs on every call (paged_attention_optimized_ops.cu:43-57); here one zeroed buffer
# per device and stream is kept and grown on demand.  Several Python threads, each bound
# to its own GPU, may call in concurrently (nanoPD/router/central_scheduler.py:132-135).
# ---------------------------------------------------------------------------
_ws_lock = threading.Lock()
_workspaces: Dict[Tuple[int, int], torch.Tensor] = {}


def _workspace(device: torch.device, stream_handle: int, nbytes: int) -> torch.Tensor:
    key = (device.index, stream_handle)
    ws = _workspaces.get(key)                 # dict reads are atomic under the GIL: the common case takes no lock
    if ws is not None and ws.numel() >= nbytes:
        return ws
    with _ws_lock:
        ws = _workspaces.get(key)
        if ws is None or ws.numel() < nbytes:
            grown = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)
            if ws is not None:
                grown[:4].copy_(ws[:4])       # carry the status word over, on the device (no host wait)
            _workspaces[key] = ws = grown
        return ws


def release_workspaces(device=None) -> None:
    """Drops the cached per-stream workspaces of ``device`` (default: all devices), e.g. after destroying the
    streams they belonged to.  Synchronises the devices concerned first; the next call on a stream makes a new one."""
    with _ws_lock:
        idx = None if device is None else torch.device(device).index
        keys = [k for k in _workspaces if idx is None or k[0] == idx]
        for d in {k[0] for k in keys}:
            torch.cuda.synchronize(d)
        for k in keys:
            del _workspaces[k]
    scratch_keys = [k for k in list(_scratch) if idx is None or k[0] == idx]
    dropped = []
    for k in scratch_keys + [k for k in list(_captured_scratch) if idx is None or k[0] == idx]:
        with _scratch_lock(*k):                # no call of another thread is between its scratch and its launches
            _scratch_at.pop(k, None)
            dropped.append(_scratch.pop(k, None))
            _captured_scratch.pop(k, None)     # the graph's own pool keeps the memory
    for d in {k[0] for k in scratch_keys}:
        torch.cuda.synchronize(d)              # before the memory goes back
    del dropped


def check_status(device=None, raise_on_error: bool = True) -> int:
    """Reads (and clears) the device-side status words of ``device`` (default: current).

    Returns the OR of the NPD_STATUS_* bits seen since the last call; raises RuntimeError
    for a non-zero word unless ``raise_on_error`` is false.  Synchronises the streams involved.
    """
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    bits = 0
    with _ws_lock:
        items = [(k, w) for k, w in _workspaces.items() if k[0] == idx]
    with torch.cuda.device(idx):
        for (_, stream_handle), ws in items:
            out = ctypes.c_int32(0)
            _lib.check(_C.npd_read_status(ws.data_ptr(), ctypes.byref(out), stream_handle))
            bits |= out.value
            if out.value & _lib.NPD_STATUS_WAIT_TIMEOUT:
                ws.zero_()          # a launch that gave up may have left arrival tickets behind
                torch.cuda.synchronize(idx)
        word = _status_words.get(idx)
        if word is not None:
            torch.cuda.synchronize(idx)         # any stream may have set it
            seen = int(word[0].item())
            if seen:
                bits |= seen
                word.zero_()
                if seen & _lib.NPD_STATUS_WAIT_TIMEOUT:
                    for k in [k for k in list(_scratch) if k[0] == idx]:
                        with _scratch_lock(*k):
                            if k in _scratch:
                                _scratch[k].zero_()
                                torch.cuda.synchronize(idx)
                torch.cuda.synchronize(idx)
    if bits and raise_on_error:
        names = [n for n, b in (("bad block id", 1), ("bad position / seq_len", 2), ("wait time-out", 4)) if bits & b]
        raise RuntimeError("nanopd_b200 device status: " + ", ".join(names))
    return bits


def _stream_handle(device: torch.device) -> int:
    return _raw_stream(device.index)


try:
    _raw_stream = torch._C._cuda_getCurrentRawStream       # the current stream's handle without building a Stream object
except AttributeError:                                     # pragma: no cover
    def _raw_stream(device_index: int) -> int:
        return torch.cuda.current_stream(device_index).cuda_stream


# ---------------------------------------------------------------------------
# Validated call shapes.  The reference's caller is eager and small (at most 16 running sequences,
# nanoPD/engine/engine.py:21), where the host cost of a call matters as much as the kernel.  Every op therefore
# remembers the call shapes it has validated: the key is what the checks look at (shape, strides, dtype and device
# of every tensor, and the integer arguments), the value the scalar arguments of the C call.  A repeated shape skips
# the checks; a new one takes the checks and is remembered if it needed no conversion.
# ---------------------------------------------------------------------------
_PLAN_LIMIT = 1024
_store_plans: Dict[tuple, tuple] = {}
_attn_plans: Dict[tuple, tuple] = {}
_rope_plans: Dict[tuple, tuple] = {}


def _sig(*tensors) -> tuple:
    return tuple([(t.shape, t.stride(), t.dtype, t.device) for t in tensors])


def _remember(table: Dict[tuple, tuple], key: tuple, plan: tuple) -> None:
    if len(table) >= _PLAN_LIMIT:
        table.clear()
    table[key] = plan


def _call(dev_index: int, fn, *args) -> None:
    """The C call with ``dev_index`` current (switching only when it is not)."""
    if torch.cuda.current_device() == dev_index:
        rc = fn(*args)
    else:
        with torch.cuda.device(dev_index):
            rc = fn(*args)
    if rc:
        _lib.check(rc)


def _ws_ptr(dev_index: int, handle: int, nbytes: int):
    ws = _workspaces.get((dev_index, handle))
    if ws is None or ws.numel() < nbytes:
        ws = _workspace(torch.device("cuda", dev_index), handle, nbytes)
    return ws


# ---------------------------------------------------------------------------
# Scratch of the operators below (scored and shared-prefix attention).  Eager calls share one buffer per device and
# stream.  A call that is being captured takes scratch that belongs to its capture (allocated from the graph's own
# pool, cleared by a node of the graph): two graphs captured on one stream may then be replayed side by side.  The
# status bits of all of them go to one word per device, which lives as long as the process.
# Threads may share a stream (all threads of a program begin on the same one): a call holds the stream's lock from the
# choice of its scratch to its last launch.  A shared-prefix call is three launches that hand plan and rows over in the
# scratch, another thread's must not come between them; and a call that needs a larger buffer must not give back the
# one that another call is about to launch on.  One lock per stream: a launch may wait for room in its stream's queue.
# ---------------------------------------------------------------------------
_scratch_locks: Dict[Tuple[int, int], "threading.RLock"] = {}
_scratch: Dict[Tuple[int, int], torch.Tensor] = {}
_scratch_at: Dict[Tuple[int, int], Tuple[int, int]] = {}            # address and size of each, for the common path
_packed_call = _C.npd_call_packed
_pack_scored = struct.Struct("<q6Q2dQ11qQqQqQ").pack           # device, then the entry point's arguments
_pack_scored_prefill = struct.Struct("<q8Qq2dQ10qQqQqQ").pack
_pack_shared = struct.Struct("<q8Qd11qQqQqQ").pack


def _packed_op(op: int, pack, *args) -> None:
    """An operator's entry point, its arguments packed (see npd_call_packed)."""
    try:
        slots = pack(*args)
    except struct.error:
        raise RuntimeError("a number was expected") from None
    rc = _packed_call(op, slots)
    if rc:
        _lib.check(rc)


_capturing = torch._C._cuda_isCurrentStreamCapturing
_current_device = torch._C._cuda_getDevice
_captured_scratch: Dict[Tuple[int, int], Tuple[int, torch.Tensor, int]] = {}     # the stream's latest capture; bytes cleared
_status_words: Dict[int, torch.Tensor] = {}
_status_addresses: Dict[int, int] = {}


def _status_ptr(dev_index: int) -> int:
    address = _status_addresses.get(dev_index)
    if address is None:
        _require(not _capturing(),
                 "call the operator once on this device before capturing it (it allocates its status word on first use)")
        with _ws_lock:
            word = _status_words.get(dev_index)
            if word is None:
                made = torch.zeros(64, dtype=torch.int32, device=torch.device("cuda", dev_index))
                torch.cuda.synchronize(dev_index)            # other streams may write it from now on
                _status_words[dev_index] = word = made
        address = _status_addresses[dev_index] = word.data_ptr()
    return address


def _scratch_lock(dev_index: int, handle: int):
    key = (dev_index, handle)
    lock = _scratch_locks.get(key)
    return lock if lock is not None else _scratch_locks.setdefault(key, threading.RLock())


def _scratch_for(dev_index: int, handle: int, nbytes: int, cleared: int) -> Tuple[int, int]:
    """Address and size of at least ``nbytes`` of scratch for a call on the stream ``handle`` of device ``dev_index``, the first
    ``cleared`` bytes zero when it is first used.  The caller holds the stream's lock until it has launched."""
    key = (dev_index, handle)
    capture_id = 0
    if _capturing() or _current_device() != dev_index:          # the first asks about the current device's stream only
        found = ctypes.c_uint64(0)
        _lib.check(_C.npd_capture_id(handle, ctypes.byref(found)))
        capture_id = found.value
    if capture_id == 0:
        at = _scratch_at.get(key)
        if at is not None and at[1] >= nbytes:
            return at
        with _ws_lock:
            ws = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=torch.device("cuda", dev_index))
            _scratch[key] = ws
            _scratch_at[key] = at = (ws.data_ptr(), ws.numel())
        return at
    held = _captured_scratch.get(key)
    if held is None or held[0] != capture_id or held[1].numel() < nbytes:
        ws, before = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=torch.device("cuda", dev_index)), 0
    else:
        ws, before = held[1], held[2]
    if before < cleared:
        ws[before:cleared].zero_()
        with _ws_lock:
            _captured_scratch[key] = (capture_id, ws, cleared)
    return ws.data_ptr(), ws.numel()


def _cache_geometry(cache: torch.Tensor, name: str):
    _require(cache.dim() == 4, f"{name} must be [num_blocks, num_kv_heads, block_size, head_dim]")
    nb, hkv, bs, d = cache.shape
    _require(cache.stride(3) == 1 and cache.stride(2) == d and cache.stride(1) == bs * d,
             f"{name}: the last three dims must be contiguous")
    return nb, hkv, bs, d, cache.stride(0)


# ---------------------------------------------------------------------------
# (1) KV store
# ---------------------------------------------------------------------------
def paged_kv_store(k_cache, v_cache, k_src, v_src, block_tables, positions) -> None:
    """Scatter new K/V rows into their block slots, in place.

    Same contract as the reference op (nanoPD/paged_attention/csrc/kvstore/paged_kv_store.h:23-27,
    paged_kv_store_ops.cu:7-50): caches ``[blocks, Hkv, B, D]``, sources ``[Hkv, T, D]``,
    ``block_tables`` int32 ``[T, max_blk]`` with one row per token (a stride-0 ``expand`` of a
    single row is accepted as is), ``positions`` int32 ``[T]`` absolute positions.

    The call shape the reference's own tests still use is accepted too
    (tests/test_paged_kernels.py:280,311): sources ``[1, Hkv, T, D]``, a 1-D block table of
    the sequence and an ``int`` start position, meaning token ``t`` sits at ``start + t``.
    """
    key = None
    if type(positions) is not int:
        try:
            key = _sig(k_cache, v_cache, k_src, v_src, block_tables, positions)
        except AttributeError:
            key = None
        plan = _store_plans.get(key) if key is not None else None
        if plan is not None:
            dev_index = plan[0]
            handle = _raw_stream(dev_index)
            _call(dev_index, _C.npd_kv_store, k_cache.data_ptr(), v_cache.data_ptr(), k_src.data_ptr(), v_src.data_ptr(),
                  block_tables.data_ptr(), positions.data_ptr(), *plan[1:], _ws_ptr(dev_index, handle, 256).data_ptr(), handle)
            return
    given = (k_src, v_src, block_tables, positions)
    _require(k_src.is_cuda, "k src is must be on CUDA")
    _require(v_src.is_cuda, "v src is must be on CUDA")
    if k_src.dim() == 4 and k_src.size(0) == 1:
        k_src, v_src = k_src[0], v_src[0]
    _require(k_src.dim() == 3, "k_src must be [num_kv_heads, num_tokens, head_dim]")
    _require(v_src.shape == k_src.shape, "k_src and v_src must have the same shape")
    _require(k_cache.is_cuda and v_cache.is_cuda and k_cache.device == k_src.device == v_cache.device,
             "caches and sources must be on the same CUDA device")
    dev = k_src.device
    hkv, T, d = k_src.shape
    if isinstance(positions, int):
        positions = torch.arange(positions, positions + T, dtype=torch.int32, device=dev)
    if block_tables.dim() == 1:
        block_tables = block_tables.unsqueeze(0).expand(T, -1)
    _require(block_tables.dtype == torch.int32 and positions.dtype == torch.int32,
             "block_tables and positions must be int32")
    _require(block_tables.dim() == 2 and block_tables.size(0) == T and positions.dim() == 1 and positions.numel() == T,
             "block_tables must be [num_tokens, max_blocks] and positions [num_tokens]")
    _require(block_tables.device == dev and positions.device == dev, "index tensors must be on the cache device")
    _require(k_cache.dtype == v_cache.dtype == k_src.dtype == v_src.dtype, "cache and source dtypes differ")
    _require(k_cache.dtype in _DTYPE_CODE, f"unsupported dtype {k_cache.dtype}")
    nb, chkv, bs, cd, cstride = _cache_geometry(k_cache, "k_cache")
    _require(_cache_geometry(v_cache, "v_cache") == (nb, chkv, bs, cd, cstride), "k_cache and v_cache layouts differ")
    _require(chkv == hkv and cd == d, "source heads / head_dim do not match the cache")
    _require(k_src.stride(2) == 1 and v_src.stride(2) == 1, "sources need a contiguous last dim")
    # The stride of a size-1 dimension means nothing (torch leaves whatever the producing view had, e.g. on the
    # decode branch's [Hkv, 1, D] slices, nanoPD/engine/model_runner.py:190-193): only real strides must agree.
    def _strides(t):
        return (t.stride(0) if hkv > 1 else T * d, t.stride(1) if T > 1 else d)
    if _strides(k_src) != _strides(v_src):
        k_src, v_src = k_src.contiguous(), v_src.contiguous()
    src_head_stride, src_token_stride = _strides(k_src)
    if block_tables.stride(1) != 1 and block_tables.size(1) > 1:
        block_tables = block_tables.contiguous()
    if positions.stride(0) != 1:
        positions = positions.contiguous()
    if T == 0:
        return
    plan = (dev.index, T, hkv, d, bs, nb, block_tables.size(1), cstride, src_head_stride, src_token_stride,
            block_tables.stride(0), _DTYPE_CODE[k_cache.dtype])
    if key is not None and all(a is b for a, b in zip(given, (k_src, v_src, block_tables, positions))):
        _remember(_store_plans, key, plan)
    handle = _raw_stream(dev.index)
    _call(dev.index, _C.npd_kv_store, k_cache.data_ptr(), v_cache.data_ptr(), k_src.data_ptr(), v_src.data_ptr(),
          block_tables.data_ptr(), positions.data_ptr(), *plan[1:], _ws_ptr(dev.index, handle, 256).data_ptr(), handle)


# ---------------------------------------------------------------------------
# (1b) fused QK-norm + rotary embedding + KV store
# ---------------------------------------------------------------------------
def paged_qk_norm_rope_store(q, k, v, cos, sin, k_cache, v_cache, block_tables, positions,
                             q_norm_weight=None, k_norm_weight=None, eps: float = 1e-6, q_out=None):
    """Per-head RMSNorm (when weights are given) and rotary embedding of Q and K, K and V written into
    their block slots, in one launch.

    Stands for the passes the reference runs between the projections and the store
    (nanoPD/engine/model_runner.py:97-115, then paged_kv_store at :142-149 / :188-194), with the
    rounding steps of the Hugging Face modules it calls.  ``q`` ``[T, Hq, D]``, ``k``/``v``
    ``[T, Hkv, D]`` token-major (views into a fused projection output are fine: only the last two
    dims must be contiguous); ``cos``/``sin`` ``[T, D]`` (or ``[1, T, D]``) in the tensors' dtype;
    ``block_tables`` int32 one row per token, ``positions`` int32 ``[T]`` as for ``paged_kv_store``.
    Returns the rotated queries ``[T, Hq, D]`` (``q_out``, default: in place over ``q``) — the layout
    ``paged_attention_forward`` and ``paged_prefill_attention`` take.
    """
    if q_out is None:
        q_out = q
    try:
        key = (_sig(q, k, v, cos, sin, k_cache, v_cache, block_tables, positions, q_out),
               None if q_norm_weight is None else _sig(q_norm_weight),
               None if k_norm_weight is None else _sig(k_norm_weight))
    except AttributeError:
        key = None
    plan = _rope_plans.get(key) if key is not None else None
    if plan is not None:
        dev_index = plan[0]
        handle = _raw_stream(dev_index)
        _call(dev_index, _C.npd_qk_norm_rope_store, q_out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
              None if q_norm_weight is None else q_norm_weight.data_ptr(),
              None if k_norm_weight is None else k_norm_weight.data_ptr(),
              cos.data_ptr(), sin.data_ptr(), float(eps), k_cache.data_ptr(), v_cache.data_ptr(),
              block_tables.data_ptr(), positions.data_ptr(), *plan[1:], _ws_ptr(dev_index, handle, 256).data_ptr(), handle)
        return q_out
    given = (cos, sin, block_tables, positions)
    _require(q.is_cuda and k.is_cuda and v.is_cuda, "q, k and v must be on CUDA")
    _require(q.dim() == 3 and k.dim() == 3 and v.dim() == 3, "q must be [T, Hq, D] and k, v [T, Hkv, D]")
    T, hq, d = q.shape
    _require(k.shape == v.shape and k.size(0) == T and k.size(2) == d, "k and v must be [T, Hkv, D] with q's T and D")
    hkv = k.size(1)
    dev = q.device
    if cos.dim() == 3 and cos.size(0) == 1:
        cos, sin = cos[0], sin[0]
    _require(cos.shape == sin.shape and cos.dim() == 2 and cos.size(1) == d and cos.size(0) in (1, T),
             "cos and sin must be [T, D]")
    _require(q_out.shape == q.shape, "q_out must have q's shape")
    for name, t_ in (("q", q), ("k", k), ("v", v), ("q_out", q_out)):
        _require(t_.stride(2) == 1 and t_.stride(1) == d, f"{name}: the last two dims must be contiguous")
    _require(cos.stride(1) == 1 and sin.stride(1) == 1 and cos.stride(0) == sin.stride(0), "cos/sin rows must be contiguous")
    _require(q.dtype in (torch.float16, torch.bfloat16), f"unsupported dtype {q.dtype}")
    _require(all(t_.dtype == q.dtype for t_ in (k, v, cos, sin, q_out, k_cache, v_cache)), "dtypes differ")
    _require(all(t_.device == dev for t_ in (k, v, cos, sin, q_out, k_cache, v_cache, block_tables, positions)),
             "all tensors must be on the same CUDA device")
    for w_ in (q_norm_weight, k_norm_weight):
        _require(w_ is None or (w_.dtype == q.dtype and w_.device == dev and w_.numel() == d and w_.is_contiguous()),
                 "norm weights must be contiguous [D] tensors of q's dtype")
    if block_tables.dim() == 1:
        block_tables = block_tables.unsqueeze(0).expand(T, -1)
    _require(block_tables.dtype == torch.int32 and positions.dtype == torch.int32,
             "block_tables and positions must be int32")
    _require(block_tables.dim() == 2 and block_tables.size(0) == T and positions.dim() == 1 and positions.numel() == T,
             "block_tables must be [num_tokens, max_blocks] and positions [num_tokens]")
    nb, chkv, bs, cd, cstride = _cache_geometry(k_cache, "k_cache")
    _require(_cache_geometry(v_cache, "v_cache") == (nb, chkv, bs, cd, cstride), "k_cache and v_cache layouts differ")
    _require(chkv == hkv and cd == d, "k/v heads / head_dim do not match the cache")
    if block_tables.stride(1) != 1 and block_tables.size(1) > 1:
        block_tables = block_tables.contiguous()
    if positions.stride(0) != 1:
        positions = positions.contiguous()
    if T == 0:
        return q_out
    plan = (dev.index, T, hq, hkv, d, bs, nb, block_tables.size(1), cstride, q.stride(0), k.stride(0), v.stride(0),
            q_out.stride(0), 0 if cos.size(0) == 1 else cos.stride(0), block_tables.stride(0), _DTYPE_CODE[q.dtype])
    if key is not None and all(a is b for a, b in zip(given, (cos, sin, block_tables, positions))):
        _remember(_rope_plans, key, plan)
    handle = _raw_stream(dev.index)
    _call(dev.index, _C.npd_qk_norm_rope_store, q_out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
          None if q_norm_weight is None else q_norm_weight.data_ptr(),
          None if k_norm_weight is None else k_norm_weight.data_ptr(),
          cos.data_ptr(), sin.data_ptr(), float(eps), k_cache.data_ptr(), v_cache.data_ptr(),
          block_tables.data_ptr(), positions.data_ptr(), *plan[1:], _ws_ptr(dev.index, handle, 256).data_ptr(), handle)
    return q_out


# ---------------------------------------------------------------------------
# (2) decode attention
# ---------------------------------------------------------------------------
def paged_attention_forward(out, query, key_cache, value_cache, block_tables, seq_lens,
                            scale: float, block_size: int, max_num_blocks_per_seq: int,
                            _flags: int = 0, max_ctas: int = 0) -> None:
    """``out[s, h] = softmax(scale * q[s, h] . K_s^T) . V_s`` over paged K/V, written in place.

    Same contract as the reference op (nanoPD/paged_attention/csrc/attention/paged_attention.h:24-34,
    paged_attention_ops.cu:7-59): ``out``/``query`` ``[S, Hq, D]`` contiguous, caches
    ``[blocks, Hkv, B, D]``, ``block_tables`` int32 ``[S, max_num_blocks_per_seq]`` zero padded,
    ``seq_lens`` int32 ``[S]``; int64 index tensors raise RuntimeError as they do there
    (pinned by tests/test_paged_kernels.py:218-227).  As in the reference's pointer math
    (paged_attention_kernel.cu:72), row ``s`` of a contiguous table starts at
    ``s * max_num_blocks_per_seq``.

    The interleaved layouts the reference's split-K op and its kernel tests use are accepted under the
    same name (csrc/paged_attention_optimized/paged_attention_optimized_ops.cu:33-34,
    tests/test_paged_kernels.py:39-56): a 5-D ``key_cache`` ``[blocks, Hkv, D/8, B, 8]`` goes with a
    ``value_cache`` ``[blocks, Hkv, D, B]``.

    ``max_ctas`` (an addition, 0 = one CTA per SM) caps the persistent grid so that the call can share the GPU
    with another kernel on a second stream (see ``paged_forward.paged_attention_step``).
    """
    try:
        key = (_sig(out, query, key_cache, value_cache, block_tables, seq_lens), block_size, max_num_blocks_per_seq,
               _flags, max_ctas)
    except AttributeError:
        key = None
    plan = _attn_plans.get(key) if key is not None else None
    if plan is not None:
        dev_index, need, flags = plan[0], plan[1], plan[2]
        handle = _raw_stream(dev_index)
        ws = _ws_ptr(dev_index, handle, need)
        _call(dev_index, _C.npd_paged_decode_attention, out.data_ptr(), query.data_ptr(), key_cache.data_ptr(),
              value_cache.data_ptr(), block_tables.data_ptr(), seq_lens.data_ptr(), float(scale), *plan[3:],
              ws.data_ptr(), ws.numel(), flags, handle)
        return
    _require(query.is_cuda, "query is must be on CUDA")
    _require(query.dim() == 3, "query must be [num seqs, num_heads, head_size]")
    _require(key_cache.dim() in (4, 5), "key_cache must be [num_blocks, num_kv_heads, block_size, head_size] "
                                        "or [num_blocks, num_kv_heads, head_size/8, block_size, 8]")
    interleaved = key_cache.dim() == 5
    _require(block_tables.dtype == torch.int32, "block_tables must be int32")
    _require(seq_lens.dtype == torch.int32, "seq_lens must be int32")
    dev = query.device
    S, hq, d = query.shape
    _require(out.shape == query.shape and out.dtype == query.dtype and out.device == dev,
             "out must match query in shape, dtype and device")
    _require(query.is_contiguous() and out.is_contiguous(), "query and out must be contiguous")
    _require(query.dtype in (torch.float16, torch.bfloat16),
             f"paged_attention_forward supports float16 and bfloat16, got {query.dtype}")
    _require(key_cache.dtype == query.dtype and value_cache.dtype == query.dtype, "cache dtype differs from query")
    _require(key_cache.device == dev and value_cache.device == dev and block_tables.device == dev
             and seq_lens.device == dev, "all tensors must be on the query's device")
    if interleaved:
        nb, hkv, pieces, bs, x = key_cache.shape
        _require(x == 8 and pieces * x == d, "interleaved key_cache must be [blocks, Hkv, head_size/8, block_size, 8]")
        _require(value_cache.dim() == 4 and tuple(value_cache.shape) == (nb, hkv, d, bs),
                 "interleaved value_cache must be [blocks, Hkv, head_size, block_size]")
        _require(key_cache[0].is_contiguous() and value_cache[0].is_contiguous()
                 and key_cache.stride(0) == value_cache.stride(0), "interleaved caches must be contiguous per block")
        cd, cstride = d, key_cache.stride(0)
        _flags = int(_flags) | _lib.NPD_DECODE_KV_INTERLEAVED
    else:
        nb, hkv, bs, cd, cstride = _cache_geometry(key_cache, "key_cache")
        _require(_cache_geometry(value_cache, "value_cache") == (nb, hkv, bs, cd, cstride),
                 "key_cache and value_cache layouts differ")
    _require(cd == d, "head_size of query and cache differ")
    _require(int(block_size) == bs, f"block_size argument {block_size} != cache block size {bs}")
    _require(hq % hkv == 0, "num_heads must be a multiple of num_kv_heads")
    _require(seq_lens.dim() == 1 and seq_lens.numel() == S and seq_lens.stride(0) == 1, "seq_lens must be contiguous [S]")
    max_blk = int(max_num_blocks_per_seq)
    _require(max_blk >= 1, "max_num_blocks_per_seq must be positive")
    if block_tables.dim() == 2 and block_tables.stride(1) == 1 and not block_tables.is_contiguous():
        row_stride = block_tables.stride(0)          # a row-strided view: honour it
        _require(block_tables.size(1) >= max_blk, "block_tables rows shorter than max_num_blocks_per_seq")
    else:
        _require(block_tables.is_contiguous(), "block_tables must be contiguous")
        row_stride = max_blk                         # the reference's flat indexing
        _require(block_tables.numel() >= S * max_blk, "block_tables smaller than num_seqs * max_num_blocks_per_seq")
    if S == 0:
        return
    need = _C.npd_decode_workspace_bytes(S, hq, hkv, d, dev.index)
    flags = int(_flags) | ((int(max_ctas) & 0xffff) << 8)
    plan = (dev.index, need, flags, S, hq, hkv, d, bs, max_blk, nb, cstride, row_stride, _DTYPE_CODE[query.dtype])
    if key is not None:
        _remember(_attn_plans, key, plan)
    handle = _raw_stream(dev.index)
    ws = _ws_ptr(dev.index, handle, need)
    _call(dev.index, _C.npd_paged_decode_attention, out.data_ptr(), query.data_ptr(), key_cache.data_ptr(),
          value_cache.data_ptr(), block_tables.data_ptr(), seq_lens.data_ptr(), float(scale), *plan[3:],
          ws.data_ptr(), ws.numel(), flags, handle)


# ---------------------------------------------------------------------------
# (3) chunked-prefill attention over paged K/V
# ---------------------------------------------------------------------------
def paged_prefill_attention(out, query, key_cache, value_cache, block_tables,
                            chunk_q_offsets: Sequence[int], chunk_tokens: Sequence[int],
                            chunk_starts: Sequence[int], scale: float, block_size: int,
                            max_num_blocks_per_seq: int, _flags: int = 0, max_ctas: int = 0) -> None:
    """Causal attention of prompt chunks over their paged K/V (the chunk's own rows included).

    Replaces the prefill branch of ``paged_forward`` (nanoPD/engine/model_runner.py:152-169).
    ``query``/``out`` are ``[total_tokens, Hq, D]`` with the chunks packed one after another;
    chunk ``c`` occupies rows ``chunk_q_offsets[c] : + chunk_tokens[c]``, its first token sits
    at absolute position ``chunk_starts[c]`` and row ``c`` of ``block_tables`` (int32
    ``[num_chunks, max_num_blocks_per_seq]``) names its pages.  Store the chunk's K/V with
    :func:`paged_kv_store` first, as the caller does (model_runner.py:132-150).
    """
    _require(query.is_cuda and query.dim() == 3, "query must be a CUDA tensor [tokens, num_heads, head_size]")
    _require(block_tables.dtype == torch.int32 and block_tables.dim() == 2, "block_tables must be int32 [chunks, max_blk]")
    dev = query.device
    total, hq, d = query.shape
    nchunks = len(chunk_tokens)
    _require(len(chunk_q_offsets) == nchunks and len(chunk_starts) == nchunks and block_tables.size(0) == nchunks,
             "one offset, token count, start position and table row per chunk")
    _require(out.shape == query.shape and out.dtype == query.dtype and query.is_contiguous() and out.is_contiguous(),
             "out must match query; both contiguous")
    _require(query.dtype in (torch.float16, torch.bfloat16), f"unsupported dtype {query.dtype}")
    nb, hkv, bs, cd, cstride = _cache_geometry(key_cache, "key_cache")
    _require(_cache_geometry(value_cache, "value_cache") == (nb, hkv, bs, cd, cstride), "cache layouts differ")
    _require(cd == d and int(block_size) == bs and key_cache.dtype == query.dtype == value_cache.dtype,
             "cache does not match query")
    _require(block_tables.stride(1) == 1 or block_tables.size(1) == 1, "block_tables rows must be contiguous")
    max_blk = int(max_num_blocks_per_seq)
    _require(1 <= max_blk <= block_tables.size(1), "max_num_blocks_per_seq out of range")
    for off, n, start in zip(chunk_q_offsets, chunk_tokens, chunk_starts):
        _require(n >= 0 and off >= 0 and off + n <= total and start >= 0, "chunk outside the query tensor")
        _require(start + n <= max_blk * bs, "chunk reaches beyond its block table")
    if nchunks == 0 or total == 0:
        return
    arr = ctypes.c_int32 * nchunks
    handle = _stream_handle(dev)
    with torch.cuda.device(dev):
        need = _C.npd_prefill_workspace_bytes(total, hq, hkv, d, dev.index)
        ws = _workspace(dev, handle, need)
        _lib.check(_C.npd_paged_prefill_attention(
            out.data_ptr(), query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
            block_tables.data_ptr(), arr(*chunk_q_offsets), arr(*chunk_tokens), arr(*chunk_starts),
            nchunks, float(scale), hq, hkv, d, bs, max_blk, nb, cstride, block_tables.stride(0),
            _DTYPE_CODE[query.dtype], ws.data_ptr(), ws.numel(),
            int(_flags) | ((int(max_ctas) & 0xffff) << 8), handle))


# ---------------------------------------------------------------------------
# (2c) decode attention with shaped scores
# ---------------------------------------------------------------------------
_scored_plans: Dict[tuple, tuple] = {}


def _score_shape(name: str, score_cap, distance_slopes, window, hq: int, dev) -> None:
    _require(distance_slopes is None or (distance_slopes.dtype == torch.float32 and distance_slopes.device == dev
                                         and distance_slopes.shape == (hq,) and distance_slopes.stride(0) == 1),
             f"{name}: distance_slopes must be a contiguous float32 [num_heads] tensor on the query's device")
    _require(int(window) == window and 0 <= window < 2 ** 31, f"{name}: window must be a whole number, 0 for none")
    _require(math.isfinite(score_cap) and score_cap >= 0, f"{name}: score_cap must be finite and not negative, 0 for none")


def _check_single_token_call(name: str, out, query, key_cache, value_cache, block_tables, seq_lens, block_size, max_num_blocks_per_seq):
    """The checks that the operators for one query token per sequence share; returns
    (device, S, hq, hkv, d, block, blocks, cache stride, table width, table row stride)."""
    _require(query.is_cuda and query.dim() == 3, f"{name}: query must be a CUDA tensor [num_seqs, num_heads, head_size]")
    dev = query.device
    S, hq, d = query.shape
    _require(out.shape == query.shape and out.dtype == query.dtype and out.device == dev and query.is_contiguous() and out.is_contiguous(),
             f"{name}: out must match query in shape, dtype and device; both contiguous")
    _require(query.dtype in (torch.float16, torch.bfloat16), f"{name} supports float16 and bfloat16, got {query.dtype}")
    _require(block_tables.dtype == torch.int32 and seq_lens.dtype == torch.int32, f"{name}: block_tables and seq_lens must be int32")
    _require(key_cache.dtype == query.dtype == value_cache.dtype and all(t.device == dev for t in (key_cache, value_cache, block_tables, seq_lens)),
             f"{name}: caches and tables must match query's dtype and device")
    nb, hkv, bs, cd, cstride = _cache_geometry(key_cache, "key_cache")
    _require(_cache_geometry(value_cache, "value_cache") == (nb, hkv, bs, cd, cstride), "key_cache and value_cache layouts differ")
    _require(cd == d, "head_size of query and cache differ")
    _require(int(block_size) == bs, f"block_size argument {block_size} != cache block size {bs}")
    _require(hq % hkv == 0, "num_heads must be a multiple of num_kv_heads")
    _require(seq_lens.dim() == 1 and seq_lens.numel() == S and (S < 2 or seq_lens.stride(0) == 1), "seq_lens must be contiguous [S]")
    max_blk = int(max_num_blocks_per_seq)
    _require(block_tables.dim() == 2 and block_tables.size(0) == S, f"{name}: block_tables must be [num_seqs, max_blocks]")
    _require(1 <= max_blk <= block_tables.size(1), "max_num_blocks_per_seq out of range")
    _require(block_tables.stride(1) == 1 or block_tables.size(1) == 1, f"{name}: block_tables rows must be contiguous")
    row_stride = block_tables.stride(0) if S > 1 else block_tables.size(1)
    return dev, S, hq, hkv, d, bs, nb, cstride, max_blk, row_stride


def paged_scored_attention(out, query, key_cache, value_cache, block_tables, seq_lens, scale: float, block_size: int,
                           max_num_blocks_per_seq: int, score_cap: float = 0.0, distance_slopes=None, window: int = 0,
                           max_ctas: int = 0) -> None:
    """:func:`paged_attention_forward` with the scores shaped before the softmax, written in place.

    For the query of sequence ``s``, at position ``n - 1`` with ``n = seq_lens[s]``, and key ``j``:
    ``x = scale * q . k_j``; with ``score_cap > 0`` ``x = score_cap * tanh(x / score_cap)``; with ``distance_slopes`` (float32
    ``[num_heads]``) ``x -= distance_slopes[h] * (n - 1 - j)``; over the keys ``max(0, n - window) <= j < n``, all of them with
    ``window == 0``.  Pages wholly before the window are not read and their table entries may be stale.  A sequence of length 0
    gets a zero row.  ``block_tables`` is int32 ``[S, >= max_num_blocks_per_seq]`` with contiguous rows; the other arguments are
    those of :func:`paged_attention_forward` (the interleaved layouts are not taken).
    """
    try:
        # one flat key: what the checks look at (the calls are small, and nested tuples cost as much as the checks)
        key = (out.shape, out.stride(), out.dtype, out.device, query.shape, query.stride(), query.dtype, query.device,
               key_cache.shape, key_cache.stride(), key_cache.dtype, key_cache.device, value_cache.shape, value_cache.stride(),
               value_cache.dtype, value_cache.device, block_tables.shape, block_tables.stride(), block_tables.dtype, block_tables.device,
               seq_lens.shape, seq_lens.stride(), seq_lens.dtype, seq_lens.device, block_size, max_num_blocks_per_seq,
               None if distance_slopes is None else _sig(distance_slopes), score_cap, window, max_ctas)
        plan = _scored_plans.get(key)
    except (AttributeError, TypeError):
        raise RuntimeError("paged_scored_attention takes tensors and numbers") from None
    if plan is None:
        dev, S, hq, hkv, d, bs, nb, cstride, max_blk, row_stride = _check_single_token_call(
            "paged_scored_attention", out, query, key_cache, value_cache, block_tables, seq_lens, block_size, max_num_blocks_per_seq)
        _score_shape("paged_scored_attention", score_cap, distance_slopes, window, hq, dev)
        _require(0 <= int(max_ctas) <= 0xffff, "max_ctas out of range")
        if S == 0:
            return
        need = _C.npd_decode_workspace_bytes(S, hq, hkv, d, dev.index)
        plan = (dev.index, need, min(256 + 4 * S * hq, need), int(max_ctas) << 8, float(score_cap), int(window),
                (S, hq, hkv, d, bs, max_blk, nb, cstride, row_stride, _DTYPE_CODE[query.dtype]))
        _remember(_scored_plans, key, plan)
    dev_index, need, cleared, flags, cap, win, args = plan
    handle = _raw_stream(dev_index)
    with _scratch_lock(dev_index, handle):
        ws, ws_bytes = _scratch_for(dev_index, handle, need, cleared)
        _packed_op(_lib.NPD_OP_SCORED_ATTENTION, _pack_scored,
            dev_index, out.data_ptr(), query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(), seq_lens.data_ptr(),
            scale, cap, 0 if distance_slopes is None else distance_slopes.data_ptr(), win, *args, ws, ws_bytes,
            _status_addresses.get(dev_index) or _status_ptr(dev_index), flags, handle)


# ---------------------------------------------------------------------------
# (2d) decode attention for a batch that shares prefixes
# ---------------------------------------------------------------------------
_shared_plans: Dict[tuple, tuple] = {}
_scored_prefill_plans: Dict[tuple, tuple] = {}


def paged_shared_prefix_attention(out, query, key_cache, value_cache, block_tables, seq_lens, group_offsets, shared_lens,
                                  scale: float, block_size: int, max_num_blocks_per_seq: int, max_ctas: int = 0) -> None:
    """:func:`paged_attention_forward` for a batch whose sequences share the first pages of their tables, written in place.

    Group ``g`` is the sequences ``group_offsets[g] <= s < group_offsets[g + 1]`` (int32 ``[groups + 1]`` on the device, ascending);
    the first ``shared_lens[g]`` tokens (int32 ``[groups]``) of each lie in the same pages: their ``block_tables`` rows agree there
    (those of sequences of length 0 are not read).
    Those pages are read once per group, on the tensor cores, instead of once per sequence.  Sequences outside every group and
    groups of one are attended to as usual, and so is what ``shared_lens`` reaches beyond the shortest non-empty sequence of the
    group.  Lengths, offsets and tables are read on the device, so they may change between replays of a captured call; offsets
    that do not ascend within the batch are reported by :func:`check_status` and share nothing.  ``block_tables`` is int32
    ``[S, >= max_num_blocks_per_seq]`` with contiguous rows, at most 4096 groups; the other arguments are those of
    :func:`paged_attention_forward` (the interleaved layouts are not taken).
    """
    try:
        key = (out.shape, out.stride(), out.dtype, out.device, query.shape, query.stride(), query.dtype, query.device,
               key_cache.shape, key_cache.stride(), key_cache.dtype, key_cache.device, value_cache.shape, value_cache.stride(),
               value_cache.dtype, value_cache.device, block_tables.shape, block_tables.stride(), block_tables.dtype, block_tables.device,
               seq_lens.shape, seq_lens.stride(), seq_lens.dtype, seq_lens.device, group_offsets.shape, group_offsets.stride(),
               group_offsets.dtype, group_offsets.device, shared_lens.shape, shared_lens.stride(), shared_lens.dtype, shared_lens.device,
               block_size, max_num_blocks_per_seq, max_ctas)
        plan = _shared_plans.get(key)
    except (AttributeError, TypeError):
        raise RuntimeError("paged_shared_prefix_attention takes tensors and numbers") from None
    if plan is None:
        name = "paged_shared_prefix_attention"
        dev, S, hq, hkv, d, bs, nb, cstride, max_blk, row_stride = _check_single_token_call(
            name, out, query, key_cache, value_cache, block_tables, seq_lens, block_size, max_num_blocks_per_seq)
        for t, what in ((group_offsets, "group_offsets"), (shared_lens, "shared_lens")):
            _require(t.dtype == torch.int32 and t.device == dev and t.dim() == 1 and (t.numel() < 2 or t.stride(0) == 1),
                     f"{name}: {what} must be a contiguous int32 vector on the query's device")
        groups = shared_lens.numel()
        _require(1 <= groups <= 4096 and group_offsets.numel() == groups + 1,
                 f"{name}: between 1 and 4096 groups, group_offsets one longer than shared_lens")
        _require(0 <= int(max_ctas) <= 0xffff, "max_ctas out of range")
        if S == 0:
            return
        need = _C.npd_shared_prefix_workspace_bytes(S, groups, hq, hkv, d, dev.index)
        plan = (dev.index, need, min(256 + 4 * S * hq, need), int(max_ctas) << 8,
                (S, groups, hq, hkv, d, bs, max_blk, nb, cstride, row_stride, _DTYPE_CODE[query.dtype]))
        _remember(_shared_plans, key, plan)
    dev_index, need, cleared, flags, args = plan
    handle = _raw_stream(dev_index)
    with _scratch_lock(dev_index, handle):
        ws, ws_bytes = _scratch_for(dev_index, handle, need, cleared)
        _packed_op(_lib.NPD_OP_SHARED_PREFIX_ATTENTION, _pack_shared,
            dev_index, out.data_ptr(), query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(), seq_lens.data_ptr(),
            group_offsets.data_ptr(), shared_lens.data_ptr(), scale, *args, ws, ws_bytes, _status_addresses.get(dev_index) or _status_ptr(dev_index), flags, handle)


# ---------------------------------------------------------------------------
# (3b) chunked-prefill attention with shaped scores
# ---------------------------------------------------------------------------
def paged_scored_prefill_attention(out, query, key_cache, value_cache, block_tables, chunk_q_offsets: Sequence[int],
                                   chunk_tokens: Sequence[int], chunk_starts: Sequence[int], scale: float, block_size: int,
                                   max_num_blocks_per_seq: int, score_cap: float = 0.0, distance_slopes=None, window: int = 0,
                                   max_ctas: int = 0) -> None:
    """:func:`paged_prefill_attention` with the scores shaped before the softmax, written in place.

    The shaping is that of :func:`paged_scored_attention`: a query at position ``i`` sees the keys ``i - window < j <= i`` (all up to
    ``i`` with ``window == 0``), its distance to key ``j`` is ``i - j``.  Pages wholly before the window of a chunk's first query are
    not read and their table entries may be stale.  The other arguments are those of :func:`paged_prefill_attention`.
    """
    name = "paged_scored_prefill_attention"
    try:
        offs, toks, starts = array("i", chunk_q_offsets), array("i", chunk_tokens), array("i", chunk_starts)
        key = (out.shape, out.stride(), out.dtype, out.device, query.shape, query.stride(), query.dtype, query.device,
               key_cache.shape, key_cache.stride(), key_cache.dtype, key_cache.device, value_cache.shape, value_cache.stride(),
               value_cache.dtype, value_cache.device, block_tables.shape, block_tables.stride(), block_tables.dtype, block_tables.device,
               block_size, max_num_blocks_per_seq, None if distance_slopes is None else _sig(distance_slopes), score_cap, window, max_ctas)
        plan = _scored_prefill_plans.get(key)
        if plan is None:
            _require(query.is_cuda and query.dim() == 3, f"{name}: query must be a CUDA tensor [tokens, num_heads, head_size]")
            _require(block_tables.dtype == torch.int32 and block_tables.dim() == 2, f"{name}: block_tables must be int32 [chunks, max_blk]")
            dev = query.device
            _, hq, d = query.shape
            _require(out.shape == query.shape and out.dtype == query.dtype and out.device == dev and query.is_contiguous() and out.is_contiguous(),
                     f"{name}: out must match query in shape, dtype and device; both contiguous")
            _require(query.dtype in (torch.float16, torch.bfloat16), f"{name}: unsupported dtype {query.dtype}")
            nb, hkv, bs, cd, cstride = _cache_geometry(key_cache, "key_cache")
            _require(_cache_geometry(value_cache, "value_cache") == (nb, hkv, bs, cd, cstride), "cache layouts differ")
            _require(cd == d and int(block_size) == bs and key_cache.dtype == query.dtype == value_cache.dtype, f"{name}: cache does not match query")
            _require(all(t.device == dev for t in (key_cache, value_cache, block_tables)), f"{name}: all tensors must be on the query's device")
            _require(hq % hkv == 0, "num_heads must be a multiple of num_kv_heads")
            _require(block_tables.stride(1) == 1 or block_tables.size(1) == 1, "block_tables rows must be contiguous")
            max_blk = int(max_num_blocks_per_seq)
            _require(1 <= max_blk <= block_tables.size(1), "max_num_blocks_per_seq out of range")
            _require(0 <= int(max_ctas) <= 0xffff, "max_ctas out of range")
            _score_shape(name, score_cap, distance_slopes, window, hq, dev)
            row_stride = block_tables.stride(0) if block_tables.size(0) > 1 else block_tables.size(1)
            plan = (dev.index, query.size(0), max_blk * bs, block_tables.size(0), float(score_cap), int(window),
                    (hq, hkv, d, bs, max_blk, nb, cstride, row_stride, _DTYPE_CODE[query.dtype]), int(max_ctas) << 8)
            _remember(_scored_prefill_plans, key, plan)
    except (AttributeError, TypeError, OverflowError):
        raise RuntimeError(f"{name} takes tensors, lists of whole numbers and numbers") from None
    dev_index, total, capacity, rows, cap, win, args, flags = plan
    nchunks = len(toks)
    _require(len(offs) == nchunks and len(starts) == nchunks and rows == nchunks,
             f"{name}: one offset, token count, start position and table row per chunk")
    for off, n, start in zip(offs, toks, starts):
        if n < 0 or off < 0 or off + n > total or start < 0:
            raise RuntimeError(f"{name}: chunk outside the query tensor")
        if start + n > capacity:
            raise RuntimeError(f"{name}: chunk reaches beyond its block table")
    if nchunks == 0 or total == 0:
        return
    handle = _raw_stream(dev_index)
    with _scratch_lock(dev_index, handle):
        ws, ws_bytes = _scratch_for(dev_index, handle, 256, 256)
        _packed_op(_lib.NPD_OP_SCORED_PREFILL_ATTENTION, _pack_scored_prefill,
            dev_index, out.data_ptr(), query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(),
            offs.buffer_info()[0], toks.buffer_info()[0], starts.buffer_info()[0], nchunks, scale, cap,
            0 if distance_slopes is None else distance_slopes.data_ptr(), win, *args, ws, ws_bytes,
            _status_addresses.get(dev_index) or _status_ptr(dev_index), flags, handle)


# ---------------------------------------------------------------------------
# (4) KV page migration
# ---------------------------------------------------------------------------
def _pool_geometry(pool: torch.Tensor, name: str):
    _require(pool.dim() == 5, f"{name} must be [layers, blocks, num_kv_heads, block_size, head_dim]")
    L, nb = pool.shape[:2]
    block_elems = pool.shape[2] * pool.shape[3] * pool.shape[4]
    _require(pool[0, 0].is_contiguous(), f"{name}: a block must be contiguous")
    return L, nb, block_elems, pool.stride(0), pool.stride(1)


def _block_list(ids, dev: torch.device) -> torch.Tensor:
    """A block list as an int32 tensor on ``dev``.  A Python list goes through pinned host memory and a
    non-blocking copy on the current stream, so the calling thread never waits behind work already queued on
    that stream (a pageable source would make the copy synchronous with the stream's earlier work)."""
    if torch.is_tensor(ids):
        return ids
    host = torch.tensor(list(ids), dtype=torch.int32)
    if host.numel() == 0:
        return host.to(dev)
    return host.pin_memory().to(dev, non_blocking=True)


def paged_kv_migrate(src_k, src_v, dst_k, dst_v, src_blocks, dst_blocks=None, max_ctas: int = 0) -> None:
    """Copy blocks ``src_blocks[i] -> dst_blocks[i]`` of every layer between two 5-D pools.

    One kernel on the current stream of the CURRENT device, which must be able to address
    both pools (same device, or peer access enabled — see ``kv_transfer.transfer_kv``).  One of the
    two pools may be a PINNED host buffer (``kv_transfer.PinnedKVBuffer``): the kernel then reads or writes
    it over PCIe through the unified address space with plain loads and stores.
    ``src_blocks``/``dst_blocks``: int32 tensors on the current device, or Python lists, which are staged in
    pinned memory and copied there without blocking the host.  ``max_ctas`` > 0 caps the grid of the
    bulk-copy kernel (one warp per CTA; 0 = 64 CTAs) so a side-stream migration leaves the SMs to compute; a
    negative value selects the plain load/store kernel with that many CTAs.
    """
    dev = torch.device("cuda", torch.cuda.current_device())
    L, snb, belems, sls, sbs = _pool_geometry(src_k, "src_k")
    _require(_pool_geometry(src_v, "src_v") == (L, snb, belems, sls, sbs), "src_k and src_v layouts differ")
    L2, dnb, belems2, dls, dbs = _pool_geometry(dst_k, "dst_k")
    _require(_pool_geometry(dst_v, "dst_v") == (L2, dnb, belems2, dls, dbs), "dst_k and dst_v layouts differ")
    _require(L == L2 and belems == belems2 and src_k.dtype == dst_k.dtype == src_v.dtype == dst_v.dtype,
             "source and destination pools differ in layers, block shape or dtype")
    for name, pool in (("src_k", src_k), ("src_v", src_v), ("dst_k", dst_k), ("dst_v", dst_v)):
        _require(pool.is_cuda or pool.is_pinned(), f"{name} must be a CUDA tensor or a pinned host tensor")
    _require(src_k.is_cuda or dst_k.is_cuda, "one of the two pools must be on a GPU")
    src_blocks = _block_list(src_blocks, dev)
    dst_blocks = src_blocks if dst_blocks is None else _block_list(dst_blocks, dev)
    _require(src_blocks.dtype == torch.int32 and dst_blocks.dtype == torch.int32, "block lists must be int32")
    _require(src_blocks.device == dev and dst_blocks.device == dev, "block lists must live on the current device")
    _require(src_blocks.numel() == dst_blocks.numel() and src_blocks.is_contiguous() and dst_blocks.is_contiguous(),
             "block lists must be contiguous and of equal length")
    n = src_blocks.numel()
    if n == 0:
        return
    handle = _stream_handle(dev)
    ws = _workspace(dev, handle, 256)
    _lib.check(_C.npd_kv_migrate(
        src_k.data_ptr(), src_v.data_ptr(), dst_k.data_ptr(), dst_v.data_ptr(),
        src_blocks.data_ptr(), dst_blocks.data_ptr(), n, L, belems, src_k.element_size(),
        sls, sbs, snb, dls, dbs, dnb, int(max_ctas), ws.data_ptr(), handle))


def enable_peer_access(peer_device: int) -> None:
    """Map ``peer_device``'s memory into the current device (idempotent)."""
    _lib.check(_C.npd_enable_peer_access(int(peer_device)))
