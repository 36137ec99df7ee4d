"""Tensor-level wrappers over the libkvoff C ABI.

Every function enqueues work on a CUDA stream (default: the current stream of
the pool's device) and never synchronizes the host. Slots are addressed by raw
pointers so that one call can target pinned host slabs, their device aliases
(zero-copy) or device staging buffers.
"""

from __future__ import annotations

import ctypes
import math
import struct
from dataclasses import dataclass

import torch

from kvoff import _lib
from kvoff._lib import COPY_ENGINE, COPY_SM, COPY_TMA  # noqa: F401  (re-exported)


@dataclass(frozen=True)
class PoolGeometry:
    """Geometry of a paged pool [2, L, NB, BS, H, D] (strides in elements).

    Chunk c = kv * L + layer of block b starts at c * chunk_stride +
    b * block_stride and holds rows_per_chunk = BS * H dense rows of D.
    """

    num_chunks: int
    chunk_stride: int
    block_stride: int
    num_blocks: int
    rows_per_chunk: int
    head_dim: int
    elem_size: int

    @property
    def rows(self) -> int:
        return self.num_chunks * self.rows_per_chunk

    @property
    def chunk_bytes(self) -> int:
        return self.rows_per_chunk * self.head_dim * self.elem_size

    @property
    def block_bytes(self) -> int:
        """Raw (BF16-mode) bytes of one block."""
        return self.num_chunks * self.chunk_bytes

    @property
    def fp8_payload_bytes(self) -> int:
        return self.rows * self.head_dim

    @property
    def fp8_scale_bytes(self) -> int:
        return self.rows * 2


def geometry(pool: torch.Tensor) -> PoolGeometry:
    """Validate a pool's layout and return its geometry."""
    if pool.ndim != 6 or pool.shape[0] != 2 or min(pool.shape) <= 0:
        raise ValueError("KV pool must be a non-empty [2, L, NB, BS, H, D] tensor")
    _, layers, num_blocks, block_size, heads, dim = pool.shape
    s = pool.stride()
    if s[5] != 1 or s[4] != dim or s[3] != heads * dim:
        raise ValueError("each KV block chunk [BS, H, D] must be dense")
    if layers > 1 and s[0] != layers * s[1]:
        raise ValueError("(K/V, layer) chunks of the pool must be evenly strided")
    chunk_stride = s[1] if layers > 1 else s[0]
    return PoolGeometry(2 * layers, chunk_stride, s[2], num_blocks, block_size * heads, dim,
                        pool.element_size())


def _stream(device: torch.device, stream) -> int:
    if stream is None:
        stream = torch.cuda.current_stream(device)
    return int(stream.cuda_stream) if hasattr(stream, "cuda_stream") else int(stream)


def _require_cuda(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")


def _require_bf16(pool: torch.Tensor) -> None:
    if pool.dtype != torch.bfloat16:
        raise ValueError("the FP8 codec quantizes bf16 KV pools")


def save_fp8(pool: torch.Tensor, block_ids, payload_ptrs, scale_ptrs, *, stream=None,
             max_ctas: int = 0) -> None:
    """Quantize blocks into device-accessible slots (device staging or mapped host)."""
    _require_cuda(pool, "pool")
    _require_bf16(pool)
    g = geometry(pool)
    n = len(block_ids)
    if len(payload_ptrs) != n or len(scale_ptrs) != n:
        raise ValueError("one payload and scale pointer per block")
    with torch.cuda.device(pool.device):
        _lib.call("kvoff_fp8_save_blocks", pool.data_ptr(), g.num_chunks, g.chunk_stride,
                  g.block_stride, g.num_blocks, g.rows_per_chunk, g.head_dim,
                  _lib.int64_array(block_ids), n, _lib.pointer_array(payload_ptrs),
                  _lib.pointer_array(scale_ptrs), max_ctas, _stream(pool.device, stream))


def restore_fp8(pool: torch.Tensor, block_ids, payload_ptrs, scale_ptrs, *, stream=None,
                max_ctas: int = 0) -> None:
    """Dequantize device-accessible slots into pool blocks."""
    _require_cuda(pool, "pool")
    _require_bf16(pool)
    g = geometry(pool)
    n = len(block_ids)
    if len(payload_ptrs) != n or len(scale_ptrs) != n:
        raise ValueError("one payload and scale pointer per block")
    with torch.cuda.device(pool.device):
        _lib.call("kvoff_fp8_restore_blocks", pool.data_ptr(), g.num_chunks, g.chunk_stride,
                  g.block_stride, g.num_blocks, g.rows_per_chunk, g.head_dim,
                  _lib.int64_array(block_ids), n, _lib.pointer_array(payload_ptrs),
                  _lib.pointer_array(scale_ptrs), max_ctas, _stream(pool.device, stream))


def _staging_blocks(g: PoolGeometry, staging_payload: torch.Tensor,
                    staging_scale: torch.Tensor) -> int:
    _require_cuda(staging_payload, "staging payload")
    _require_cuda(staging_scale, "staging scale")
    count = min(staging_payload.numel() * staging_payload.element_size() // g.fp8_payload_bytes,
                staging_scale.numel() * staging_scale.element_size() // g.fp8_scale_bytes)
    if count < 1:
        raise ValueError("staging buffers hold less than one block")
    return count


def _event(event) -> int:
    """Raw cudaEvent_t of a recorded torch.cuda.Event (or a raw handle)."""
    handle = int(getattr(event, "cuda_event", event))
    if handle == 0:  # torch creates the CUDA event on its first record
        raise ValueError("pass an event that has been recorded at least once")
    return handle


def save_fp8_staged(pool: torch.Tensor, block_ids, host_payload_ptrs, host_scale_ptrs,
                    staging_payload: torch.Tensor, staging_scale: torch.Tensor, *,
                    stream=None, wait_events=None, source_done=None) -> None:
    """Quantize into device staging, then cudaMemcpyAsync each slot to pinned host.

    By default the quantize kernels follow all earlier work on `stream`. With
    `wait_events` (recorded torch.cuda.Events) they follow only those, so they
    can overlap the host copies of earlier calls; `source_done` is re-recorded
    once the kernels have read every pool block of the call.
    """
    _require_cuda(pool, "pool")
    _require_bf16(pool)
    g = geometry(pool)
    n = len(block_ids)
    if len(host_payload_ptrs) != n or len(host_scale_ptrs) != n:
        raise ValueError("one payload and scale pointer per block")
    staged = _staging_blocks(g, staging_payload, staging_scale)
    common = (pool.data_ptr(), g.num_chunks, g.chunk_stride, g.block_stride, g.num_blocks,
              g.rows_per_chunk, g.head_dim, _lib.int64_array(block_ids), n,
              _lib.pointer_array(host_payload_ptrs), _lib.pointer_array(host_scale_ptrs),
              staging_payload.data_ptr(), staging_scale.data_ptr(), staged)
    with torch.cuda.device(pool.device):
        if wait_events is None and source_done is None:
            _lib.call("kvoff_fp8_save_blocks_staged", *common, _stream(pool.device, stream))
            return
        waits = [_event(e) for e in (wait_events or ())]
        _lib.call("kvoff_fp8_save_blocks_staged_ev", *common,
                  _lib.pointer_array(waits) if waits else None, len(waits),
                  _event(source_done) if source_done is not None else None,
                  _stream(pool.device, stream))


def restore_fp8_staged(pool: torch.Tensor, block_ids, host_payload_ptrs, host_scale_ptrs,
                       staging_payload: torch.Tensor, staging_scale: torch.Tensor, *,
                       stream=None, done_event=None) -> None:
    """cudaMemcpyAsync each pinned slot into device staging, then dequantize.

    By default `stream` waits for the dequantize kernels before it returns to
    the caller's later work. With `done_event` (a recorded torch.cuda.Event)
    the event is re-recorded after the last pool write instead and `stream` is
    left free to start the next call's copies; order readers on the event, or
    call join_pipeline(stream) before synchronizing `stream`.
    """
    _require_cuda(pool, "pool")
    _require_bf16(pool)
    g = geometry(pool)
    n = len(block_ids)
    if len(host_payload_ptrs) != n or len(host_scale_ptrs) != n:
        raise ValueError("one payload and scale pointer per block")
    staged = _staging_blocks(g, staging_payload, staging_scale)
    common = (pool.data_ptr(), g.num_chunks, g.chunk_stride, g.block_stride, g.num_blocks,
              g.rows_per_chunk, g.head_dim, _lib.int64_array(block_ids), n,
              _lib.pointer_array(host_payload_ptrs), _lib.pointer_array(host_scale_ptrs),
              staging_payload.data_ptr(), staging_scale.data_ptr(), staged)
    with torch.cuda.device(pool.device):
        if done_event is None:
            _lib.call("kvoff_fp8_restore_blocks_staged", *common, _stream(pool.device, stream))
        else:
            _lib.call("kvoff_fp8_restore_blocks_staged_ev", *common, _event(done_event),
                      _stream(pool.device, stream))


def _fp8_staged_ev(save: bool, g: PoolGeometry, pool_ptr: int, block_ids, payload_ptrs,
                   scale_ptrs, staging_payload_ptr: int, staging_scale_ptr: int,
                   staging_blocks: int, stream: int, wait_events=(), event: int = 0) -> None:
    """Lean form of save_fp8_staged / restore_fp8_staged for a caller that
    already holds a checked geometry, raw pointers, raw stream and event
    handles, and has the pool's device current (the drop-in cache's per-block
    path, which runs once per saved or restored block on the engine thread).

    Save: the kernels wait for `wait_events` (none: all earlier work on the
    stream) and `event`, when non-zero, is recorded once the pool blocks are
    read. Restore: `event`, when non-zero, is recorded after the last pool
    write and the stream is not joined (see restore_fp8_staged).
    """
    so = _lib.lib()
    n = len(block_ids)
    ids = (ctypes.c_int64 * n)(*block_ids)
    payload = (ctypes.c_void_p * n)(*payload_ptrs)
    scale = (ctypes.c_void_p * n)(*scale_ptrs)
    if save:
        waits = (ctypes.c_void_p * max(1, len(wait_events)))(*wait_events)
        rc = so.kvoff_fp8_save_blocks_staged_ev(
            pool_ptr, g.num_chunks, g.chunk_stride, g.block_stride, g.num_blocks,
            g.rows_per_chunk, g.head_dim, ids, n, payload, scale, staging_payload_ptr,
            staging_scale_ptr, staging_blocks, waits, len(wait_events), event or None, stream)
        _lib.check(rc, "kvoff_fp8_save_blocks_staged_ev")
    else:
        rc = so.kvoff_fp8_restore_blocks_staged_ev(
            pool_ptr, g.num_chunks, g.chunk_stride, g.block_stride, g.num_blocks,
            g.rows_per_chunk, g.head_dim, ids, n, payload, scale, staging_payload_ptr,
            staging_scale_ptr, staging_blocks, event or None, stream)
        _lib.check(rc, "kvoff_fp8_restore_blocks_staged_ev")


def join_pipeline(device, stream=None) -> None:
    """Make `stream` wait for the staged calls' kernels queued on its behalf."""
    device = torch.device(device)
    with torch.cuda.device(device):
        _lib.call("kvoff_stream_join_pipeline", _stream(device, stream))


def copy_blocks(pool: torch.Tensor, block_ids, slot_ptrs, *, restore: bool = False,
                method: int = COPY_ENGINE, stream=None, max_ctas: int = 0) -> None:
    """Byte-exact block moves pool <-> dense slots (BF16 passthrough)."""
    _require_cuda(pool, "pool")
    g = geometry(pool)
    e = g.elem_size
    n = len(block_ids)
    if len(slot_ptrs) != n:
        raise ValueError("one slot pointer per block")
    with torch.cuda.device(pool.device):
        _lib.call("kvoff_copy_blocks", pool.data_ptr(), g.num_chunks, g.chunk_stride * e,
                  g.block_stride * e, g.num_blocks, g.chunk_bytes, _lib.int64_array(block_ids), n,
                  _lib.pointer_array(slot_ptrs), _lib.RESTORE if restore else _lib.SAVE, method,
                  max_ctas, _stream(pool.device, stream))


def copy_blocks_staged(pool: torch.Tensor, block_ids, host_slot_ptrs, staging: torch.Tensor, *,
                       restore: bool = False, stream=None, wait_events=(), event=None) -> None:
    """Byte-exact block moves pool <-> pinned host slots through device staging.

    staging is a [n, block_bytes] uint8 device buffer; with n >= 2 the gather /
    scatter kernels of one half overlap the DMA of the other (a library-owned
    kernel stream; see join_pipeline). Save: the kernels wait for wait_events
    (recorded torch.cuda.Events; none: earlier work on the stream) and `event`
    is recorded once the pool blocks are read. Restore: `event` is recorded
    after the last pool write and the stream is not joined; without it the
    stream waits for the kernels.
    """
    _require_cuda(pool, "pool")
    _require_cuda(staging, "staging")
    g = geometry(pool)
    n = len(block_ids)
    if len(host_slot_ptrs) != n:
        raise ValueError("one slot pointer per block")
    if staging.dtype != torch.uint8 or staging.dim() != 2 or staging.shape[1] != g.block_bytes:
        raise ValueError(f"staging must be uint8 [n, {g.block_bytes}]")
    if restore and wait_events:
        raise ValueError("wait_events apply to saves only")
    with torch.cuda.device(pool.device):
        _copy_staged_ev(not restore, g, pool.data_ptr(), block_ids, host_slot_ptrs,
                        staging.data_ptr(), staging.shape[0], _stream(pool.device, stream),
                        [_event(e) for e in wait_events], _event(event) if event is not None else 0)


def _copy_staged_ev(save: bool, g: PoolGeometry, pool_ptr: int, block_ids, slot_ptrs,
                    staging_ptr: int, staging_blocks: int, stream: int, wait_events=(),
                    event: int = 0) -> None:
    """Lean form of copy_blocks_staged for the drop-in cache's per-block path
    (checked geometry, raw pointers, stream and event handles, the pool's
    device current)."""
    n = len(block_ids)
    ids = (ctypes.c_int64 * n)(*block_ids)
    slots = (ctypes.c_void_p * n)(*slot_ptrs)
    waits = (ctypes.c_void_p * max(1, len(wait_events)))(*wait_events)
    e = g.elem_size
    rc = _lib.lib().kvoff_copy_blocks_staged(
        pool_ptr, g.num_chunks, g.chunk_stride * e, g.block_stride * e, g.num_blocks,
        g.chunk_bytes, ids, n, slots, staging_ptr, staging_blocks,
        _lib.SAVE if save else _lib.RESTORE, waits, len(wait_events), event or None, stream)
    _lib.check(rc, "kvoff_copy_blocks_staged")


def copy_tokens(pool: torch.Tensor, block_ids, num_tokens: int, dense_ptr: int, *,
                restore: bool = False, stream=None) -> None:
    """Tokens [0, num_tokens) of a sequence's blocks <-> dense [2, L, num_tokens, H, D]."""
    _require_cuda(pool, "pool")
    g = geometry(pool)
    block_size = pool.shape[3]
    token_bytes = pool.shape[4] * pool.shape[5] * g.elem_size
    needed = -(-num_tokens // block_size)
    if len(block_ids) < needed:
        raise ValueError("sequence is missing KV blocks")
    with torch.cuda.device(pool.device):
        _lib.call("kvoff_copy_tokens", pool.data_ptr(), g.num_chunks, g.chunk_stride * g.elem_size,
                  g.block_stride * g.elem_size, g.num_blocks, block_size, token_bytes,
                  _lib.int64_array(block_ids[:needed]), int(num_tokens), int(dense_ptr),
                  _lib.RESTORE if restore else _lib.SAVE, _stream(pool.device, stream))


def memcpy(dst_ptr: int, src_ptr: int, nbytes: int, *, device, stream=None) -> None:
    """cudaMemcpyAsync(cudaMemcpyDefault) on `stream`."""
    device = torch.device(device)
    with torch.cuda.device(device):
        _lib.call("kvoff_memcpy", int(dst_ptr), int(src_ptr), int(nbytes), _stream(device, stream))


_raw_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _fast_stream(device: torch.device, stream) -> int:
    """Raw handle of `stream`, or of the device's current stream (cheap path)."""
    if stream is None and _raw_current_stream is not None:
        return _raw_current_stream(device.index)
    return _stream(device, stream)


def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, slot_mapping: torch.Tensor, *,
                  bad_slots: torch.Tensor | None = None, stream=None) -> None:
    """Write row i of key/value [N, H, D] to cache slot slot_mapping[i] (-1: skip).

    Same contract as nanovllm/layers/attention.py:33-40 (including its layout
    assertions); the scatter is one CUDA-graph-capturable kernel launch. This
    runs once per layer per forward, so the host path is kept short: one
    stride tuple per tensor, the raw current-stream handle, and a device
    switch only when the tensors live on another device than the current one.
    """
    num_tokens, num_heads, head_dim = key.shape
    row = num_heads * head_dim
    ks, vs = key.stride(), value.stride()
    if ks[2] != 1 or vs[2] != 1:
        raise AssertionError("key/value last dim must be contiguous")
    if ks[1] != head_dim or vs[1] != head_dim:
        raise AssertionError("key/value heads must be dense")
    if k_cache.stride(1) != row or v_cache.stride(1) != row:
        raise AssertionError("cache slots must hold dense [H, D] rows")
    if slot_mapping.numel() != num_tokens:
        raise AssertionError("one slot per token")
    if value.shape != key.shape:
        raise ValueError("key and value shapes differ")
    dtype = key.dtype
    if value.dtype != dtype or k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise ValueError("key, value and caches must share a dtype")
    if slot_mapping.dtype != torch.int32:
        raise ValueError("slot_mapping must be int32")
    if not (key.is_cuda and value.is_cuda and k_cache.is_cuda and v_cache.is_cuda
            and slot_mapping.is_cuda):
        raise ValueError("key, value, caches and slot_mapping must be CUDA tensors")
    if bad_slots is not None and (bad_slots.dtype != torch.int32 or not bad_slots.is_cuda):
        raise ValueError("bad_slots must be a CUDA int32 tensor")
    e = key.element_size()
    num_slots = k_cache.numel() // row if row else 0
    device = key.device
    args = (key.data_ptr(), ks[0] * e, value.data_ptr(), vs[0] * e, k_cache.data_ptr(),
            v_cache.data_ptr(), row * e, slot_mapping.data_ptr(), num_tokens, num_slots,
            bad_slots.data_ptr() if bad_slots is not None else None)
    if device.index == torch.cuda.current_device():
        status = _store_fn()(*args, _fast_stream(device, stream))
    else:
        with torch.cuda.device(device):
            status = _store_fn()(*args, _fast_stream(device, stream))
    if status:
        _lib.check(status, "kvoff_store_kvcache")


_STORE = None


def _store_fn():
    global _STORE
    if _STORE is None:
        _STORE = _lib.lib().kvoff_store_kvcache
    return _STORE


# ---------------------------------------------------------------------------
# Rotary positions, the e4m3 paged cache and attention over it
#
# A layer's three calls, in order: rotary(q, k), store_kvcache_fp8(k, v) and
# attention_fp8(q). Like store_kvcache they run once per layer per forward, so
# their host paths are kept short.

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16, torch.float32: _lib.FP32}
_FP8 = torch.float8_e4m3fn


# Argument arrays of the packed entry points (include/kvoff.h): one foreign
# argument instead of twenty, 6 us less a call.
_ROTARY_ARGS = struct.Struct("21q").pack
_STORE_ARGS = struct.Struct("17q").pack
_ATTENTION_ARGS = struct.Struct("24qd3q").pack
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_ENTRIES: dict = {}


def _entry(name: str):
    fn = _ENTRIES.get(name)
    if fn is None:
        fn = _ENTRIES[name] = getattr(_lib.lib(), name)
    return fn


def _launch(name: str, args: bytes, index: int) -> None:
    """Call packed entry point `name` on device `index` and raise KvoffError on a failure."""
    if index == _current_device():
        status = _entry(name)(args)
    else:
        with torch.cuda.device(index):
            status = _entry(name)(args)
    if status:
        _lib.check(status, name)


def _raw_stream(index: int, stream) -> int:
    if stream is None and _raw_current_stream is not None:
        return _raw_current_stream(index)
    return _stream(torch.device("cuda", index), stream)


_ONE_DEVICE = "the tensors must be CUDA tensors on one device"
_NO_GRADIENT = "autograd does not see this call: use torch.no_grad(), or detach the inputs"
_grad_enabled = torch.is_grad_enabled


def _one_device(index: int, *tensors) -> None:
    """Refuse tensors that are not all on CUDA device `index` (-1: the first is not on any)."""
    for t in tensors:
        if index < 0 or t.get_device() != index:
            raise ValueError(_ONE_DEVICE)


def _rows(x: torch.Tensor, what: str, size: int = 2) -> int:
    """Bytes from one token to the next of x [N, H, D] with dense heads of `size`-byte values."""
    token, head, value = x.stride()
    tokens, heads, dim = x.shape
    if (value != 1 and dim > 1) or (head != dim and heads > 1):
        raise ValueError(f"the heads of {what} must be dense")
    return (token if tokens > 1 else heads * dim) * size  # a stride of one row means nothing


def rotary_table(positions: int, rotary_dim: int, *, base: float = 10000.0,
                 scaling: dict | None = None, device=None) -> torch.Tensor:
    """Cosines and sines of the first `positions` positions, for `rotary`.

    Returns fp32 [positions, rotary_dim]: row p holds cos(p * f_j), then
    sin(p * f_j), of the rotary_dim / 2 pairs, f_j = base^(-2j / rotary_dim).
    Angles are formed in 64 bits. `scaling` stretches the frequencies for
    contexts longer than the model was trained on; its "type" is one of

    * "linear": f_j / factor;
    * "ntk": the base grows to base * factor^(R / (R - 2)), R = rotary_dim;
    * "yarn": f_j / factor for pairs that turn less than beta_slow (1) times
      over original_max_position_embeddings, f_j for those that turn more than
      beta_fast (32) times, a linear ramp over the pair index between; cosines
      and sines carry attention_factor (0.1 ln(factor) + 1);
    * "llama3": f_j / factor for pairs that turn less than low_freq_factor (1)
      times over original_max_position_embeddings, f_j for those that turn more
      than high_freq_factor (4) times, a linear blend over the turns between.
    """
    if rotary_dim <= 0 or rotary_dim % 2 or positions < 0:
        raise ValueError("rotary_dim must be even and positive, positions not negative")
    half = rotary_dim // 2
    scaling = dict(scaling or {})
    kind = scaling.pop("type", scaling.pop("rope_type", "none"))
    known = {"none": (), "linear": ("factor",), "ntk": ("factor",),
             "yarn": ("factor", "original_max_position_embeddings", "beta_fast", "beta_slow",
                      "attention_factor"),
             "llama3": ("factor", "original_max_position_embeddings", "low_freq_factor",
                        "high_freq_factor")}
    if kind not in known:
        raise ValueError(f"unknown rotary scaling {kind!r}")
    unknown = set(scaling) - set(known[kind])
    if unknown:
        raise ValueError(f"rotary scaling {kind!r} does not know {sorted(unknown)}")
    if kind != "none" and not float(scaling.get("factor", 0.0)) >= 1.0:
        raise ValueError(f"rotary scaling {kind!r} needs a factor of 1 or more")
    if kind in ("yarn", "llama3") and not scaling.get("original_max_position_embeddings", 0) > 0:
        raise ValueError(f"rotary scaling {kind!r} needs original_max_position_embeddings")
    factor = float(scaling.get("factor", 1.0))
    original = float(scaling.get("original_max_position_embeddings", 0))
    if kind == "ntk":
        base = base * factor ** (rotary_dim / max(1, rotary_dim - 2))
    freq = float(base) ** (-torch.arange(half, dtype=torch.float64) / half)
    attention = 1.0
    if kind == "linear":
        freq = freq / factor
    elif kind == "yarn":
        def pair_that_turns(times: float) -> float:
            return half * math.log(original / (times * 2 * math.pi)) / math.log(base)

        low = max(math.floor(pair_that_turns(float(scaling.get("beta_fast", 32.0)))), 0)
        high = min(math.ceil(pair_that_turns(float(scaling.get("beta_slow", 1.0)))), rotary_dim - 1)
        ramp = ((torch.arange(half, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        attention = float(scaling.get("attention_factor", 0.1 * math.log(factor) + 1.0))
    elif kind == "llama3":
        low = float(scaling.get("low_freq_factor", 1.0))
        high = float(scaling.get("high_freq_factor", 4.0))
        if not high > low:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        blend = ((original * freq / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        freq = (1 - blend) * freq / factor + blend * freq
    angle = torch.outer(torch.arange(positions, dtype=torch.float64, device=device), freq.to(device))
    return torch.cat([angle.cos() * attention, angle.sin() * attention], dim=1).float()


def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, *,
           interleaved: bool = False, inverse: bool = False, out=None,
           bad_positions: torch.Tensor | None = None, stream=None):
    """Turn q [N, Hq, D] and k [N, Hk, D] to their positions; returns (q, k).

    `table` [P, R] comes from `rotary_table`; positions are int64 or int32
    [N]. Pairs are (x_j, x_{j + R/2}), or (x_2j, x_2j+1) when `interleaved`;
    values from R on pass through. In place unless out=(q_out, k_out) is given
    (tensors that do not overlap q and k). `inverse` applies the transposed map:
    the gradient of q and k from that of the result. A negative position
    leaves its token's rows unwritten, as -1 does in store_kvcache; so does one
    behind the table, which `bad_positions` (int32, CUDA) counts.

    Autograd does not see the call, nor what it writes: in grad mode inputs
    that require a gradient are refused. In an autograd.Function the backward
    pass is the call on the gradients with `inverse`.
    """
    q_out, k_out = (q, k) if out is None else out
    if _grad_enabled() and (q.requires_grad or k.requires_grad or table.requires_grad
                            or q_out.requires_grad or k_out.requires_grad):
        raise ValueError(_NO_GRADIENT)
    n, q_heads, dim = q.shape
    n_k, kv_heads, dim_k = k.shape
    if n_k != n or dim_k != dim:
        raise ValueError("q and k must have the same tokens and head_dim")
    dtype = q.dtype
    code = _DTYPES.get(dtype)
    if code is None or k.dtype != dtype:
        raise ValueError("q, k and the outputs must share a dtype: bf16, fp16 or fp32")
    kind = positions.dtype
    if (kind != torch.int64 and kind != torch.int32) or positions.shape != (n,) \
            or not positions.is_contiguous():
        raise ValueError("positions must be contiguous int64 or int32, one for each token")
    if table.dtype != torch.float32 or table.dim() != 2 or not table.is_contiguous():
        raise ValueError("table must be contiguous fp32 [positions, rotary_dim]")
    if out is not None:
        if q_out.dtype != dtype or k_out.dtype != dtype:
            raise ValueError("q, k and the outputs must share a dtype: bf16, fp16 or fp32")
        if q_out.shape != q.shape or k_out.shape != k.shape:
            raise ValueError("the outputs must have the shapes of q and k")
    size = 4 if code == _lib.FP32 else 2
    index = q.get_device()
    if index < 0 or k.get_device() != index or positions.get_device() != index \
            or table.get_device() != index:
        raise ValueError(_ONE_DEVICE)
    q_stride, k_stride = _rows(q, "q", size), _rows(k, "k", size)
    if out is None:
        q_out_stride, k_out_stride = q_stride, k_stride
    else:
        _one_device(index, q_out, k_out)
        q_out_stride, k_out_stride = _rows(q_out, "q_out", size), _rows(k_out, "k_out", size)
    bad = 0
    if bad_positions is not None:
        if bad_positions.dtype != torch.int32 or bad_positions.numel() < 1:
            raise ValueError("bad_positions must be int32")
        _one_device(index, bad_positions)
        bad = bad_positions.data_ptr()
    rows, rotary_dim = table.shape
    _launch("kvoff_rotary_packed",
            _ROTARY_ARGS(q.data_ptr(), q_stride, q_out.data_ptr(), q_out_stride, q_heads,
                         k.data_ptr(), k_stride, k_out.data_ptr(), k_out_stride, kv_heads, dim,
                         rotary_dim, code, positions.data_ptr(), 8 if kind == torch.int64 else 4,
                         table.data_ptr(), rows, n, (1 if interleaved else 0) | (2 if inverse else 0),
                         bad, _raw_stream(index, stream)), index)
    return q_out, k_out


def _fp8_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
               v_scale: torch.Tensor, index: int):
    """Check an e4m3 cache [pages, page, H, D] and its scales, all on device `index` (-1: on any).

    Returns the cache's shape and the tokens of a scale block."""
    shape, scales = k_cache.shape, k_scale.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must be [pages, page, heads, head_dim], alike")
    if k_cache.dtype != _FP8 or v_cache.dtype != _FP8:
        raise ValueError("the caches must be float8_e4m3fn")
    if v_scale.shape != scales or len(scales) != 3 or scales[0] != shape[0] or scales[2] != shape[2] \
            or scales[1] <= 0 or shape[1] % scales[1]:
        raise ValueError("the scales must be [pages, page / scale_block, heads]")
    if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
        raise ValueError("the scales must be fp32")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and k_scale.is_contiguous()
            and v_scale.is_contiguous()):
        raise ValueError("caches and scales must be contiguous")
    if index >= 0 and not (k_cache.get_device() == index == v_cache.get_device()
                           and k_scale.get_device() == index == v_scale.get_device()):
        raise ValueError(_ONE_DEVICE)
    return shape, shape[1] // scales[1]


def store_kvcache_fp8(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                      v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                      slot_mapping: torch.Tensor, *, bad_slots: torch.Tensor | None = None,
                      stream=None) -> None:
    """Quantize row i of key/value [N, H, D] into e4m3 cache slot slot_mapping[i] (-1: skip).

    Caches are float8_e4m3fn [pages, page, H, D], scales fp32 [pages, page /
    scale_block, H]: one power of two for each block of scale_block tokens and
    head. A call that writes a block's first token opens the block; later calls
    that need a larger scale rescale the rows that are there (see
    include/kvoff.h). Allocate the scales zeroed. One CUDA-graph-capturable
    launch, at most 65536 tokens. attention_fp8 reads scale blocks of 16 * 2^n
    tokens and heads of 64 and 128 only. Autograd does not see the call: in grad mode
    rows that require a gradient are refused.
    """
    if _grad_enabled() and (key.requires_grad or value.requires_grad or k_scale.requires_grad
                            or v_scale.requires_grad):
        raise ValueError(_NO_GRADIENT)
    shape = key.shape
    num_tokens, heads, dim = shape
    if value.shape != shape:
        raise ValueError("key and value shapes differ")
    dtype = key.dtype
    code = _DTYPES.get(dtype, _lib.FP32)
    if code == _lib.FP32 or value.dtype != dtype:
        raise ValueError("key and value must both be bf16 or fp16")
    index = key.get_device()
    (pages, page, cache_heads, cache_dim), block = _fp8_cache(k_cache, v_cache, k_scale, v_scale, index)
    if cache_heads != heads or cache_dim != dim:
        raise ValueError("cache slots must hold [H, D] rows")
    if slot_mapping.dtype != torch.int32 or slot_mapping.numel() != num_tokens \
            or not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous int32, one slot per token")
    if index < 0 or value.get_device() != index or slot_mapping.get_device() != index:
        raise ValueError(_ONE_DEVICE)
    bad = 0
    if bad_slots is not None:
        if bad_slots.dtype != torch.int32 or bad_slots.numel() < 1:
            raise ValueError("bad_slots must be int32")
        _one_device(index, bad_slots)
        bad = bad_slots.data_ptr()
    _launch("kvoff_store_kvcache_fp8_packed",
            _STORE_ARGS(key.data_ptr(), _rows(key, "key", 2), value.data_ptr(), _rows(value, "value", 2),
                        k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                        heads, dim, code, block, slot_mapping.data_ptr(), num_tokens, pages * page, bad,
                        _raw_stream(index, stream)), index)


_WORKSPACE_BYTES: dict = {}


def attention_fp8_workspace(num_seqs: int, max_seqlen_q: int, table_width: int, page_size: int,
                            q_heads: int, kv_heads: int, head_dim: int, *, device=None) -> int:
    """Workspace bytes that an attention_fp8 call of these sizes needs on `device`."""
    index = torch.device(device).index if device is not None else None
    if index is None:
        index = torch.cuda.current_device()
    return _workspace_bytes(index, (num_seqs, max_seqlen_q, table_width, page_size, q_heads, kv_heads,
                                    head_dim))


def _workspace_bytes(index: int, sizes: tuple) -> int:
    found = _WORKSPACE_BYTES.get((index, sizes))
    if found is None:
        answer = ctypes.c_int64(0)
        with torch.cuda.device(index):
            _lib.call("kvoff_attention_fp8_workspace", *sizes, ctypes.byref(answer))
        if len(_WORKSPACE_BYTES) >= 4096:  # sizes only; a program meets a handful
            _WORKSPACE_BYTES.clear()
        found = _WORKSPACE_BYTES[(index, sizes)] = answer.value
    return found


def _empty_on(stream, q: torch.Tensor, shape, dtype: torch.dtype) -> torch.Tensor:
    """An empty tensor on q's device whose memory belongs to `stream` (None: the current stream)."""
    if stream is None:
        return q.new_empty(shape, dtype=dtype)
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(_stream(q.device, stream), device=q.device)
    with torch.cuda.stream(stream):
        return q.new_empty(shape, dtype=dtype)


def attention_fp8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  k_scale: torch.Tensor, v_scale: torch.Tensor, block_tables: torch.Tensor,
                  context_lens: torch.Tensor, *, cu_seqlens_q: torch.Tensor | None = None,
                  max_seqlen_q: int = 1, softmax_scale: float | None = None,
                  out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                  workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Causal attention of q [N, Hq, D] over an e4m3 paged cache; returns out [N, Hq, D].

    The cache and its scales are store_kvcache_fp8's. Sequence s has its
    context_lens[s] keys (int32, new tokens included) in the pages that row s
    of block_tables (int32 [B, width]) names. Without cu_seqlens_q token s is
    sequence s (a decode step, N == B); with it (int32 [B + 1]) sequence s has
    the tokens cu_seqlens_q[s] .. cu_seqlens_q[s + 1] - 1, at most
    max_seqlen_q, the last of them at its context's end. A row that sees no key
    is zero. softmax_scale defaults to D^-0.5; lse (fp32 [N, Hq]) receives the
    rows' log-sum-exp. See include/kvoff.h for bad pages and padded rows.

    `out` and `workspace` (uint8, attention_fp8_workspace bytes) are allocated
    on the call's stream when not given; calls that may overlap need workspaces
    of their own. Enqueues at most two kernels, copies nothing to the host.
    For inference: the result has no graph, and in grad mode inputs that
    require a gradient are refused.
    """
    if _grad_enabled() and (q.requires_grad or k_scale.requires_grad or v_scale.requires_grad
                            or (out is not None and out.requires_grad)):
        raise ValueError(_NO_GRADIENT)
    q_shape = q.shape
    n, q_heads, dim = q_shape
    index = q.get_device()
    (pages, page, kv_heads, cache_dim), block = _fp8_cache(k_cache, v_cache, k_scale, v_scale, index)
    if cache_dim != dim:
        raise ValueError("q and the caches must have the same head_dim")
    dtype = q.dtype
    code = _DTYPES.get(dtype, _lib.FP32)
    if code == _lib.FP32:
        raise ValueError("q must be bf16 or fp16")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2:
        raise ValueError("block_tables must be int32 [sequences, pages] with dense rows")
    seqs, width = block_tables.shape
    table_stride, entry_stride = block_tables.stride()
    if entry_stride != 1 and width > 1:
        raise ValueError("block_tables must be int32 [sequences, pages] with dense rows")
    if context_lens.dtype != torch.int32 or context_lens.shape != (seqs,) \
            or not context_lens.is_contiguous():
        raise ValueError("context_lens must be contiguous int32, one for each row of block_tables")
    if index < 0 or block_tables.get_device() != index or context_lens.get_device() != index:
        raise ValueError(_ONE_DEVICE)
    starts = 0
    if cu_seqlens_q is not None:
        if cu_seqlens_q.dtype != torch.int32 or cu_seqlens_q.shape != (seqs + 1,) \
                or not cu_seqlens_q.is_contiguous():
            raise ValueError("cu_seqlens_q must be contiguous int32 with one entry more than sequences")
        _one_device(index, cu_seqlens_q)
        starts = cu_seqlens_q.data_ptr()
    elif n != seqs or max_seqlen_q != 1:
        raise ValueError("without cu_seqlens_q each sequence has one token")
    if out is None:
        out = _empty_on(stream, q, q_shape, dtype)
        out_stride = 2 * q_heads * dim
    else:
        if out.shape != q_shape or out.dtype != dtype:
            raise ValueError("out must have the shape and dtype of q")
        _one_device(index, out)
        out_stride = _rows(out, "out", 2)
    lse_ptr = 0
    if lse is not None:
        if lse.dtype != torch.float32 or lse.shape != (n, q_heads) or not lse.is_contiguous():
            raise ValueError("lse must be contiguous fp32 [tokens, q_heads]")
        _one_device(index, lse)
        lse_ptr = lse.data_ptr()
    space = have = 0
    if workspace is None:
        have = _workspace_bytes(index, (seqs, max_seqlen_q, width, page, q_heads, kv_heads, dim))
        if have:
            workspace = _empty_on(stream, q, (have,), torch.uint8)
            space = workspace.data_ptr()
    else:
        if workspace.dtype != torch.uint8 or not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous uint8")
        _one_device(index, workspace)
        have, space = workspace.numel(), workspace.data_ptr()
    _launch("kvoff_attention_fp8_packed",
            _ATTENTION_ARGS(q.data_ptr(), _rows(q, "q", 2), out.data_ptr(), out_stride, lse_ptr,
                            k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                            pages, page, block, block_tables.data_ptr(), table_stride, width,
                            context_lens.data_ptr(), starts, seqs, n, max_seqlen_q, q_heads, kv_heads, dim,
                            code, dim ** -0.5 if softmax_scale is None else softmax_scale, space, have,
                            _raw_stream(index, stream)), index)
    return out
