"""Python mirror of Aegaeon's ``aegaeon.ops`` operator module, backed by the sm_100a C ABI.

``swap`` keeps the exact call signature and meaning of the reference operator
(``aegaeon/ops/ops.h:4-10``, ``aegaeon/ops/swap.cu:25-60``): it runs on the current torch stream,
returns before the copy completes, and takes the block geometry from ``kv_cache``. The other
operators are the per-layer cache write and decode attention that the reference reaches through
vLLM 0.5.1 (``aegaeon/aegaeon/worker.py:517-523``) and the block copy of vLLM's cache ops, on
Aegaeon's ``(N, L, 2, 16, Hkv, D)`` block layout.

Every operator validates its arguments on the host and raises ``ValueError`` (bad argument),
``NotImplementedError`` (unsupported shape) or ``AegaeonError`` (CUDA failure). There is no CPU
or PyTorch fallback: the work always runs in the CUDA library.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Sequence

import numpy as np
import torch

from . import _native
from ._native import AEG_DECODE_PREFETCH, AEG_DECODE_PREFETCH_AFTER_DECODE_WRITE, check, lib
from .layout import BLOCK_SIZE, INT4_TILE, block_bytes

_DTYPES = {torch.float16: _native.AEG_DTYPE_FP16, torch.bfloat16: _native.AEG_DTYPE_BF16}


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _launch(index: int, what: str, fn, *args) -> None:
    """Calls ``fn(*args, stream)`` with device ``index`` current, on its current stream. A decode step is
    dozens of such calls: the device is switched only when it has to be."""
    if _current_device() == index:
        st = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, _raw_stream(index))
    if st:
        check(st, what)


def _on_device(index: int, t: torch.Tensor, name: str) -> None:
    """Raises ValueError unless ``t`` is a tensor on CUDA device ``index``, where the work runs."""
    if not isinstance(t, torch.Tensor) or t.get_device() != index:
        _require_cuda(t, name)
        raise ValueError(f"{name} is on {t.device}, the operation runs on cuda:{index}")


def _on_devices(index: int, tensors: dict) -> None:
    """Raises the error of the tensor that is not on device ``index`` (after a comparison found one)."""
    for name, t in tensors.items():
        _on_device(index, t, name)


def _token_rows(t: torch.Tensor, name: str, what: str) -> torch.Size:
    """The shape of a CUDA ``[tokens, heads, head_dim]`` tensor whose heads are contiguous."""
    _require_cuda(t, name)
    shape = t.shape
    if len(shape) == 3:
        stride = t.stride()
        if stride[2] == 1 and (stride[1] == shape[2] or shape[1] == 1):
            return shape
    raise ValueError(f"{name} must be {what} with contiguous heads")


def _row_stride(t: torch.Tensor) -> int:
    """Elements between the tokens of a ``_token_rows`` tensor; of a single token, whose stride means nothing,
    the row's length."""
    return t.stride(0) if t.size(0) != 1 else t.size(1) * t.size(2)


def _table_stride(t: torch.Tensor) -> int:
    """Entries between the rows of a block table; of a single row, its width."""
    return t.stride(0) if t.size(0) != 1 else t.size(1)


def _require_cuda(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")


def _same_device(dev: torch.device, **tensors) -> None:
    """Raises ValueError unless every given tensor lives on ``dev`` (the device the work runs on):
    a kernel handed another GPU's address would read across NVLink or fault."""
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the operation runs on {dev}")


def _ids_array(ids, name: str) -> np.ndarray:
    if isinstance(ids, torch.Tensor):
        ids = ids.detach().cpu().numpy()
    arr = np.ascontiguousarray(np.asarray(ids, dtype=np.int64).reshape(-1))
    return arr


def _device_ids(ids, device: torch.device, name: str) -> torch.Tensor:
    if isinstance(ids, torch.Tensor):
        if ids.dtype != torch.int64:
            ids = ids.to(torch.int64)
        return ids.to(device, non_blocking=True).contiguous().view(-1)
    return torch.as_tensor(np.asarray(ids, dtype=np.int64).reshape(-1)).to(device, non_blocking=True)


def read_device_errors(device: torch.device | int | None = None) -> int:
    """Reads and clears the library's sticky device error bits (synchronises the stream)."""
    dev = torch.device("cuda") if device is None else torch.device(device)
    if isinstance(device, int):
        dev = torch.device("cuda", device)
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    flags = ctypes.c_uint32(0)
    with torch.cuda.device(dev):
        check(lib.aeg_read_device_errors(_stream(dev), ctypes.byref(flags)), "read_device_errors")
    return int(flags.value)


# --------------------------------------------------------------------------------------------
# Block movement


def _check_pools(kv_cache: torch.Tensor, kv_swap: torch.Tensor) -> int:
    _require_cuda(kv_cache, "kv_cache")
    if not isinstance(kv_swap, torch.Tensor) or kv_swap.device.type != "cpu":
        raise ValueError("kv_swap must be a CPU (host) tensor")
    if not kv_cache.is_contiguous() or not kv_swap.is_contiguous():
        raise ValueError("kv_cache and kv_swap must be contiguous")
    bb = block_bytes(kv_cache)
    if kv_swap.dim() > 0 and kv_swap.size(0) > 0:
        host_bb = kv_swap.numel() * kv_swap.element_size() // kv_swap.size(0)
        if host_bb != bb:
            raise ValueError(f"kv_swap block of {host_bb} bytes differs from kv_cache block of {bb} bytes")
    return bb


def swap(source_block_ids: Sequence[int], target_block_ids: Sequence[int], is_swap_in: bool,
         kv_cache: torch.Tensor, kv_swap: torch.Tensor) -> None:
    """Copies whole KV blocks between the device cache and the host swap pool.

    ``is_swap_in``: host block ``source_block_ids[i]`` -> device block ``target_block_ids[i]``;
    otherwise device -> host. Enqueued on the current stream of ``kv_cache``'s device.
    """
    src = _ids_array(source_block_ids, "source_block_ids")
    dst = _ids_array(target_block_ids, "target_block_ids")
    if src.shape != dst.shape:
        raise ValueError(f"{src.size} source ids but {dst.size} target ids")
    bb = _check_pools(kv_cache, kv_swap)
    if src.size == 0:
        return
    n_host = kv_swap.size(0) if kv_swap.dim() > 0 else 0
    with torch.cuda.device(kv_cache.device):
        st = lib.aeg_swap(kv_cache.data_ptr(), kv_swap.data_ptr(), bb, kv_cache.size(0), n_host,
                          src.ctypes.data, dst.ctypes.data, src.size, int(bool(is_swap_in)),
                          _stream(kv_cache.device))
    check(st, "swap")


def swap_sm(source_block_ids, target_block_ids, is_swap_in: bool, kv_cache: torch.Tensor,
            kv_swap: torch.Tensor) -> None:
    """``swap`` done by one kernel over the mapped page-locked host pool (scattered ids, one launch).

    ``kv_swap`` must be page-locked (``pin_memory()`` or ``cudaHostRegister``). Ids may be lists or
    int64 tensors; they are staged to the device on the current stream.
    """
    bb = _check_pools(kv_cache, kv_swap)
    dev = kv_cache.device
    src = _device_ids(source_block_ids, dev, "source_block_ids")
    dst = _device_ids(target_block_ids, dev, "target_block_ids")
    if src.numel() != dst.numel():
        raise ValueError(f"{src.numel()} source ids but {dst.numel()} target ids")
    if src.numel() == 0:
        return
    n_host = kv_swap.size(0) if kv_swap.dim() > 0 else 0
    with torch.cuda.device(dev):
        st = lib.aeg_swap_sm(kv_cache.data_ptr(), kv_swap.data_ptr(), bb, kv_cache.size(0), n_host,
                             src.data_ptr(), dst.data_ptr(), src.numel(), int(bool(is_swap_in)), _stream(dev))
    check(st, "swap_sm")
    # keep the staged id tensors alive until the kernel has consumed them
    src.record_stream(torch.cuda.current_stream(dev))
    dst.record_stream(torch.cuda.current_stream(dev))


def swap_batched(src: torch.Tensor, dst: torch.Tensor, is_swap_in: bool, kv_cache: torch.Tensor,
                 kv_swap: torch.Tensor, engine: str = "dma") -> None:
    """``swap`` for id lists already held as int64 tensors (no Python list conversion).

    ``engine="dma"``: host (CPU) id tensors, read in place; one copy-engine transfer per run of
    blocks adjacent on both sides, as ``swap``. ``engine="sm"``: ids on the device (or staged
    there), one kernel over the mapped page-locked ``kv_swap``, as ``swap_sm``. Same stream and
    completion rules as ``swap``.
    """
    for t, name in ((src, "src"), (dst, "dst")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int64:
            raise ValueError(f"{name} must be an int64 tensor")
    if engine == "sm":
        swap_sm(src, dst, is_swap_in, kv_cache, kv_swap)
        return
    if engine != "dma":
        raise ValueError(f"engine must be 'dma' or 'sm', not {engine!r}")
    if src.device.type != "cpu" or dst.device.type != "cpu":
        raise ValueError("engine='dma' reads the ids on the host: src and dst must be CPU tensors")
    swap(src.contiguous(), dst.contiguous(), is_swap_in, kv_cache, kv_swap)


def copy_blocks(src_ids, dst_ids, kv_cache: torch.Tensor) -> None:
    """``kv_cache[dst_ids[i]] = kv_cache[src_ids[i]]`` for whole multi-layer blocks (device to device)."""
    _require_cuda(kv_cache, "kv_cache")
    if not kv_cache.is_contiguous():
        raise ValueError("kv_cache must be contiguous")
    dev = kv_cache.device
    src = _device_ids(src_ids, dev, "src_ids")
    dst = _device_ids(dst_ids, dev, "dst_ids")
    if src.numel() != dst.numel():
        raise ValueError(f"{src.numel()} source ids but {dst.numel()} destination ids")
    if src.numel() == 0:
        return
    with torch.cuda.device(dev):
        st = lib.aeg_copy_blocks(kv_cache.data_ptr(), block_bytes(kv_cache), kv_cache.size(0), src.data_ptr(),
                                 dst.data_ptr(), src.numel(), _stream(dev))
    check(st, "copy_blocks")
    src.record_stream(torch.cuda.current_stream(dev))
    dst.record_stream(torch.cuda.current_stream(dev))


# --------------------------------------------------------------------------------------------
# GPU <-> GPU block migration. The reference stubs this path (Worker.register_kvcache_mem_handles
# and Worker.migrate_blocks, aegaeon/aegaeon/worker.py:841-872; BlockManager._migrate_requests,
# aegaeon/aegaeon/block_manager.py:876-950): the target engine opens the source engine's KV-cache
# IPC handles (aegaeon/aegaeon/cuda_wrapper.py:190-208) and copies each request's blocks into
# blocks of its own pool.

IPC_HANDLE_BYTES = _native.AEG_IPC_HANDLE_BYTES


def export_kv_cache(kv_cache: torch.Tensor) -> bytes:
    """The IPC handle of a device block pool, for ``open_kv_cache`` in another process.

    ``kv_cache`` must live in memory from cudaMalloc (PyTorch's default allocator). The handle is
    plain bytes; send it through any host channel (``torch.distributed`` object collectives, a
    store, a pipe). The exporter keeps ``kv_cache`` alive while others have it open.
    """
    _require_cuda(kv_cache, "kv_cache")
    buf = ctypes.create_string_buffer(IPC_HANDLE_BYTES)
    with torch.cuda.device(kv_cache.device):
        check(lib.aeg_ipc_export(kv_cache.data_ptr(), buf), "ipc_export")
    return buf.raw


class PeerKVCache:
    """Another process's block pool mapped into this process (``aeg_ipc_open``).

    ``num_blocks`` and ``block_bytes`` describe the pool (the exporter's ``kv_cache.size(0)`` and
    ``layout.block_bytes(kv_cache)``); the mapping must cover them. ``close()`` (or leaving a
    ``with`` block) unmaps it once the work that reads it has completed.
    """

    def __init__(self, handle: bytes, num_blocks: int, block_bytes_: int):
        if not isinstance(handle, (bytes, bytearray)) or len(handle) != IPC_HANDLE_BYTES:
            raise ValueError(f"an IPC handle is {IPC_HANDLE_BYTES} bytes")
        if num_blocks < 0 or block_bytes_ <= 0:
            raise ValueError("num_blocks must be >= 0 and block_bytes positive")
        ptr = ctypes.c_void_p()
        avail = ctypes.c_int64()
        check(lib.aeg_ipc_open(bytes(handle), ctypes.byref(ptr), ctypes.byref(avail)), "ipc_open")
        self.ptr = int(ptr.value or 0)
        self.num_blocks = int(num_blocks)
        self.block_bytes = int(block_bytes_)
        if num_blocks * block_bytes_ > avail.value:
            self.close()
            raise ValueError(f"the mapped pool holds {avail.value} bytes, fewer than "
                             f"{num_blocks} blocks x {block_bytes_} bytes")

    def close(self) -> None:
        if self.ptr:
            ptr, self.ptr = self.ptr, 0
            check(lib.aeg_ipc_close(ptr), "ipc_close")

    def __enter__(self) -> "PeerKVCache":
        return self

    def __exit__(self, *exc) -> None:
        self.close()


def open_kv_cache(handle: bytes, num_blocks: int, block_bytes_: int) -> PeerKVCache:
    """Maps a pool exported by ``export_kv_cache`` in another process."""
    return PeerKVCache(handle, num_blocks, block_bytes_)


def _pool(p, name: str) -> tuple[int, int, int, torch.device | None]:
    """(address, blocks, block bytes, device of a local tensor or None) of a migration pool."""
    if isinstance(p, PeerKVCache):
        if not p.ptr:
            raise ValueError(f"{name} is closed")
        return p.ptr, p.num_blocks, p.block_bytes, None
    _require_cuda(p, name)
    if not p.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return p.data_ptr(), p.size(0), block_bytes(p), p.device


def migrate_blocks(source_block_ids, target_block_ids, source, target, *, engine: str = "sm") -> None:
    """``target[target_block_ids[i]] <- source[source_block_ids[i]]`` for whole multi-layer blocks
    between two GPUs' pools.

    ``source`` / ``target`` are device tensors of this process (on any GPU it can reach) or
    ``PeerKVCache`` mappings of another process's pool. The work runs on the device of ``target``
    when it is a tensor (a pull, as the reference's target engine does), else on the device of
    ``source`` (a push), on that device's current stream, and returns before it completes.
    ``engine="sm"``: one kernel streams 16-byte vectors over NVLink (ids staged to the device);
    ``engine="dma"``: the copy engines, one transfer per run of blocks adjacent on both sides.
    """
    s_ptr, s_n, s_bb, s_dev = _pool(source, "source")
    t_ptr, t_n, t_bb, t_dev = _pool(target, "target")
    if s_bb != t_bb:
        raise ValueError(f"block sizes differ: source {s_bb} bytes, target {t_bb} bytes")
    dev = t_dev if t_dev is not None else s_dev
    if dev is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    if engine == "dma":
        src = _ids_array(source_block_ids, "source_block_ids")
        dst = _ids_array(target_block_ids, "target_block_ids")
        if src.shape != dst.shape:
            raise ValueError(f"{src.size} source ids but {dst.size} target ids")
        if src.size == 0:
            return
        with torch.cuda.device(dev):
            st = lib.aeg_migrate_blocks_dma(t_ptr, t_n, s_ptr, s_n, s_bb, src.ctypes.data, dst.ctypes.data,
                                            src.size, _stream(dev))
        check(st, "migrate_blocks_dma")
        return
    if engine != "sm":
        raise ValueError(f"engine must be 'sm' or 'dma', not {engine!r}")
    src = _device_ids(source_block_ids, dev, "source_block_ids")
    dst = _device_ids(target_block_ids, dev, "target_block_ids")
    if src.numel() != dst.numel():
        raise ValueError(f"{src.numel()} source ids but {dst.numel()} target ids")
    if src.numel() == 0:
        return
    with torch.cuda.device(dev):
        st = lib.aeg_migrate_blocks(t_ptr, t_n, s_ptr, s_n, s_bb, src.data_ptr(), dst.data_ptr(), src.numel(),
                                    _stream(dev))
    check(st, "migrate_blocks")
    src.record_stream(torch.cuda.current_stream(dev))
    dst.record_stream(torch.cuda.current_stream(dev))


# --------------------------------------------------------------------------------------------
# Prefill attention (vLLM 0.5.1 FlashAttention backend, prompt tokens: flash_attn_varlen_func)


def flash_attn_varlen_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                              max_seqlen: int, softmax_scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of every prompt over itself, the call vLLM makes for prompts:
    ``flash_attn_varlen_func(q, k, v, cu_seqlens, cu_seqlens, max_seqlen, max_seqlen,
    softmax_scale, causal=True)``.

    ``q`` [T, Hq, 128], ``k``/``v`` [T, Hkv, 128] (fp16 or bf16, token-major, head dim
    contiguous), ``cu_seqlens`` int32 [B + 1] on the device (prompt b = tokens cu[b] .. cu[b+1] - 1),
    ``max_seqlen`` the longest prompt. Returns ``out`` [T, Hq, 128].
    """
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _require_cuda(t, name)
        if t.dim() != 3 or t.stride(2) != 1 or t.stride(1) != t.size(2):
            raise ValueError(f"{name} must be [tokens, heads, head_dim] with contiguous heads")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k, v must share an fp16 or bf16 dtype")
    T, Hq, D = q.shape
    if k.shape[0] != T or v.shape != k.shape:
        raise ValueError("k and v must be [tokens, Hkv, head_dim] with q's token count")
    _require_cuda(cu_seqlens, "cu_seqlens")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be a contiguous int32 vector")
    if out is None:
        out = torch.empty_like(q)
    if out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 or out.stride(1) != D:
        raise ValueError("out must match q")
    dev = q.device
    _same_device(dev, k=k, v=v, cu_seqlens=cu_seqlens, out=out)
    with torch.cuda.device(dev):
        st = lib.aeg_prefill_attention(out.data_ptr(), out.stride(0), q.data_ptr(), q.stride(0), k.data_ptr(),
                                       k.stride(0), v.data_ptr(), v.stride(0), cu_seqlens.data_ptr(), T,
                                       cu_seqlens.numel() - 1, int(max_seqlen), Hq, k.size(1), D, float(softmax_scale),
                                       _DTYPES[q.dtype], _stream(dev))
    check(st, "prefill_attention")
    return out


# --------------------------------------------------------------------------------------------
# Model-weight switch (aegaeon/aegaeon/worker.py:358-365: one copy_ per parameter)


def copy_segments(dst: torch.Tensor, src: torch.Tensor, src_offsets, dst_offsets, sizes, *,
                  engine: str = "dma") -> None:
    """Copies byte segments ``src[src_offsets[i]:+sizes[i]] -> dst[dst_offsets[i]:+sizes[i]]``
    between two storages in one call (offsets and sizes in bytes, relative to each tensor's
    first byte), on the current stream of the CUDA side.

    The weight-switch use: ``src`` the page-locked host model cache, ``dst`` the device weight
    arena, one segment per parameter. ``engine="dma"``: copy engines, one transfer per run of
    segments adjacent on both sides; ``engine="sm"``: one kernel through the mapped host memory.
    Destination segments must not overlap; every segment must lie inside both tensors.
    """
    so, do, sz = (_ids_array(x, n) for x, n in ((src_offsets, "src_offsets"), (dst_offsets, "dst_offsets"),
                                                (sizes, "sizes")))
    if not (so.shape == do.shape == sz.shape):
        raise ValueError("src_offsets, dst_offsets and sizes must have the same length")
    if so.size == 0:
        return
    if not (dst.is_contiguous() and src.is_contiguous()):
        raise ValueError("dst and src must be contiguous")
    if (sz < 0).any() or (so < 0).any() or (do < 0).any():
        raise ValueError("offsets and sizes must be non-negative")
    if int((so + sz).max()) > src.numel() * src.element_size() or int((do + sz).max()) > dst.numel() * dst.element_size():
        raise ValueError("a segment runs past the end of its tensor")
    dev = dst.device if dst.device.type == "cuda" else src.device
    if dev.type != "cuda":
        raise ValueError("one of dst / src must be a CUDA tensor")
    eng = {"dma": _native.AEG_COPY_ENGINE_DMA, "sm": _native.AEG_COPY_ENGINE_SM}.get(engine)
    if eng is None:
        raise ValueError(f"engine must be 'dma' or 'sm', not {engine!r}")
    ws_bytes = lib.aeg_copy_segments_workspace_size(so.size) if eng == _native.AEG_COPY_ENGINE_SM else 0
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        st = lib.aeg_copy_segments(dst.data_ptr(), src.data_ptr(), so.ctypes.data, do.ctypes.data, sz.ctypes.data,
                                   so.size, eng, ws.data_ptr(), ws_bytes, _stream(dev))
    check(st, "copy_segments")
    ws.record_stream(torch.cuda.current_stream(dev))


def tensor_segments(tensors, storage: torch.Tensor) -> tuple[np.ndarray, np.ndarray]:
    """(byte offsets within ``storage``, byte sizes) of tensors that live inside ``storage``."""
    base = storage.data_ptr()
    end = base + storage.numel() * storage.element_size()
    offs, sizes = [], []
    for t in tensors:
        n = t.numel() * t.element_size()
        if not (base <= t.data_ptr() and t.data_ptr() + n <= end) or not t.is_contiguous():
            raise ValueError("every tensor must be contiguous and inside the storage")
        offs.append(t.data_ptr() - base)
        sizes.append(n)
    return np.asarray(offs, dtype=np.int64), np.asarray(sizes, dtype=np.int64)


# --------------------------------------------------------------------------------------------
# Per-step model inputs on the device (Worker._prepare_model_inputs, aegaeon/aegaeon/worker.py:596-682)


class StepInputs:
    """Device tensors of one step's model inputs (see ``prepare_step_inputs``)."""

    def __init__(self, B: int, table_stride: int, capacity: int, device: torch.device):
        self.capacity = int(capacity)
        self.slot_mapping = torch.empty(self.capacity, dtype=torch.int64, device=device)
        self.positions = torch.empty(self.capacity, dtype=torch.int64, device=device)
        self.query_lens = torch.empty(B, dtype=torch.int64, device=device)
        self.query_start_loc = torch.empty(B + 1, dtype=torch.int32, device=device)
        self.seq_start_loc = torch.empty(B + 1, dtype=torch.int32, device=device)
        self.block_tables = torch.empty((B, table_stride), dtype=torch.int32, device=device)
        self.num_tokens = torch.empty(1, dtype=torch.int64, device=device)


def prepare_step_inputs(block_tables: torch.Tensor, context_lens: torch.Tensor, seq_lens: torch.Tensor,
                        capacity: int | None = None, out: StepInputs | None = None) -> StepInputs:
    """Slot mapping, positions, start offsets and attention table rows of a step, on the device.

    ``block_tables`` (int32 [B, W], request i's blocks in row i), ``context_lens`` and ``seq_lens``
    (int32 [B]) are device tensors that stay resident across steps (``update_block_tables`` applies
    a step's new blocks). ``capacity`` bounds the new tokens written (default B, i.e. a decode
    batch); ``out.num_tokens`` holds the true count, and a larger count raises a device error.
    Runs on the current stream; nothing is copied to the host.
    """
    for t, name in ((block_tables, "block_tables"), (context_lens, "context_lens"), (seq_lens, "seq_lens")):
        _require_cuda(t, name)
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor")
    if block_tables.dim() != 2:
        raise ValueError("block_tables must be [B, W]")
    B, W = block_tables.shape
    if context_lens.numel() != B or seq_lens.numel() != B:
        raise ValueError("context_lens and seq_lens must have one entry per table row")
    dev = block_tables.device
    _same_device(dev, context_lens=context_lens, seq_lens=seq_lens)
    if out is None:
        out = StepInputs(B, W, B if capacity is None else capacity, dev)
    _same_device(dev, slot_mapping=out.slot_mapping, step_block_tables=out.block_tables)
    with torch.cuda.device(dev):
        st = lib.aeg_prepare_step_inputs(block_tables.data_ptr(), W, context_lens.data_ptr(), seq_lens.data_ptr(), B,
                                         out.slot_mapping.data_ptr(), out.positions.data_ptr(), out.capacity,
                                         out.query_lens.data_ptr(), out.query_start_loc.data_ptr(),
                                         out.seq_start_loc.data_ptr(), out.block_tables.data_ptr(),
                                         out.num_tokens.data_ptr(), _stream(dev))
    check(st, "prepare_step_inputs")
    return out


def update_block_tables(block_tables: torch.Tensor, updates) -> None:
    """Writes ``block_tables[row, col] = block`` for every (row, col, block) triple of ``updates``
    (an int32 [n, 3] tensor or a sequence of triples), on the current stream."""
    _require_cuda(block_tables, "block_tables")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or not block_tables.is_contiguous():
        raise ValueError("block_tables must be a contiguous int32 [rows, W] tensor")
    dev = block_tables.device
    if isinstance(updates, torch.Tensor):
        u = updates.to(device=dev, dtype=torch.int32).contiguous().view(-1, 3)
    else:
        u = torch.as_tensor(np.asarray(updates, dtype=np.int32).reshape(-1, 3)).to(dev, non_blocking=True)
    if u.numel() == 0:
        return
    with torch.cuda.device(dev):
        st = lib.aeg_update_block_tables(block_tables.data_ptr(), block_tables.size(1), block_tables.size(0),
                                         u.data_ptr(), u.size(0), _stream(dev))
    check(st, "update_block_tables")
    u.record_stream(torch.cuda.current_stream(dev))


# --------------------------------------------------------------------------------------------
# Per-layer cache write


def _layer_views(kv_cache: torch.Tensor, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
    _require_cuda(kv_cache, "kv_cache")
    if kv_cache.dim() != 6 or kv_cache.size(2) != 2 or kv_cache.size(3) != BLOCK_SIZE:
        raise ValueError(f"kv_cache must have shape (N, L, 2, 16, Hkv, D), got {tuple(kv_cache.shape)}")
    if not kv_cache.is_contiguous():
        raise ValueError("kv_cache must be contiguous")
    if not 0 <= layer < kv_cache.size(1):
        raise ValueError(f"layer {layer} outside [0, {kv_cache.size(1)})")
    return kv_cache[:, layer, 0], kv_cache[:, layer, 1]


def _check_paged_view(t: torch.Tensor, name: str) -> None:
    _require_cuda(t, name)
    if t.dim() != 4 or t.size(1) != BLOCK_SIZE:
        raise ValueError(f"{name} must be (N, 16, Hkv, D), got {tuple(t.shape)}")
    Hkv, D = t.size(2), t.size(3)
    if t.stride(3) != 1 or t.stride(2) != D or t.stride(1) != Hkv * D:
        raise ValueError(f"{name} must have a contiguous (16, Hkv, D) block interior")


def reshape_and_cache_flash(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor,
                            value_cache: torch.Tensor, slot_mapping: torch.Tensor,
                            kv_cache_dtype: str = "auto") -> None:
    """vLLM-shaped cache write: ``key_cache[s // 16, s % 16] = key[t]`` (same for value), s = slot_mapping[t] >= 0."""
    if kv_cache_dtype != "auto":
        raise NotImplementedError("only kv_cache_dtype='auto' (cache dtype == key dtype) is supported")
    _check_paged_view(key_cache, "key_cache")
    _check_paged_view(value_cache, "value_cache")
    for name, t in (("key", key), ("value", value)):
        _require_cuda(t, name)
        if t.dim() != 3 or t.stride(2) != 1 or t.stride(1) != t.size(2):
            raise ValueError(f"{name} must be [T, Hkv, D] with contiguous heads")
        if t.dtype != key_cache.dtype:
            raise ValueError(f"{name} dtype {t.dtype} differs from cache dtype {key_cache.dtype}")
    if key.shape != value.shape or key.shape[1:] != key_cache.shape[2:]:
        raise ValueError("key/value shapes do not match the cache (Hkv, D)")
    if key_cache.shape != value_cache.shape or key_cache.stride() != value_cache.stride():
        raise ValueError("key_cache and value_cache must have the same shape and strides")
    _require_cuda(slot_mapping, "slot_mapping")
    if slot_mapping.dtype != torch.int64 or slot_mapping.dim() != 1 or slot_mapping.numel() != key.size(0):
        raise ValueError("slot_mapping must be int64 [T]")
    if key.element_size() != 2:
        raise NotImplementedError("only 2-byte cache elements (fp16/bf16) are supported")
    slot_mapping = slot_mapping.contiguous()
    dev = key_cache.device
    _same_device(dev, key=key, value=value, value_cache=value_cache, slot_mapping=slot_mapping)
    with torch.cuda.device(dev):
        st = lib.aeg_reshape_and_cache(key.data_ptr(), value.data_ptr(), key.stride(0), value.stride(0),
                                       key_cache.data_ptr(), value_cache.data_ptr(), key_cache.stride(0),
                                       key_cache.size(0), slot_mapping.data_ptr(), key.size(0), key.size(1),
                                       key.size(2), _stream(dev))
    check(st, "reshape_and_cache")


def reshape_and_cache(key: torch.Tensor, value: torch.Tensor, kv_cache: torch.Tensor, layer: int,
                      slot_mapping: torch.Tensor) -> None:
    """Writes the new tokens' K/V of ``layer`` into Aegaeon's ``(N, L, 2, 16, Hkv, D)`` cache."""
    kc, vc = _layer_views(kv_cache, layer)
    reshape_and_cache_flash(key, value, kc, vc, slot_mapping)


# --------------------------------------------------------------------------------------------
# 4-bit KV cache (layout.int4_block_shape): write and read-back


def _int4_layer(kv_cache: torch.Tensor, layer: int) -> tuple[int, int, int, int]:
    """Checks a 4-bit cache; returns the address of ``layer``'s first tile, the elements between blocks,
    the blocks and the KV heads."""
    _require_cuda(kv_cache, "kv_cache")
    shape = kv_cache.shape
    if len(shape) != 4 or shape[3] != INT4_TILE or kv_cache.dtype not in _DTYPES:
        raise ValueError(f"kv_cache must be a 4-bit cache (N, L, Hkv, {INT4_TILE}) of fp16 or bf16, got "
                         f"{tuple(shape)} of {kv_cache.dtype}")
    if not kv_cache.is_contiguous():
        raise ValueError("kv_cache must be contiguous")
    N, L, Hkv, _ = shape
    if not 0 <= layer < L:
        raise ValueError(f"layer {layer} outside [0, {L})")
    return kv_cache.data_ptr() + layer * Hkv * INT4_TILE * 2, L * Hkv * INT4_TILE, N, Hkv


def _int4_move(fn, what: str, key: torch.Tensor | None, value: torch.Tensor | None, kv_cache: torch.Tensor, layer: int,
               slot_mapping: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Moves rows between ``key``/``value`` (new ones when None) and ``slot_mapping``'s slots of ``layer``."""
    base, block_stride, N, Hkv = _int4_layer(kv_cache, layer)
    dtype, index = kv_cache.dtype, kv_cache.get_device()
    _on_device(index, slot_mapping, "slot_mapping")
    if key is None:
        T, D = slot_mapping.numel(), 128
        key = kv_cache.new_empty((T, Hkv, D))
        value = torch.empty_like(key)
        k_stride = v_stride = Hkv * D
    else:
        T, heads, D = shape = _token_rows(key, "key", "[T, Hkv, D]")
        if _token_rows(value, "value", "[T, Hkv, D]") != shape:
            raise ValueError("key and value must have the same shape")
        if key.dtype != dtype or value.dtype != dtype:
            raise ValueError(f"key dtype {key.dtype} or value dtype {value.dtype} differs from cache dtype {dtype}")
        if heads != Hkv:
            raise ValueError(f"kv_cache holds {Hkv} KV heads, not {heads}")
        if not (index == key.get_device() == value.get_device()):
            _on_devices(index, dict(key=key, value=value))
        k_stride, v_stride = _row_stride(key), _row_stride(value)
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (T,):
        raise ValueError("slot_mapping must be int64 [T]")
    slot_mapping = slot_mapping.contiguous()
    _launch(index, what, fn, key.data_ptr(), value.data_ptr(), k_stride, v_stride, base, block_stride, N,
            slot_mapping.data_ptr(), T, Hkv, D, _DTYPES[dtype])
    return key, value


def reshape_and_cache_int4(key: torch.Tensor, value: torch.Tensor, kv_cache: torch.Tensor, layer: int,
                           slot_mapping: torch.Tensor) -> None:
    """Rounds the new tokens' K/V of ``layer`` to 4 bits and writes them into a 4-bit cache.

    ``key``/``value`` ``[T, Hkv, 128]`` of the cache's dtype (any token stride), ``kv_cache``
    ``(N, L, Hkv, 1152)`` (``layout.int4_block_shape``), ``slot_mapping`` int64 ``[T]``: slot s is row
    s % 16 of block s // 16, s < 0 is padding. Every 64-dim group of a row is held as ``code * scale +
    minimum`` with a 4-bit code; a group with a NaN or an infinity reads back as NaN. The slots of one
    call must be distinct.
    """
    _require_cuda(key, "key")
    _int4_move(lib.aeg_reshape_and_cache_int4, "reshape_and_cache_int4", key, value, kv_cache, layer, slot_mapping)


def gather_cache_int4(kv_cache: torch.Tensor, layer: int, slot_mapping: torch.Tensor, key: torch.Tensor | None = None,
                      value: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values ``[T, Hkv, 128]`` held at ``slot_mapping`` (int64 ``[T]``) of ``layer``, in the
    cache's dtype: what a prompt that continues a cached prefix attends to, or what a 16-bit cache
    takes over. Slots < 0 give zero rows. ``key``/``value`` receive the result when given."""
    if (key is None) != (value is None):
        raise ValueError("key and value are given together")
    return _int4_move(lib.aeg_gather_cache_int4, "gather_cache_int4", key, value, kv_cache, layer, slot_mapping)


# --------------------------------------------------------------------------------------------
# Rotary positions with several axes


@functools.lru_cache(maxsize=64)
def _axis_of(sections: tuple[int, ...], interleaved: bool) -> bytes:
    """The axis of each frequency, one byte each."""
    if not 1 <= len(sections) <= 4 or any(n < 0 for n in sections) or sum(sections) < 1:
        raise ValueError(f"sections must be 1 to 4 non-negative counts of frequencies, got {sections}")
    if not interleaved:
        return bytes(a for a, n in enumerate(sections) for _ in range(n))
    left, order = list(sections), []
    while any(left):
        for a, n in enumerate(left):
            if n:
                left[a] -= 1
                order.append(a)
    return bytes(order)


def rotary_multi_axis(query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                      sections: Sequence[int], *, interleaved: bool = False, scaling: float = 1.0,
                      query_out: torch.Tensor | None = None,
                      key_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotates ``query`` ``[T, Hq, D]`` and ``key`` ``[T, Hkv, D]`` (fp16 or bf16, any token stride) by
    positions with up to four axes (time, height, width of image and video tokens).

    ``positions`` int64 ``[axes, T]`` (``[T]`` for one axis, as ``prepare_step_inputs`` gives them; text
    tokens on several axes may be ``positions.expand(axes, -1)``),
    ``inv_freq`` float32 ``[half]``; ``sections[a]`` frequencies belong to axis a: one section after
    another, or with ``interleaved=True`` dealt to the axes in turn until an axis has its number. Pairs
    are dims (i, i + half); dims from ``2 * half`` on are copied. ``scaling`` multiplies the rotated
    dims. Returns new tensors unless ``query_out``/``key_out`` are given; those may be the inputs.
    """
    sections = tuple(sections)
    axis_of = _axis_of(sections, bool(interleaved))
    axes, half = len(sections), len(axis_of)
    # The usual form is recognised in one expression; anything else is checked piece by piece.
    try:
        T, Hq, D = query.shape
        kT, Hkv, kD = key.shape
        q_stride, q1, q2 = query.stride()
        k_stride, k1, k2 = key.stride()
        axis_stride, step = positions.stride()
        dtype, index = query.dtype, query.get_device()
        usual = (q1 == D == k1 == kD and q2 == 1 == k2 == step and kT == T and dtype in _DTYPES and key.dtype is dtype
                 and 0 <= index == key.get_device() == positions.get_device() == inv_freq.get_device()
                 and positions.dtype is torch.int64 and positions.shape == (axes, T)
                 and inv_freq.dtype is torch.float32 and inv_freq.shape == (half,) and inv_freq.is_contiguous())
    except (AttributeError, TypeError, ValueError, IndexError):
        usual = False
    if not usual:
        positions, inv_freq = _check_rotary(query, key, positions, inv_freq, axes, half)
        (T, Hq, D), Hkv = query.shape, key.size(1)
        q_stride, k_stride, axis_stride = _row_stride(query), _row_stride(key), positions.stride(0)
        dtype, index = query.dtype, query.get_device()
    elif T == 1:  # a single token's stride means nothing
        q_stride, k_stride = Hq * D, Hkv * D
    if query_out is None:
        query_out = torch.empty_like(query) if query.is_contiguous() else query.new_empty(query.shape)
    else:
        _check_rotary_out(index, query_out, query, "query_out")
    if key_out is None:
        key_out = torch.empty_like(key) if key.is_contiguous() else key.new_empty(key.shape)
    else:
        _check_rotary_out(index, key_out, key, "key_out")
    _launch(index, "rotary_multi_axis", lib.aeg_rotary_multi_axis, query_out.data_ptr(), _row_stride(query_out),
            key_out.data_ptr(), _row_stride(key_out), query.data_ptr(), q_stride, key.data_ptr(), k_stride,
            positions.data_ptr(), axis_stride, axes, inv_freq.data_ptr(), axis_of, half, float(scaling), T, Hq, Hkv, D,
            _DTYPES[dtype])
    return query_out, key_out


def _check_rotary(query, key, positions, inv_freq, axes: int, half: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Checks the inputs of ``rotary_multi_axis``; returns positions ``[axes, T]`` with contiguous rows and
    contiguous frequencies."""
    T, _, D = _token_rows(query, "query", "[T, Hq, D]")
    k_shape = _token_rows(key, "key", "[T, Hkv, D]")
    if query.dtype not in _DTYPES or key.dtype != query.dtype:
        raise ValueError("query and key must share an fp16 or bf16 dtype")
    if k_shape[0] != T or k_shape[2] != D:
        raise ValueError("query and key must have the same tokens and head_dim")
    _require_cuda(positions, "positions")
    _require_cuda(inv_freq, "inv_freq")
    if positions.dim() == 1:
        positions = positions.unsqueeze(0)
    if positions.dtype != torch.int64 or positions.shape != (axes, T):
        raise ValueError(f"positions must be int64 [{axes}, {T}]")
    if inv_freq.dtype != torch.float32 or inv_freq.shape != (half,):
        raise ValueError(f"inv_freq must be float32 [{half}], one per frequency of the sections")
    index = query.get_device()
    for name, t in (("key", key), ("positions", positions), ("inv_freq", inv_freq)):
        _on_device(index, t, name)
    if positions.stride(1) != 1 and T > 1:
        positions = positions.contiguous()
    return positions, inv_freq.contiguous()


def _check_rotary_out(index: int, out: torch.Tensor, src: torch.Tensor, name: str) -> None:
    shape = _token_rows(out, name, "its input's shape")
    if shape != src.shape or out.dtype != src.dtype:
        raise ValueError(f"{name} must match its input's shape and dtype")
    if out.data_ptr() == src.data_ptr() and _row_stride(out) != _row_stride(src):
        raise ValueError(f"{name} shares its input's memory with another stride")
    _on_device(index, out, name)


# --------------------------------------------------------------------------------------------
# Shared blocks: forking, freeing and compacting over reference counts


def _check_shared(ref_counts: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor):
    """Checks the state; returns (device index, blocks, table width, rows)."""
    for t, name, dims in ((ref_counts, "ref_counts", 1), (block_tables, "block_tables", 2), (seq_lens, "seq_lens", 1)):
        _require_cuda(t, name)
        if t.dtype != torch.int32 or t.dim() != dims or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor, ref_counts [num_blocks], block_tables [rows, W], "
                             "seq_lens [rows]")
    rows, width = block_tables.shape
    if seq_lens.size(0) != rows:
        raise ValueError("seq_lens must have one entry per table row")
    if width == 0:
        raise ValueError("block_tables has no columns")
    index = ref_counts.get_device()
    _on_device(index, block_tables, "block_tables")
    _on_device(index, seq_lens, "seq_lens")
    return index, ref_counts.size(0), width, rows


def _check_pool(kv_cache: torch.Tensor, index: int, num_blocks: int) -> int:
    """Checks a block pool; returns the bytes of a block."""
    _on_device(index, kv_cache, "kv_cache")
    if kv_cache.dim() < 1 or not kv_cache.is_contiguous():
        raise ValueError("kv_cache must be contiguous")
    if kv_cache.size(0) != num_blocks:
        raise ValueError(f"kv_cache has {kv_cache.size(0)} blocks but ref_counts {num_blocks} entries")
    return block_bytes(kv_cache)


def _row_ids(rows, ref_counts: torch.Tensor, index: int, name: str) -> torch.Tensor:
    if isinstance(rows, torch.Tensor) and rows.dtype == torch.int64 and rows.get_device() == index and rows.dim() == 1:
        return rows.contiguous()
    return _device_ids(rows, ref_counts.device, name)


def fork_blocks(kv_cache: torch.Tensor, ref_counts: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                src_rows, dst_rows) -> torch.Tensor:
    """Turns the empty table row ``dst_rows[i]`` into a fork of row ``src_rows[i]`` (a parallel sample or
    a beam): full blocks are shared (``ref_counts`` goes up), a partly filled last block is copied into
    the lowest free block.

    ``kv_cache`` is any block pool (16-bit or 4-bit, one entry of dim 0 per block), ``ref_counts``
    int32 ``[num_blocks]`` (0 = free), ``block_tables`` int32 ``[rows, W]``, ``seq_lens`` int32 ``[rows]``
    (0 = empty row); ``kv_cache``, ``ref_counts``, ``block_tables`` and ``seq_lens`` are updated in place
    on the current stream, without reading anything back. Returns int32 ``[n]``: the block each fork
    took, or -1. Refused entries leave their row empty and raise a device error
    (``read_device_errors``): a row out of range, a target row that is not empty or named before, a
    last block that is free itself, a pool with no free block left.
    """
    index, N, width, rows = _check_shared(ref_counts, block_tables, seq_lens)
    nbytes = _check_pool(kv_cache, index, N)
    src = _row_ids(src_rows, ref_counts, index, "src_rows")
    dst = _row_ids(dst_rows, ref_counts, index, "dst_rows")
    n = src.size(0)
    if dst.size(0) != n:
        raise ValueError(f"{n} source rows but {dst.size(0)} target rows")
    # One allocation: the result, then the entries' scratch (16-byte aligned).
    ws_bytes = lib.aeg_fork_blocks_workspace_size(n)
    at = (n + 3) // 4 * 4
    buf = ref_counts.new_empty(at + (ws_bytes + 3) // 4)
    new_blocks = buf[:n]
    if n == 0:
        return new_blocks
    ptr = buf.data_ptr()
    _launch(index, "fork_blocks", lib.aeg_fork_blocks, kv_cache.data_ptr(), nbytes, N, ref_counts.data_ptr(),
            block_tables.data_ptr(), width, rows, seq_lens.data_ptr(), src.data_ptr(), dst.data_ptr(), n, ptr, ptr + 4 * at,
            ws_bytes)
    return new_blocks


def free_blocks(ref_counts: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor, rows) -> None:
    """Empties the table rows ``rows``: every block of a row gives back one reference (a block at 0 is
    free), and the row's length becomes 0. A row named twice is freed once."""
    index, N, width, n_rows = _check_shared(ref_counts, block_tables, seq_lens)
    ids = _row_ids(rows, ref_counts, index, "rows")
    if ids.size(0):
        _launch(index, "free_blocks", lib.aeg_free_blocks, N, ref_counts.data_ptr(), block_tables.data_ptr(), width, n_rows,
                seq_lens.data_ptr(), ids.data_ptr(), ids.size(0))


class CompactedBlocks(NamedTuple):
    """What ``compact_blocks`` returns (device tensors)."""
    block_tables: torch.Tensor  # int32 [rows, W], the tables with the new ids
    ref_counts: torch.Tensor    # int32 [num_blocks], of the new ids
    remap: torch.Tensor         # int32 [num_blocks], old id -> new id, -1 for a free block
    num_live: torch.Tensor      # int32 [1]: ids 0 .. num_live - 1 are live, all others free


def compact_blocks(kv_cache: torch.Tensor, ref_counts: torch.Tensor, block_tables: torch.Tensor,
                   seq_lens: torch.Tensor) -> CompactedBlocks:
    """Moves a fragmented pool's live blocks to its lowest ids, so that its tail can be given to another
    model, on the current stream and without reading anything back.

    The live blocks' contents are copied within ``kv_cache``: the k-th live id that is not below the
    number of live blocks goes to the k-th free id below it. ``ref_counts``, ``block_tables`` and
    ``seq_lens`` are only read: adopt the returned tables and counts. The old places keep their
    contents, so reads through the old tables stay right until their ids are given out; writes through
    them after this call do not reach the moved blocks.
    """
    index, N, width, rows = _check_shared(ref_counts, block_tables, seq_lens)
    nbytes = _check_pool(kv_cache, index, N)
    out = CompactedBlocks(torch.empty_like(block_tables), torch.empty_like(ref_counts), torch.empty_like(ref_counts),
                          ref_counts.new_empty(1))
    ws_bytes = lib.aeg_compact_blocks_workspace_size(N)
    ws = ref_counts.new_empty((ws_bytes + 3) // 4)
    _launch(index, "compact_blocks", lib.aeg_compact_blocks, kv_cache.data_ptr(), nbytes, N, ref_counts.data_ptr(),
            block_tables.data_ptr(), width, rows, seq_lens.data_ptr(), out.ref_counts.data_ptr(),
            out.block_tables.data_ptr(), out.remap.data_ptr(), out.num_live.data_ptr(), ws.data_ptr(), ws_bytes)
    return out


# --------------------------------------------------------------------------------------------
# Decode attention


class DecodePlan:
    """Per-step work plan + scratch for ``paged_attention_decode`` (built once, used by every layer).

    The plan depends only on ``seq_lens`` (like the per-step attention metadata of
    ``aegaeon/aegaeon/worker.py:694-711``). Its workspace is device memory owned by this object;
    one plan must not be used by two streams at the same time. ``cache="int4"`` plans for
    ``paged_attention_decode_int4``, ``"auto"`` for the calls on 16-bit caches.
    """

    def __init__(self, batch: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                 device: torch.device | str = "cuda", cache: str = "auto"):
        if cache not in ("auto", "int4"):
            raise ValueError(f"cache must be 'auto' or 'int4', not {cache!r}")
        self.cache = cache
        self.batch, self.num_q_heads, self.num_kv_heads, self.head_dim = batch, num_q_heads, num_kv_heads, head_dim
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("DecodePlan needs a CUDA device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        nbytes = lib.aeg_decode_workspace_size(batch, num_q_heads, num_kv_heads, head_dim)
        if nbytes == 0:
            raise ValueError(f"invalid decode shape B={batch} Hq={num_q_heads} Hkv={num_kv_heads} D={head_dim}")
        self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        self.table_width: int | None = None
        self.seq_lens: torch.Tensor | None = None
        self.block_tables: torch.Tensor | None = None

    def plan(self, seq_lens: torch.Tensor, block_tables: torch.Tensor) -> "DecodePlan":
        """Builds the unit list for ``seq_lens`` (int32 CUDA [B]) and ``block_tables`` (int32 CUDA
        [B, W]) on the current stream. Both must stay unchanged while the plan is in use."""
        _require_cuda(seq_lens, "seq_lens")
        _require_cuda(block_tables, "block_tables")
        if seq_lens.dtype != torch.int32 or seq_lens.shape != (self.batch,):
            raise ValueError(f"seq_lens must be int32 [{self.batch}]")
        if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.size(0) != self.batch:
            raise ValueError(f"block_tables must be int32 [{self.batch}, W]")
        if block_tables.size(1) == 0:
            raise ValueError("block_tables has no columns")
        index = self.device.index
        _on_device(index, seq_lens, "seq_lens")
        _on_device(index, block_tables, "block_tables")
        seq_lens = seq_lens.contiguous()
        if block_tables.stride(1) != 1:
            block_tables = block_tables.contiguous()
        int4 = self.cache == "int4"
        _launch(index, "decode_plan_int4" if int4 else "decode_plan", lib.aeg_decode_plan_int4 if int4 else lib.aeg_decode_plan,
                self.workspace.data_ptr(), self.workspace.numel(), block_tables.data_ptr(), _table_stride(block_tables),
                seq_lens.data_ptr(), self.batch, self.num_q_heads, self.num_kv_heads, self.head_dim)
        self.table_width = block_tables.size(1)
        self.seq_lens = seq_lens
        self.block_tables = block_tables
        return self

    def stats(self) -> dict:
        """What the last ``plan`` built, read back from the workspace header (waits for the plan):
        the cost-axis positions (blocks plus the starting cost per non-empty (sequence, head) pair), the
        worker warps the positions were cut for, the units (pieces of pairs between pair ends and
        warp starts), the split-pair entries (pairs cut across warps, plus empty pairs), the
        partial-result slots those pieces write, and the split-merge items."""
        words = self.workspace[:24].view(torch.int32).cpu().tolist()
        keys = ("items", "workers", "units", "split_pair_entries", "partial_slots", "merge_items")
        return dict(zip(keys, words))

    def matches(self, B: int, Hq: int, Hkv: int, D: int, block_table: torch.Tensor, seq_lens: torch.Tensor,
                cache: str = "auto") -> bool:
        tables, lens = self.block_tables, self.seq_lens
        return ((self.batch, self.num_q_heads, self.num_kv_heads, self.head_dim, self.cache) == (B, Hq, Hkv, D, cache)
                and tables is not None and (tables is block_table or (tables.data_ptr() == block_table.data_ptr()
                                                                      and _table_stride(tables) == _table_stride(block_table)))
                and (lens is seq_lens or lens.data_ptr() == seq_lens.data_ptr())
                and self.table_width == block_table.size(1))


def flash_attn_decode(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                      block_table: torch.Tensor, cache_seqlens: torch.Tensor, softmax_scale: float | None = None,
                      out: torch.Tensor | None = None, plan: DecodePlan | None = None,
                      prefetch: bool = False, after_decode_write: bool = False) -> torch.Tensor:
    """Paged decode attention with one query token per sequence (vLLM FlashAttention decode call).

    query ``[B, Hq, D]``; key_cache/value_cache ``(N, 16, Hkv, D)`` views (any block stride);
    block_table int32 ``[B, W]``; cache_seqlens int32 ``[B]``. Returns ``out [B, Hq, D]``.
    ``plan`` must have been built for these ``cache_seqlens`` and ``W``; without one a plan is built
    on the fly (an extra launch). ``prefetch=True`` promises that the kernel launched just before
    on this stream writes neither these cache blocks nor the block table (``AEG_DECODE_PREFETCH``).
    ``after_decode_write=True`` promises that it wrote at most each sequence's newest position
    ``cache_seqlens[b] - 1`` (the decode ``reshape_and_cache_flash``) and no block table
    (``AEG_DECODE_PREFETCH_AFTER_DECODE_WRITE``): tiles are requested early and that row is read
    again after the preceding kernel has finished.
    """
    _require_cuda(query, "query")
    if query.dim() != 3 or query.stride(2) != 1 or query.stride(1) != query.size(2):
        raise ValueError("query must be [B, Hq, D] with contiguous heads")
    _check_paged_view(key_cache, "key_cache")
    _check_paged_view(value_cache, "value_cache")
    if key_cache.shape != value_cache.shape or key_cache.stride() != value_cache.stride():
        raise ValueError("key_cache and value_cache must have the same shape and strides")
    B, Hq, D = query.shape
    Hkv = key_cache.size(2)
    if key_cache.size(3) != D:
        raise ValueError("head_dim of query and cache differ")
    if query.dtype not in _DTYPES or key_cache.dtype != query.dtype:
        raise ValueError("query and caches must share an fp16 or bf16 dtype")
    _require_cuda(block_table, "block_table")
    _require_cuda(cache_seqlens, "cache_seqlens")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.size(0) != B:
        raise ValueError("block_table must be int32 [B, W]")
    if block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    if cache_seqlens.dtype != torch.int32 or cache_seqlens.shape != (B,):
        raise ValueError("cache_seqlens must be int32 [B]")
    cache_seqlens = cache_seqlens.contiguous()
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    else:
        _require_cuda(out, "out")
        if out.shape != query.shape or out.dtype != query.dtype or out.stride(2) != 1 or out.stride(1) != D:
            raise ValueError("out must match query's shape/dtype with contiguous heads")
    if B == 0:
        return out
    W = block_table.size(1)
    if W == 0:
        raise ValueError("block_table has no columns")
    if plan is None:
        plan = DecodePlan(B, Hq, Hkv, D, query.device).plan(cache_seqlens, block_table)
    elif not plan.matches(B, Hq, Hkv, D, block_table, cache_seqlens):
        raise ValueError("plan was built for a different batch / head layout / block tables / sequence lengths")
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    dev = query.device
    _same_device(dev, key_cache=key_cache, value_cache=value_cache, block_table=block_table,
                 cache_seqlens=cache_seqlens, out=out, plan_workspace=plan.workspace)
    with torch.cuda.device(dev):
        st = lib.aeg_paged_attn_decode(out.data_ptr(), out.stride(0), query.data_ptr(), query.stride(0),
                                       key_cache.data_ptr(), value_cache.data_ptr(), key_cache.stride(0),
                                       key_cache.size(0), block_table.data_ptr(), block_table.stride(0),
                                       cache_seqlens.data_ptr(), B, Hq, Hkv, D, scale, _DTYPES[query.dtype],
                                       plan.workspace.data_ptr(), plan.workspace.numel(),
                                       (AEG_DECODE_PREFETCH if prefetch else 0)
                                       | (AEG_DECODE_PREFETCH_AFTER_DECODE_WRITE if after_decode_write else 0),
                                       _stream(dev))
    check(st, "paged_attention_decode")
    return out


def decode_layer_flash(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor,
                       value_cache: torch.Tensor, block_table: torch.Tensor, cache_seqlens: torch.Tensor,
                       softmax_scale: float | None = None, out: torch.Tensor | None = None,
                       plan: DecodePlan | None = None, prefetch: bool = False) -> torch.Tensor:
    """Cache write of each sequence's new token + decode attention, in one launch.

    ``key``/``value`` ``[B, Hkv, D]`` are written at position ``cache_seqlens[b] - 1`` of sequence b
    (the decode slot the reference builds, ``aegaeon/aegaeon/worker.py:628-633``), then attention runs
    over ``[0, cache_seqlens[b])``. Same result as ``reshape_and_cache_flash`` with those slots followed
    by ``flash_attn_decode``. ``prefetch`` as for ``flash_attn_decode``.
    """
    _require_cuda(query, "query")
    if query.dim() != 3 or query.stride(2) != 1 or query.stride(1) != query.size(2):
        raise ValueError("query must be [B, Hq, D] with contiguous heads")
    _check_paged_view(key_cache, "key_cache")
    _check_paged_view(value_cache, "value_cache")
    if key_cache.shape != value_cache.shape or key_cache.stride() != value_cache.stride():
        raise ValueError("key_cache and value_cache must have the same shape and strides")
    B, Hq, D = query.shape
    Hkv = key_cache.size(2)
    for name, t in (("key", key), ("value", value)):
        _require_cuda(t, name)
        if tuple(t.shape) != (B, Hkv, D) or t.stride(2) != 1 or t.stride(1) != D or t.dtype != query.dtype:
            raise ValueError(f"{name} must be [B, Hkv, D] of the query dtype with contiguous heads")
    if key_cache.size(3) != D:
        raise ValueError("head_dim of query and cache differ")
    if query.dtype not in _DTYPES or key_cache.dtype != query.dtype:
        raise ValueError("query and caches must share an fp16 or bf16 dtype")
    _require_cuda(block_table, "block_table")
    _require_cuda(cache_seqlens, "cache_seqlens")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.size(0) != B:
        raise ValueError("block_table must be int32 [B, W]")
    if block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    if cache_seqlens.dtype != torch.int32 or cache_seqlens.shape != (B,):
        raise ValueError("cache_seqlens must be int32 [B]")
    cache_seqlens = cache_seqlens.contiguous()
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    elif out.shape != query.shape or out.dtype != query.dtype or out.stride(2) != 1 or out.stride(1) != D:
        raise ValueError("out must match query's shape/dtype with contiguous heads")
    if B == 0:
        return out
    if plan is None:
        plan = DecodePlan(B, Hq, Hkv, D, query.device).plan(cache_seqlens, block_table)
    elif not plan.matches(B, Hq, Hkv, D, block_table, cache_seqlens):
        raise ValueError("plan was built for a different batch / head layout / block tables / sequence lengths")
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    dev = query.device
    _same_device(dev, key=key, value=value, key_cache=key_cache, value_cache=value_cache, block_table=block_table,
                 cache_seqlens=cache_seqlens, out=out, plan_workspace=plan.workspace)
    with torch.cuda.device(dev):
        st = lib.aeg_decode_layer(out.data_ptr(), out.stride(0), query.data_ptr(), query.stride(0), key.data_ptr(),
                                  key.stride(0), value.data_ptr(), value.stride(0), key_cache.data_ptr(),
                                  value_cache.data_ptr(), key_cache.stride(0), key_cache.size(0), block_table.data_ptr(),
                                  block_table.stride(0), cache_seqlens.data_ptr(), B, Hq, Hkv, D, scale,
                                  _DTYPES[query.dtype], plan.workspace.data_ptr(), plan.workspace.numel(),
                                  AEG_DECODE_PREFETCH if prefetch else 0, _stream(dev))
    check(st, "decode_layer")
    return out


def decode_layer(out: torch.Tensor, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                 kv_cache: torch.Tensor, layer: int, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                 scale: float, plan: DecodePlan | None = None, prefetch: bool = False) -> None:
    """Fused cache write + decode attention of ``layer`` over Aegaeon's ``(N, L, 2, 16, Hkv, D)`` cache."""
    kc, vc = _layer_views(kv_cache, layer)
    decode_layer_flash(query, key, value, kc, vc, block_tables, seq_lens, scale, out=out, plan=plan, prefetch=prefetch)


def paged_attention_decode(out: torch.Tensor, query: torch.Tensor, kv_cache: torch.Tensor, layer: int,
                           block_tables: torch.Tensor, seq_lens: torch.Tensor, scale: float,
                           plan: DecodePlan | None = None, prefetch: bool = False,
                           after_decode_write: bool = False) -> None:
    """Decode attention of ``layer`` over Aegaeon's ``(N, L, 2, 16, Hkv, D)`` cache, into ``out``."""
    kc, vc = _layer_views(kv_cache, layer)
    flash_attn_decode(query, kc, vc, block_tables, seq_lens, scale, out=out, plan=plan, prefetch=prefetch,
                      after_decode_write=after_decode_write)


def paged_attention_decode_int4(out: torch.Tensor, query: torch.Tensor, kv_cache: torch.Tensor, layer: int,
                                block_tables: torch.Tensor, seq_lens: torch.Tensor, scale: float,
                                plan: DecodePlan | None = None, prefetch: bool = False) -> None:
    """Decode attention of ``layer`` over a 4-bit cache ``(N, L, Hkv, 1152)`` of the query's dtype
    (``layout.int4_block_shape``, written by ``reshape_and_cache_int4``), into ``out``.

    Arguments as for ``paged_attention_decode``; ``plan`` is a ``DecodePlan(..., cache="int4")`` built
    for these tables and lengths. ``prefetch=True`` promises that the kernel launched just before on
    this stream writes neither this layer's blocks nor the block tables (so not right after the
    layer's ``reshape_and_cache_int4``); no kernel of this library further back is passed.
    """
    # A decode loop makes this call for every layer of every step, so its usual form is recognised in one
    # expression; anything else is checked piece by piece (and refused, or brought into that form).
    try:
        B, Hq, D = shape = query.shape
        N, L, Hkv, tile = kv_cache.shape
        q_stride, q1, q2 = query.stride()
        out_stride, o1, o2 = out.stride()
        t_stride, t1 = block_tables.stride()
        dtype, index, i32 = query.dtype, query.get_device(), torch.int32
        usual = (plan is not None and q1 == D == o1 and q2 == 1 == o2 == t1 and tile == INT4_TILE and 0 <= layer < L
                 and kv_cache.dtype is dtype and out.dtype is dtype and block_tables.dtype is i32 and seq_lens.dtype is i32
                 and 0 <= index == kv_cache.get_device() == block_tables.get_device() == seq_lens.get_device()
                 == out.get_device() == plan.workspace.get_device()
                 and out.shape == shape and seq_lens.shape == (B,) and dtype in _DTYPES and kv_cache.is_contiguous()
                 and seq_lens.is_contiguous() and plan.matches(B, Hq, Hkv, D, block_tables, seq_lens, "int4"))
    except (AttributeError, TypeError, ValueError, IndexError):
        usual = False
    if not usual:
        block_tables, seq_lens, plan = _check_attention_int4(out, query, kv_cache, layer, block_tables, seq_lens, plan)
        if plan is None:  # an empty batch
            return
        (B, Hq, D), (N, L, Hkv, tile) = query.shape, kv_cache.shape
        q_stride, out_stride, t_stride = _row_stride(query), _row_stride(out), _table_stride(block_tables)
        dtype, index = query.dtype, query.get_device()
    elif B == 1:  # a single row's stride means nothing
        q_stride, out_stride, t_stride = Hq * D, Hq * D, block_tables.size(1)
    ws = plan.workspace
    head = Hkv * INT4_TILE
    _launch(index, "paged_attention_decode_int4", lib.aeg_paged_attn_decode_int4, out.data_ptr(), out_stride,
            query.data_ptr(), q_stride, kv_cache.data_ptr() + 2 * layer * head, L * head, N, block_tables.data_ptr(), t_stride,
            seq_lens.data_ptr(), B, Hq, Hkv, D, float(scale), _DTYPES[dtype], ws.data_ptr(), ws.numel(),
            AEG_DECODE_PREFETCH if prefetch else 0)


def _check_attention_int4(out, query, kv_cache, layer, block_tables, seq_lens, plan):
    """Checks every argument of ``paged_attention_decode_int4``; returns contiguous tables and lengths and
    a plan for them (None for an empty batch)."""
    B, Hq, D = shape = _token_rows(query, "query", "[B, Hq, D]")
    Hkv = _int4_layer(kv_cache, layer)[3]
    dtype = query.dtype
    if dtype != kv_cache.dtype:
        raise ValueError(f"query dtype {dtype} differs from cache dtype {kv_cache.dtype}")
    _require_cuda(block_tables, "block_tables")
    _require_cuda(seq_lens, "seq_lens")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.size(0) != B:
        raise ValueError("block_tables must be int32 [B, W]")
    if block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    if seq_lens.dtype != torch.int32 or seq_lens.shape != (B,):
        raise ValueError("seq_lens must be int32 [B]")
    seq_lens = seq_lens.contiguous()
    if _token_rows(out, "out", "query's shape") != shape or out.dtype != dtype:
        raise ValueError("out must match query's shape and dtype")
    index = query.get_device()
    for name, t in (("kv_cache", kv_cache), ("block_tables", block_tables), ("seq_lens", seq_lens), ("out", out)):
        _on_device(index, t, name)
    if B == 0:
        return block_tables, seq_lens, None
    if block_tables.size(1) == 0:
        raise ValueError("block_tables has no columns")
    if plan is None:
        plan = DecodePlan(B, Hq, Hkv, D, query.device, cache="int4").plan(seq_lens, block_tables)
    elif not plan.matches(B, Hq, Hkv, D, block_tables, seq_lens, "int4"):
        raise ValueError("plan was built for a different batch / head layout / block tables / sequence lengths / cache")
    _on_device(index, plan.workspace, "plan workspace")
    return block_tables, seq_lens, plan
