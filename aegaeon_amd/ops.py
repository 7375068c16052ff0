"""Operator API of the KV movement path (the `aegaeon.ops` drop-in).

`swap` keeps the reference's positional signature, ops/ops.h:4-10
(`swap(source_block_ids, target_block_ids, is_swap_in, kv_cache, kv_swap)`),
and runs on the current stream like ops/swap.cu:21-32. `swap_segments` is the
composite-page data plane of Worker.swap_blocks (aegaeon/worker.py:2265-2329)
and `copy_blocks` the in-HBM block copy. Every call is one C-ABI call into
libaegkv.so; there is no Python or CPU fallback. `QuantCache`, `CacheBatch` and
`quant_write`, `quant_read`, `quant_attend` hold a cache in 4 or 8 bits, which the
moves take like any other; the reference has none.
"""

from __future__ import annotations

import ctypes
import struct
import sys
import threading
import weakref
from typing import Sequence

import numpy as np
import torch

from . import _lib

MODE_AUTO = _lib.MODE_AUTO
MODE_DIRECT = _lib.MODE_DIRECT
MODE_STAGED = _lib.MODE_STAGED
FENCE_FAILED = _lib.FENCE_FAILED
MoveFailedError = _lib.MoveFailedError

_MODES = {"auto": MODE_AUTO, "direct": MODE_DIRECT, "staged": MODE_STAGED}


def _mode(mode) -> int:
    if isinstance(mode, str):
        try:
            return _MODES[mode]
        except KeyError:
            raise ValueError(f"unknown transfer mode {mode!r}") from None
    if mode not in (MODE_AUTO, MODE_DIRECT, MODE_STAGED):
        raise ValueError(f"unknown transfer mode {mode!r}")
    return int(mode)


def _ints(values) -> np.ndarray:
    """A flat integer array; floats and booleans are refused rather than
    truncated (an empty list is fine)."""
    if isinstance(values, torch.Tensor):
        values = values.detach().cpu().numpy()
    a = np.asarray(values).reshape(-1)
    if a.size and a.dtype.kind not in "iu":
        raise ValueError(f"expected integers, got {a.dtype} values")
    return a


def _i64(values) -> np.ndarray:
    return np.ascontiguousarray(_ints(values).astype(np.int64, copy=False))


def _i32(values) -> np.ndarray:
    a = _ints(values)
    if a.size and (a.min() < np.iinfo(np.int32).min or a.max() > np.iinfo(np.int32).max):
        raise ValueError("group ids must fit in 32 bits")
    return np.ascontiguousarray(a.astype(np.int32, copy=False))


def _id_arg(values):
    """(C argument, count) of an id list: packed in one native pass where it
    is a list of Python integers, as planners make it, else through _i64."""
    packed = _lib.hostargs().pack_ids(values)
    if packed is not None:
        return packed, len(packed) // 8
    a = _i64(values)
    return _p64(a), a.size   # the pointer keeps the array


def _group_arg(values):
    """_id_arg for 32-bit group ids."""
    packed = _lib.hostargs().pack_ids32(values, 1 << 31)
    if packed is not None:
        return packed, len(packed) // 4
    a = _i32(values)
    return _p32(a), a.size


def _p64(a: np.ndarray):
    return a.ctypes.data_as(ctypes.POINTER(ctypes.c_int64))


def _p32(a: np.ndarray):
    return a.ctypes.data_as(ctypes.POINTER(ctypes.c_int32))


def _pu64(a: np.ndarray):
    return a.ctypes.data_as(ctypes.POINTER(ctypes.c_uint64))


def _stream_ptr(device: torch.device, stream: torch.cuda.Stream | None) -> int:
    if stream is not None:
        return stream.cuda_stream
    if device.index is not None and torch.cuda.is_initialized():
        # the same stream without making a Stream object of it (2.6 us)
        return torch._C._cuda_getCurrentRawStream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _tensor_bytes(t: torch.Tensor) -> int:
    return t.numel() * t.element_size()


def _require_device(t: torch.Tensor, what: str) -> None:
    if t.device.type != "cuda":
        raise ValueError(f"{what} must be a device (HIP) tensor, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


def _require_host(t: torch.Tensor, what: str) -> None:
    if t.device.type != "cpu":
        raise ValueError(f"{what} must be a host tensor, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


def swap(
    source_block_ids: Sequence[int],
    target_block_ids: Sequence[int],
    is_swap_in: bool,
    kv_cache: torch.Tensor,
    kv_swap: torch.Tensor,
    *,
    mode="auto",
    stream: torch.cuda.Stream | None = None,
) -> None:
    """Whole-block swap between a device cache and a pinned host pool.

    Follows ops/swap.cu:25-60: block i moves source_block_ids[i] ->
    target_block_ids[i]; is_swap_in copies host (kv_swap) -> device
    (kv_cache), otherwise device -> host. The block size is
    kv_cache.numel() * element_size / kv_cache.size(0) bytes and is used for
    both tensors; for the 2-byte dtypes the reference supports this equals
    its `numel * 2 / size(0)` (swap.cu:34). Runs on the current stream.
    Raises ValueError on bad ids (the reference checks nothing).
    """
    _require_device(kv_cache, "kv_cache")
    _require_host(kv_swap, "kv_swap")
    src = _i64(source_block_ids)
    dst = _i64(target_block_ids)
    if src.shape != dst.shape:
        raise ValueError(
            f"source ({src.size}) and target ({dst.size}) id lists differ in length"
        )
    if kv_cache.dim() == 0 or kv_cache.size(0) == 0:
        raise ValueError("kv_cache must have a non-empty block dimension")
    block_bytes = _tensor_bytes(kv_cache) // kv_cache.size(0)
    if _tensor_bytes(kv_cache) % kv_cache.size(0):
        raise ValueError("kv_cache bytes are not divisible by its block count")
    swap_blocks_total = _tensor_bytes(kv_swap) // block_bytes
    lib = _lib.load()
    with torch.cuda.device(kv_cache.device):
        rc = lib.aegkv_swap(
            _p64(src), _p64(dst), src.size, 1 if is_swap_in else 0,
            kv_cache.data_ptr(), kv_cache.size(0),
            kv_swap.data_ptr(), swap_blocks_total, block_bytes,
            _mode(mode), _stream_ptr(kv_cache.device, stream),
        )
    _lib.check(rc)


def _guard_ptr(words: torch.Tensor | None, index: int, what: str):
    """Address of a move guard word (or None): a 1-D int64 tensor in pinned
    host memory (GuardWords) or on the device."""
    if words is None:
        return None
    if words.dtype != torch.int64 or words.dim() != 1 or not words.is_contiguous():
        raise ValueError(f"{what} must be a contiguous 1-D int64 tensor")
    if not 0 <= index < words.numel():
        raise ValueError(f"{what} index {index} outside [0, {words.numel()})")
    return words.data_ptr() + 8 * index


def _call_on(device: torch.device, fn):
    """Run fn() with `device` current, switching (and restoring) only when
    another device is current. Keeps no state, so threads may share it."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    if torch.cuda.current_device() == index:
        return fn()
    with torch.cuda.device(index):
        return fn()


class SegmentLayout:
    """A validated composite layout, reusable across swap calls.

    Holds the backing tensors (segments, each viewed as [device_num_blocks,
    page] bytes), their composite-page geometry (vllm_cache.py:75-101,
    worker.py:1419-1432) and the pinned host pool, checked once and kept as
    the C-ABI arrays the library takes, so a call only converts its id lists.
    The layout keeps references to the tensors it describes.
    """

    def __init__(self, segments: Sequence[torch.Tensor], segment_page_bytes: Sequence[int],
                 segment_host_offsets: Sequence[int], segment_owner_masks: Sequence[int],
                 device_num_blocks: int, group_kernel_blocks_per_page: Sequence[int],
                 host_pool: torch.Tensor, host_page_bytes: int, host_rank_offset: int):
        if not segments:
            raise ValueError("at least one segment is required")
        dev = segments[0].device
        for i, t in enumerate(segments):
            _require_device(t, f"segment {i}")
            if t.device != dev:
                raise ValueError("all segments must live on one device")
        _require_host(host_pool, "host_pool")
        n_seg = len(segments)
        self.page = _i64(segment_page_bytes)
        self.host_offsets = _i64(segment_host_offsets)
        self.owners = np.ascontiguousarray(
            np.asarray(segment_owner_masks, dtype=np.uint64).reshape(-1))
        self.kpp = _i64(group_kernel_blocks_per_page)
        if not (self.page.size == self.host_offsets.size == self.owners.size == n_seg):
            raise ValueError("segment metadata lengths must equal the number of segments")
        for i, t in enumerate(segments):
            if _tensor_bytes(t) < int(self.page[i]) * device_num_blocks:
                raise ValueError(
                    f"segment {i} holds {_tensor_bytes(t)} bytes < "
                    f"{device_num_blocks} x {int(self.page[i])}"
                )
        self.segments = list(segments)
        self.host_pool = host_pool
        self.device = dev
        self.num_segments = n_seg
        self.device_num_blocks = int(device_num_blocks)
        self.host_page_bytes = int(host_page_bytes)
        self.host_rank_offset = int(host_rank_offset)
        self.host_num_blocks = (_tensor_bytes(host_pool) // self.host_page_bytes
                                if self.host_page_bytes > 0 else 0)
        self._bases = (ctypes.c_void_p * n_seg)(*[t.data_ptr() for t in segments])
        self._args = (n_seg, self._bases, _p64(self.page), _p64(self.host_offsets),
                      _pu64(self.owners), self.device_num_blocks, self.kpp.size,
                      _p64(self.kpp), host_pool.data_ptr(), self.host_num_blocks,
                      self.host_page_bytes, self.host_rank_offset)

    def swap(self, source_block_ids, target_block_ids, group_ids, first_kernel_blocks,
             valid_kernel_blocks, is_swap_in: bool, *, mode="auto",
             stream: torch.cuda.Stream | None = None, guard: torch.Tensor | None = None,
             guard_index: int = 0) -> None:
        """One aegkv_swap_blocks call over this layout (see swap_segments).
        guard (with guard_index): a move guard word (GuardWords.tensor); when
        it is set by the time the stream reaches the swap, nothing moves."""
        self._swap_packed(_id_arg(source_block_ids), _id_arg(target_block_ids),
                          _group_arg(group_ids), _id_arg(first_kernel_blocks),
                          _id_arg(valid_kernel_blocks), is_swap_in, mode, stream,
                          _guard_ptr(guard, guard_index, "guard"))

    def _swap_packed(self, src, dst, grp, first, valid, is_swap_in, mode, stream, guard):
        """swap() with its lists as (C argument, count)."""
        if not (src[1] == dst[1] == grp[1] == first[1] == valid[1]):
            raise ValueError(
                f"swap lists of unequal lengths: {src[1]} sources, {dst[1]} targets, "
                f"{grp[1]} groups, {first[1]} first and {valid[1]} valid kernel blocks"
            )
        lib = _lib.load()
        rc = _call_on(self.device, lambda: lib.aegkv_swap_blocks(
            *self._args, src[1], src[0], dst[0], grp[0], first[0], valid[0],
            1 if is_swap_in else 0, _mode(mode), guard, _stream_ptr(self.device, stream)))
        _lib.check(rc)


def swap_segments(
    segments: Sequence[torch.Tensor],
    segment_page_bytes: Sequence[int],
    segment_host_offsets: Sequence[int],
    segment_owner_masks: Sequence[int],
    device_num_blocks: int,
    group_kernel_blocks_per_page: Sequence[int],
    host_pool: torch.Tensor,
    host_page_bytes: int,
    host_rank_offset: int,
    source_block_ids,
    target_block_ids,
    group_ids,
    first_kernel_blocks,
    valid_kernel_blocks,
    is_swap_in: bool,
    *,
    mode="auto",
    stream: torch.cuda.Stream | None = None,
) -> None:
    """Composite-page swap of (segment x entry) extents in one launch.

    Byte placement of aegaeon/worker.py:2265-2329: for each segment s owned
    by the entry's group, extent (off, len) = byte_extent_for_kernel_blocks
    of (page_s, kernel blocks per page, first, valid) (cache_transfer.py:
    138-165); host bytes sit at host_id * host_page_bytes + host_rank_offset
    + host_offset_s + off; device bytes at dev_id * page_s + off of segment s.
    Callers that swap over the same layout repeatedly should build a
    SegmentLayout once and call its swap().
    """
    SegmentLayout(segments, segment_page_bytes, segment_host_offsets, segment_owner_masks,
                  device_num_blocks, group_kernel_blocks_per_page, host_pool, host_page_bytes,
                  host_rank_offset).swap(source_block_ids, target_block_ids, group_ids,
                                         first_kernel_blocks, valid_kernel_blocks, is_swap_in,
                                         mode=mode, stream=stream)


def _copy_call_args(segments, src_block_ids, dst_block_ids, segment_page_bytes,
                    device_num_blocks, stream):
    """Checked C-ABI arguments of one copy_blocks call (device first)."""
    if segment_page_bytes is None:
        table = _lib.hostargs().segment_table(segments, device_num_blocks)
        if table is not None:
            _, blocks, bases, page = table
            src, n = _id_arg(src_block_ids)
            dst, n_dst = _id_arg(dst_block_ids)
            if n != n_dst:
                raise ValueError("src and dst id lists differ in length")
            dev = segments[0].device
            return dev, (len(bases) // 8, bases, page, blocks, n, src, dst,
                         _stream_ptr(dev, stream))
    if not segments:
        raise ValueError("at least one segment is required")
    dev = segments[0].device
    for i, t in enumerate(segments):
        _require_device(t, f"segment {i}")
        if t.device != dev:
            raise ValueError("all segments must live on one device")
    if device_num_blocks is None:
        device_num_blocks = segments[0].size(0)
    if segment_page_bytes is None:
        segment_page_bytes = [_tensor_bytes(t) // device_num_blocks for t in segments]
    page = _i64(segment_page_bytes)
    if page.size != len(segments):
        raise ValueError("segment_page_bytes must have one entry per segment")
    for i, t in enumerate(segments):
        if _tensor_bytes(t) < int(page[i]) * device_num_blocks:
            raise ValueError(f"segment {i} is smaller than {device_num_blocks} blocks")
    src = _i64(src_block_ids)
    dst = _i64(dst_block_ids)
    if src.shape != dst.shape:
        raise ValueError("src and dst id lists differ in length")
    bases = (ctypes.c_void_p * len(segments))(*[t.data_ptr() for t in segments])
    args = (len(segments), bases, _p64(page), int(device_num_blocks), src.size, _p64(src),
            _p64(dst), _stream_ptr(dev, stream))
    return dev, args   # the pointers keep their arrays


def copy_blocks(
    segments: Sequence[torch.Tensor],
    src_block_ids,
    dst_block_ids,
    *,
    segment_page_bytes: Sequence[int] | None = None,
    device_num_blocks: int | None = None,
    stream: torch.cuda.Stream | None = None,
) -> None:
    """In-HBM block copy: seg[dst[i]] := seg[src[i]] for every segment.

    Each segment is viewed as [num_blocks, page] bytes; by default the page
    is the tensor's bytes / size(0). Targets must be distinct and disjoint
    from the sources. The reference has no KV copy_blocks; its in-HBM
    compaction is aegaeon/allocator.py:101-137.
    """
    dev, args = _copy_call_args(segments, src_block_ids, dst_block_ids,
                                segment_page_bytes, device_num_blocks, stream)
    lib = _lib.load()
    _lib.check(_call_on(dev, lambda: lib.aegkv_copy_blocks(*args)))


PROBE_READ = _lib.PROBE_READ
PROBE_WRITE = _lib.PROBE_WRITE


def copy_probe(kind: int, segments: Sequence[torch.Tensor], src_block_ids, dst_block_ids,
               sink: torch.Tensor, *, magic: int = 0x9E3779B9,
               segment_page_bytes: Sequence[int] | None = None,
               device_num_blocks: int | None = None,
               stream: torch.cuda.Stream | None = None) -> None:
    """Measurement only: the read half (PROBE_READ: load every source tile)
    or the write half (PROBE_WRITE: store a fixed pattern into every target
    tile, destroying its contents) of copy_blocks with the same ids, work
    items and launch shape (aegkv_copy_probe). sink: a device int32/uint32
    tensor the read probe may write one word of."""
    if kind not in (PROBE_READ, PROBE_WRITE):
        raise ValueError(f"unknown probe kind {kind!r}")
    if sink.device.type != "cuda" or sink.element_size() != 4 or sink.numel() < 1:
        raise ValueError("sink must be a device tensor of 4-byte words")
    dev, args = _copy_call_args(segments, src_block_ids, dst_block_ids,
                                segment_page_bytes, device_num_blocks, stream)
    lib = _lib.load()
    _lib.check(_call_on(dev, lambda: lib.aegkv_copy_probe(
        kind, *args[:-1], sink.data_ptr(), int(magic) & 0xFFFFFFFF, args[-1])))


#: limits of copy_blocks_noalloc (the fixed descriptor array of libaegkv)
NOALLOC_MAX_SEGMENTS = 1024
NOALLOC_MAX_PAIRS = 65536


def copy_blocks_noalloc(
    segments: Sequence[torch.Tensor],
    src_block_ids,
    dst_block_ids,
    *,
    segment_page_bytes: Sequence[int] | None = None,
    device_num_blocks: int | None = None,
    stream: torch.cuda.Stream | None = None,
) -> None:
    """copy_blocks through aegkv_copy_blocks_noalloc: the library allocates
    nothing for the call (its descriptor goes to a fixed device array), for
    callers that cannot allocate. At most NOALLOC_MAX_SEGMENTS segments and
    NOALLOC_MAX_PAIRS pairs (ValueError beyond). Calls that overlap on one
    device from different streams or threads race on that array; calls on
    one stream are ordered."""
    dev, args = _copy_call_args(segments, src_block_ids, dst_block_ids,
                                segment_page_bytes, device_num_blocks, stream)
    lib = _lib.load()
    _lib.check(_call_on(dev, lambda: lib.aegkv_copy_blocks_noalloc(*args)))


def load_slices(dst: Sequence[torch.Tensor], src: Sequence[torch.Tensor], *, mode="auto",
                stream: torch.cuda.Stream | None = None) -> None:
    """dst[i] <- src[i] byte for byte for every i, pinned host -> device, in
    one aegkv_load_slices call: the weight load of a model switch, where the
    reference runs one `slice_storage.copy_(tensors_storage,
    non_blocking=True)` per tensors content
    (aegaeon/loader/quick_loader.py:325-340). mode "direct" (and "auto"):
    one kernel reads the host memory over PCIe; "staged": one runtime DMA
    copy per slice. Runs on `stream` (default: the current stream of dst's
    device)."""
    if len(dst) != len(src):
        raise ValueError(f"{len(dst)} target slices for {len(src)} source slices")
    if not dst:
        return
    dev = dst[0].device
    sizes = []
    for i, (d, h) in enumerate(zip(dst, src)):
        _require_device(d, f"target slice {i}")
        _require_host(h, f"source slice {i}")
        if d.device != dev:
            raise ValueError("all target slices must live on one device")
        if _tensor_bytes(d) != _tensor_bytes(h):
            raise ValueError(f"slice {i}: {_tensor_bytes(h)} source bytes for "
                             f"{_tensor_bytes(d)} target bytes")
        sizes.append(_tensor_bytes(d))
    n = len(dst)
    d_ptrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in dst])
    s_ptrs = (ctypes.c_void_p * n)(*[t.data_ptr() for t in src])
    b = np.ascontiguousarray(np.array(sizes, np.int64))
    lib = _lib.load()
    _lib.check(_call_on(dev, lambda: lib.aegkv_load_slices(
        n, d_ptrs, s_ptrs, _p64(b), _mode(mode), _stream_ptr(dev, stream))))


def migrate_blocks(
    src_segments: Sequence[torch.Tensor],
    dst_segments: Sequence[torch.Tensor],
    src_block_ids,
    dst_block_ids,
    *,
    segment_page_bytes: Sequence[int] | None = None,
    stream: torch.cuda.Stream | None = None,
    guard: torch.Tensor | None = None,
    guard_index: int = 0,
) -> None:
    """Whole-block copy from one cache to another of the same layout:
    dst_segments[s][dst[i]] := src_segments[s][src[i]] (aegkv_migrate_blocks).

    The reference plans this move (aegaeon/block_manager.py:1527-1601,
    aegaeon/worker.py:2420-2445) but leaves it unimplemented. The source
    tensors may be another engine's cache on this GPU, tensors received from
    another process (torch.multiprocessing, a HIP IPC memory handle), or a
    peer GPU's cache with peer access enabled; the work runs on the target
    cache's device. Each segment is viewed as [num_blocks, page] bytes; by
    default the page is the tensor's bytes / size(0), equal for both caches.
    guard: a move guard word, as for SegmentLayout.swap.
    """
    if not src_segments or len(src_segments) != len(dst_segments):
        raise ValueError("one source and one target tensor per segment are required")
    if segment_page_bytes is None:
        table = _lib.hostargs().segment_table
        st, dt = table(src_segments, None), table(dst_segments, None)
        if st is not None and dt is not None and st[3] == dt[3]:
            src, n = _id_arg(src_block_ids)
            dst, n_ids = _id_arg(dst_block_ids)
            if n != n_ids:
                raise ValueError("src and dst id lists differ in length")
            gp = _guard_ptr(guard, guard_index, "guard")
            dev = dst_segments[0].device
            lib = _lib.load()
            _lib.check(_call_on(dev, lambda: lib.aegkv_migrate_blocks(
                len(dt[2]) // 8, st[2], dt[2], dt[3], st[1], dt[1], n, src, dst, gp,
                _stream_ptr(dev, stream))))
            return
    dev = dst_segments[0].device
    for i, (a, b) in enumerate(zip(src_segments, dst_segments)):
        _require_device(a, f"source segment {i}")
        _require_device(b, f"target segment {i}")
        if b.device != dev:
            raise ValueError("all target segments must live on one device")
    n_src = src_segments[0].size(0)
    n_dst = dst_segments[0].size(0)
    if segment_page_bytes is None:
        segment_page_bytes = [_tensor_bytes(t) // n_dst for t in dst_segments]
    page = _i64(segment_page_bytes)
    if page.size != len(dst_segments):
        raise ValueError("segment_page_bytes must have one entry per segment")
    for i, (a, b) in enumerate(zip(src_segments, dst_segments)):
        if _tensor_bytes(a) < int(page[i]) * n_src or _tensor_bytes(b) < int(page[i]) * n_dst:
            raise ValueError(f"segment {i} is smaller than its block count x page")
    src = _i64(src_block_ids)
    dst = _i64(dst_block_ids)
    if src.shape != dst.shape:
        raise ValueError("src and dst id lists differ in length")
    sb = (ctypes.c_void_p * len(src_segments))(*[t.data_ptr() for t in src_segments])
    db = (ctypes.c_void_p * len(dst_segments))(*[t.data_ptr() for t in dst_segments])
    gp = _guard_ptr(guard, guard_index, "guard")
    lib = _lib.load()
    rc = _call_on(dev, lambda: lib.aegkv_migrate_blocks(
        len(dst_segments), sb, db, _p64(page), int(n_src), int(n_dst), src.size, _p64(src),
        _p64(dst), gp, _stream_ptr(dev, stream)))
    _lib.check(rc)


class _OwnedStream(torch.cuda.ExternalStream):
    """A torch stream over a HIP stream from aegkv_stream_create that
    destroys the HIP stream when the object goes (or on _aegkv_close()).
    weakref.finalize is not used: its callback was seen not to run for
    torch stream objects. Once closed, the stream's handle and its
    synchronize / query / wait / record methods raise instead of handing
    the runtime a destroyed stream."""

    def __init__(self, stream_ptr: int, device=None):
        self._aegkv_ptr = stream_ptr

    def _aegkv_close(self) -> None:
        ptr, self._aegkv_ptr = getattr(self, "_aegkv_ptr", None), None
        if ptr:
            _lib.check(_lib.load().aegkv_stream_destroy(ctypes.c_void_p(ptr)))

    def _aegkv_require_open(self) -> None:
        if getattr(self, "_aegkv_ptr", None) is None:
            raise RuntimeError("this dedicated stream is closed")

    @property
    def closed(self) -> bool:
        return getattr(self, "_aegkv_ptr", None) is None

    @property
    def cuda_stream(self):
        self._aegkv_require_open()
        return super().cuda_stream

    def synchronize(self):
        self._aegkv_require_open()
        return super().synchronize()

    def query(self):
        self._aegkv_require_open()
        return super().query()

    def wait_event(self, event):
        self._aegkv_require_open()
        return super().wait_event(event)

    def wait_stream(self, stream):
        self._aegkv_require_open()
        return super().wait_stream(stream)

    def record_event(self, event=None):
        self._aegkv_require_open()
        return super().record_event(event)

    def __del__(self, _finalizing=sys.is_finalizing):
        # At interpreter exit the HIP runtime may already be torn down, and
        # the process is ending anyway: leave the stream to it. (The check is
        # bound at definition: module globals may be gone by then.)
        if _finalizing():
            return
        try:
            self._aegkv_close()
        except Exception:
            pass


CUS_PER_XCD = 32  # MI355X (gfx950): 8 XCDs of 32 CUs


def xcd_cu_mask(cus_per_xcd: int, first: int = 0,
                device: torch.device | None = None) -> list[int]:
    """CU mask words (for DedicatedStream(cu_mask=...)) that give a stream
    `cus_per_xcd` CUs on each of the 8 XCDs: mask bits i with
    first <= i % 32 < first + cus_per_xcd. The runtime spreads every run of
    8 consecutive mask bits over the 8 XCDs, one CU each (hardware ids read
    by workgroups of such streams show bits 0-7 on one CU per XCD, bits 0-31
    on four), so the CU count per XCD is what a mask sets; a mask cannot
    confine a stream to whole XCDs. The runtime takes runs of 8 or more bits
    starting at a multiple of 8, e.g. xcd_cu_mask(8) for the swap streams
    and xcd_cu_mask(24, first=8) for the rest."""
    if cus_per_xcd <= 0 or first < 0 or first + cus_per_xcd > CUS_PER_XCD:
        raise ValueError(f"CUs [{first}, {first + cus_per_xcd}) do not fit a "
                         f"{CUS_PER_XCD}-CU XCD")
    dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
    n = torch.cuda.get_device_properties(dev).multi_processor_count
    words = [0] * ((n + 31) // 32)
    for i in range(n):
        if first <= i % CUS_PER_XCD < first + cus_per_xcd:
            words[i // 32] |= 1 << (i % 32)
    return words


class DedicatedStream:
    """A HIP stream on a hardware queue of its own (aegkv_stream_create),
    usable wherever torch takes a stream through `.stream`.

    Plain streams (torch.cuda.Stream included) share the process's 4
    hardware queues, and two streams on one queue run their work one after
    the other; a swap-out and a swap-in on dedicated streams always overlap.
    With cu_mask (see xcd_cu_mask) its kernels run only on those CUs.
    Unlike torch's pool streams, a dedicated stream is a blocking stream: it
    synchronizes with the legacy default (null) stream, so work on it waits
    for the default stream's earlier work and the other way round.
    The HIP stream lives exactly as long as the `.stream` object (which this
    object holds): it is destroyed by close() or as soon as the last
    reference to `.stream` goes, after its queued work, so dropped streams
    do not keep hardware queues until a garbage collection.
    """

    def __init__(self, device: torch.device | None = None, cu_mask: Sequence[int] | None = None):
        dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        lib = _lib.load()
        ptr = ctypes.c_void_p()
        if cu_mask is None:
            _lib.check(_call_on(dev, lambda: lib.aegkv_stream_create(ctypes.byref(ptr))))
        else:
            words = np.ascontiguousarray(np.asarray(cu_mask, dtype=np.uint32).reshape(-1))
            arg = words.ctypes.data_as(ctypes.POINTER(ctypes.c_uint32))
            _lib.check(_call_on(dev, lambda: lib.aegkv_stream_create_masked(
                ctypes.byref(ptr), arg, int(words.size))))
        self.device = dev
        self.cu_mask = None if cu_mask is None else list(cu_mask)
        self.stream = _OwnedStream(ptr.value, device=dev)

    def close(self) -> None:
        self.stream._aegkv_close()


def host_pinned_usage() -> tuple[int, int]:
    """(pinned bytes the library holds, free bytes inside its uncached
    blocks), from aegkv_host_usage: live cached pools plus every uncached
    block kept, which is what counts against the host's cap on pinned
    memory."""
    pinned, free = ctypes.c_int64(), ctypes.c_int64()
    _lib.check(_lib.load().aegkv_host_usage(ctypes.byref(pinned), ctypes.byref(free)))
    return int(pinned.value), int(free.value)


def _free_pinned(ptr: int) -> None:
    rc = _lib.load().aegkv_host_free(ptr)
    if rc:
        raise _lib.AegkvError(rc, _lib.load().aegkv_last_error().decode(errors="replace"))


class PinnedHostPool:
    """A pinned, device-mapped host byte pool from aegkv_host_alloc.

    Counterpart of the reference's host KV pool (aegaeon/llm.py:1020-1040,
    aegaeon/worker.py:251-273), allocated pinned instead of registering an
    existing /dev/shm mapping. `tensor` is a uint8 view of the whole pool.
    The memory is released when the pool and every tensor viewing it are
    gone (views keep it alive), so a kernel can never be handed freed
    memory through a surviving view. Callers still wait for GPU work on the
    pool before dropping the last view.

    uncached=True allocates from the uncached system pool
    (AEGKV_HOST_UNCACHED): faster swaps, especially both directions at
    once, but the library keeps such memory mapped until the process ends
    and carves later uncached pools out of it. coherent=True allocates
    fine-grained coherent memory (AEGKV_HOST_COHERENT), for words the GPU and
    the host both write while kernels run (GuardWords).
    """

    def __init__(self, nbytes: int, uncached: bool = False, coherent: bool = False):
        if nbytes <= 0:
            raise ValueError("pool size must be positive")
        lib = _lib.load()
        ptr = ctypes.c_void_p()
        flags = (_lib.HOST_UNCACHED if uncached else 0) | (_lib.HOST_COHERENT if coherent else 0)
        _lib.check(lib.aegkv_host_alloc_flags(ctypes.byref(ptr), int(nbytes), flags))
        self.nbytes = int(nbytes)
        self.uncached = uncached
        self.coherent = coherent
        buf = (ctypes.c_uint8 * self.nbytes).from_address(ptr.value)
        fin = weakref.finalize(buf, _free_pinned, ptr.value)
        fin.atexit = False  # at interpreter exit the process releases it
        self.tensor = torch.frombuffer(buf, dtype=torch.uint8)

    def free(self) -> None:
        """Drop this pool's reference; the memory goes once no view remains."""
        self.tensor = None


class GuardWords:
    """Move guards: `num_words` uint64 words in coherent pinned host memory,
    zeroed, that the GPU and the host both read and write (one per stream
    that waits on fences; KVSwapper keeps one per swap stream).

    A fence wait sets its stream's guard when it gives up (1) or when the
    word it waits on carries the failure mark (2); guarded swaps and
    migrations then move nothing, and guarded signals and publishes mark
    the completion they report as failed (FENCE_FAILED), so every consumer
    sees the failure. The library never clears a guard.
    """

    def __init__(self, num_words: int = 2):
        if num_words <= 0:
            raise ValueError("num_words must be positive")
        self._pool = PinnedHostPool(8 * int(num_words), coherent=True)
        self.tensor = self._pool.tensor.view(torch.int64)
        self.tensor.zero_()
        self.num_words = int(num_words)

    def ptr(self, index: int) -> int:
        return _guard_ptr(self.tensor, index, "guard")

    def value(self, index: int) -> int:
        """The guard as the host sees it now (0: not set)."""
        if not 0 <= index < self.num_words:
            raise ValueError(f"guard index {index} outside [0, {self.num_words})")
        return int(self.tensor[index])


def _fence_word(words: torch.Tensor, index: int, what: str) -> int:
    if words.dtype != torch.int64 or words.dim() != 1:
        raise ValueError(f"{what} must be a 1-D int64 tensor")
    if not words.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    if not 0 <= index < words.numel():
        raise ValueError(f"{what} index {index} outside [0, {words.numel()})")
    return words.data_ptr() + 8 * index


def _fence_value(value: int) -> int:
    if not 0 < value < FENCE_FAILED:
        raise ValueError("fence values are positive and below 2**62 (bit 62 marks a failed move)")
    return int(value)


def fence_signal(words: torch.Tensor, index: int, value: int, *,
                 guard: torch.Tensor | None = None, guard_index: int = 0,
                 stream: torch.cuda.Stream | None = None) -> None:
    """Raise words[index] to at least `value` once every operation
    enqueued earlier on `stream` (default: the current stream) has finished
    (aegkv_fence_signal). The counterpart of recording an interprocess event
    behind a swap (aegaeon/worker.py:2331,2349). With a move guard that is
    set by then, the word is raised to value | FENCE_FAILED instead.

    words: a 1-D int64 tensor on the device, e.g. one shared with other
    processes through torch.multiprocessing (a HIP IPC memory handle).
    """
    value = _fence_value(value)
    ptr = _fence_word(words, index, "fence words")
    gp = _guard_ptr(guard, guard_index, "guard")
    dev = words.device
    if dev.type != "cuda":
        raise ValueError("fence words must live on the device")
    lib = _lib.load()
    rc = _call_on(dev, lambda: lib.aegkv_fence_signal(ptr, value, gp, _stream_ptr(dev, stream)))
    _lib.check(rc)


def fence_wait(words: torch.Tensor, index: int, value: int, guard: torch.Tensor,
               guard_index: int = 0, *, timeout_s: float = 30.0,
               stream: torch.cuda.Stream | None = None) -> None:
    """Make every later operation on `stream` wait until words[index] >=
    value (aegkv_fence_wait); the counterpart of waiting on another worker's
    interprocess event (aegaeon/worker.py:2351-2394).

    A wait that has polled for `timeout_s` seconds gives up and sets the
    move guard guard[guard_index] to 1; a word that carries FENCE_FAILED
    ends the wait at once and sets it to 2. The stream then goes on, but
    guarded moves after the wait move nothing and guarded signals and
    publishes report failure. guard: GuardWords.tensor, or a device int64
    tensor on the words' device; the guard is never cleared here.
    """
    value = _fence_value(value)
    ptr = _fence_word(words, index, "fence words")
    gp = _guard_ptr(guard, guard_index, "guard")
    dev = words.device
    if dev.type != "cuda":
        raise ValueError("fence words must live on the device")
    if guard.device.type == "cuda" and guard.device != dev:
        raise ValueError("fence words and a device guard must live on one device")
    timeout_us = int(timeout_s * 1e6)
    lib = _lib.load()
    rc = _call_on(dev, lambda: lib.aegkv_fence_wait(ptr, value, timeout_us, gp,
                                                    _stream_ptr(dev, stream)))
    _lib.check(rc)


def guard_merge(guard: torch.Tensor, index: int, source: torch.Tensor, source_index: int, *,
                device: torch.device | None = None,
                stream: torch.cuda.Stream | None = None) -> None:
    """Once `stream` (default: the current stream of `device`) reaches it, set
    guard[index] to 2 (a source failed) when source[source_index] is set
    (aegkv_guard_merge): a consumer that waits on a producer's completion
    event inherits the producer's failure."""
    gp = _guard_ptr(guard, index, "guard")
    sp = _guard_ptr(source, source_index, "source guard")
    dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
    lib = _lib.load()
    _lib.check(_call_on(dev, lambda: lib.aegkv_guard_merge(gp, sp, _stream_ptr(dev, stream))))


class HostFenceWords:
    """Host fence words shared by processes: a file in /dev/shm of
    `num_words` uint64 counters, mapped shared. Workers raise them behind
    their swaps (fence_publish) and a controller in any process reads them
    (fence_host_wait), where the reference's controller polls the workers'
    interprocess events (aegaeon/block_manager.py:804-851).

    HostFenceWords(n) creates a new zeroed file (its `name` is the path) and
    removes it on close(); HostFenceWords.attach(name) maps an existing one.
    close() first waits for every stream that a publish into these words was
    enqueued on, so no host function writes into an unmapped page.
    """

    def __init__(self, num_words: int | None = None, *, _name: str | None = None):
        import mmap
        import os
        import uuid

        if _name is None:
            if num_words is None or num_words <= 0:
                raise ValueError("num_words must be positive")
            name = f"/dev/shm/aegkv-fence-{os.getpid()}-{uuid.uuid4().hex[:12]}"
            fd = os.open(name, os.O_RDWR | os.O_CREAT | os.O_EXCL, 0o600)
            try:
                os.ftruncate(fd, 8 * int(num_words))
            except BaseException:
                os.close(fd)
                os.unlink(name)
                raise
            self.owner = True
        else:
            name = _name
            # a publish writes through the mapping: only this library's own files
            if (os.path.dirname(os.path.abspath(name)) != "/dev/shm"
                    or not os.path.basename(name).startswith("aegkv-fence-")):
                raise ValueError(f"{name} is not a host fence file (/dev/shm/aegkv-fence-*)")
            fd = os.open(name, os.O_RDWR)
            self.owner = False
        try:
            size = os.fstat(fd).st_size
            if size < 8 or size % 8:
                raise ValueError(f"{name} is not a file of fence words ({size} bytes)")
            self._mm = mmap.mmap(fd, size, mmap.MAP_SHARED, mmap.PROT_READ | mmap.PROT_WRITE)
        finally:
            os.close(fd)
        self.name = name
        self.num_words = size // 8
        self._anchor = ctypes.c_char.from_buffer(self._mm)
        self._base = ctypes.addressof(self._anchor)
        self.words = np.frombuffer(self._mm, dtype=np.uint64)
        # streams holding publishes into these words: stream handle -> stream
        self._publishers: dict = {}
        self._publishers_lock = threading.Lock()

    @classmethod
    def attach(cls, name: str) -> "HostFenceWords":
        return cls(_name=name)

    def ptr(self, index: int) -> int:
        if self._mm is None:
            raise ValueError("these host fence words are closed")
        if not 0 <= index < self.num_words:
            raise ValueError(f"host fence index {index} outside [0, {self.num_words})")
        return self._base + 8 * index

    def _note_publisher(self, stream: torch.cuda.Stream) -> None:
        with self._publishers_lock:
            self._publishers[stream.cuda_stream] = stream

    def close(self) -> None:
        """Wait for the streams that publishes into these words were enqueued
        on (a closed dedicated stream was synchronized when it closed), then
        unmap, and remove the file for the creator."""
        import os

        if self._mm is None:
            return
        with self._publishers_lock:
            streams, self._publishers = list(self._publishers.values()), {}
        for st in streams:
            if not getattr(st, "closed", False):
                st.synchronize()
        self.words = None
        self._anchor = None
        self._mm.close()
        self._mm = None
        if self.owner:
            try:
                os.unlink(self.name)
            except FileNotFoundError:
                pass


_attached_lock = threading.Lock()
_attached: dict = {}


def attached_host_fence_words(name: str) -> HostFenceWords:
    """This process's mapping of the host fence words at `name` (mapped once,
    kept until the process ends)."""
    with _attached_lock:
        hw = _attached.get(name)
        if hw is None or hw._mm is None:
            hw = HostFenceWords.attach(name)
            _attached[name] = hw
        return hw


def fence_publish(host_words: HostFenceWords, index: int, value: int, *,
                  guard: torch.Tensor | None = None, guard_index: int = 0,
                  device: torch.device | None = None,
                  stream: torch.cuda.Stream | None = None) -> None:
    """Raise host_words[index] to at least `value` once every operation
    enqueued earlier on `stream` (default: the current stream of `device`)
    has finished (aegkv_fence_publish, a host function on the stream). With
    a move guard (GuardWords.tensor: the host function reads it) that is set
    by then, the word is raised to value | FENCE_FAILED instead."""
    value = _fence_value(value)
    ptr = host_words.ptr(index)
    gp = _guard_ptr(guard, guard_index, "guard")
    if guard is not None and guard.device.type != "cpu":
        raise ValueError("a published fence's guard must be pinned host memory (GuardWords)")
    dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
    st = stream if stream is not None else torch.cuda.current_stream(dev)
    lib = _lib.load()
    rc = _call_on(dev, lambda: lib.aegkv_fence_publish(ptr, value, gp, st.cuda_stream))
    _lib.check(rc)
    host_words._note_publisher(st)


def fence_host_wait(host_words: HostFenceWords, index: int, value: int,
                    timeout_s: float = 0.0) -> bool:
    """True once host_words[index] >= value; waits on this thread for at most
    timeout_s seconds (0: look once). No GPU call; the GIL is released.
    Raises MoveFailedError when the word carries the failure mark."""
    value = _fence_value(value)
    if timeout_s < 0:
        raise ValueError("timeout_s must be >= 0")
    rc = _lib.load().aegkv_fence_host_wait(host_words.ptr(index), value,
                                           int(timeout_s * 1e6))
    if rc < 0:
        _lib.check(rc)
    if rc == 2:
        raise MoveFailedError(f"host fence {host_words.name}[{index}] carries the failure mark: "
                              f"the move it counts (value {value}) or one before it on its "
                              "stream moved nothing")
    return rc == 1


# ---- quantised caches ---------------------------------------------------------

_FORMATS = {"mxfp4": _lib.FORMAT_MXFP4, "mxfp8": _lib.FORMAT_MXFP8}
_DTYPES = {torch.bfloat16: _lib.DTYPE_BFLOAT16, torch.float16: _lib.DTYPE_FLOAT16,
           torch.float32: _lib.DTYPE_FLOAT32}


def quant_page_bytes(fmt: str, block_size: int, kv_heads: int, head_dim: int) -> int:
    """Bytes of one block of K (or of V) in a quantised cache
    (aegkv_quant_page_bytes): "mxfp4" holds a value in 4 bits, "mxfp8" in 8,
    both with one scale byte for 32 values of a head."""
    if fmt not in _FORMATS:
        raise ValueError(f"unknown cache format {fmt!r}")
    n = ctypes.c_int64()
    _lib.check(_lib.load().aegkv_quant_page_bytes(_FORMATS[fmt], int(block_size), int(kv_heads),
                                                  int(head_dim), ctypes.byref(n)))
    return int(n.value)


class QuantCache:
    """K and V of one layer in a quantised format, as pages of a paged cache.

    k_pages and v_pages are device tensors of num_blocks pages each, of any
    element type (a composite cache's backing tensors over
    layout.quant_kv_tensor_specs serve as they are), which swaps, copies and
    migrations move like any other segment. A page holds block_size tokens (16,
    32, 64 or 128) of kv_heads heads, 64, 128 or 256 values wide; its layout is
    described in include/aegkv.h.
    """

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, *, kv_heads: int,
                 head_dim: int, block_size: int, fmt: str = "mxfp4"):
        self.page_bytes = quant_page_bytes(fmt, block_size, kv_heads, head_dim)
        for t, what in ((k_pages, "k_pages"), (v_pages, "v_pages")):
            _require_device(t, what)
            if _tensor_bytes(t) == 0 or _tensor_bytes(t) % self.page_bytes:
                raise ValueError(f"{what} of {_tensor_bytes(t)} bytes are no whole pages of "
                                 f"{self.page_bytes}")
        if k_pages.device != v_pages.device or _tensor_bytes(k_pages) != _tensor_bytes(v_pages):
            raise ValueError("k_pages and v_pages must be equally large and on one device")
        self.k_pages, self.v_pages = k_pages, v_pages
        self.kv_heads, self.head_dim = int(kv_heads), int(head_dim)
        self.block_size, self.fmt = int(block_size), fmt
        self.num_blocks = _tensor_bytes(k_pages) // self.page_bytes
        self.device = k_pages.device
        self._args = (_FORMATS[fmt], self.head_dim, k_pages.data_ptr(), v_pages.data_ptr())
        # CacheArgs of csrc/hostargs.cpp
        self._packed = struct.pack(
            "11q", *(_lib.address(f"aegkv_quant_{op}") for op in ("write", "read", "attend")),
            *self._args, self.kv_heads, self.block_size, self.num_blocks, self.device.index)


class CacheBatch:
    """A batch over a quantised cache: which blocks its sequences hold, and how
    attention over them is shared out (aegkv_batch_plan). One batch serves all
    layers of a model step.

    block_tables: a list of block ids for each sequence, or a 2-D array with a row
    each; column c holds the positions [c * block_size, (c + 1) * block_size), -1
    marks a released column (as BlockTable.group_blocks does), and columns behind
    the sequence's last are ignored. seq_lens counts all tokens of a
    sequence, new_lens those at its end that are new: the ones quant_write
    writes and quant_attend takes as queries. A query at position p sees the
    positions j <= p with p - j < window (0: all) or j < sinks.

    Everything is checked here, once (ValueError). update() puts another batch in
    its place, also for calls captured into a graph, if it fits the room
    that max_seqs, max_columns (of all block tables) and max_tokens (new ones) asked
    for and its sequences have as many rows (new tokens times heads / kv_heads) as
    the first batch's: up to 16, up to 64, or more. The room may be what the first
    batch holds itself. Without any (all 0) a batch takes less memory, and an update
    of the same lengths.
    """

    def __init__(self, block_tables, seq_lens, new_lens, *, num_blocks: int, block_size: int,
                 kv_heads: int, heads: int | None = None, window: int = 0, sinks: int = 0,
                 max_seqs: int = 0, max_columns: int = 0, max_tokens: int = 0,
                 device: torch.device | None = None, stream: torch.cuda.Stream | None = None):
        self.num_blocks, self.block_size = int(num_blocks), int(block_size)
        self.kv_heads = int(kv_heads)
        self.heads = self.kv_heads if heads is None else int(heads)
        self.window, self.sinks = int(window), int(sinks)
        self._room = (int(max_seqs), int(max_columns), int(max_tokens))
        self._host = None
        self._make(block_tables, seq_lens, new_lens, update=0)
        self.device = torch.device(device if device is not None else "cuda")
        if self.device.type != "cuda":
            raise ValueError(f"a batch lives on a device (HIP), not on {self.device}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._workspace = {}    # bytes by head width
        for d in (64, 128, 256):
            n = ctypes.c_int64()
            _lib.check(_lib.load().aegkv_quant_attend_workspace(self._host_ptr, d,
                                                                ctypes.byref(n)))
            self._workspace[d] = int(n.value)
        self._used: dict = {}     # raw stream -> stream of calls made elsewhere than at home
        self._home = None
        _require_stream(self.device, stream)
        with torch.cuda.device(self.device):
            st = stream if stream is not None else torch.cuda.current_stream()
            if torch.cuda.is_current_stream_capturing() or stream is not None and _capturing(st):
                raise ValueError("a batch cannot be made while a stream is captured")
            with torch.cuda.stream(st):
                self._plan = torch.empty(self._host.size, dtype=torch.uint8, device=self.device)
                self._pool = st     # whose memory pool the plan goes back to
                self._upload(st, self._pinned())

    def _make(self, block_tables, seq_lens, new_lens, update: int) -> None:
        if isinstance(block_tables, (torch.Tensor, np.ndarray)):
            if block_tables.ndim != 2:
                raise ValueError("block tables are a list a sequence or a 2-D array")
            offsets = np.arange(len(block_tables) + 1, dtype=np.int64) * block_tables.shape[1]
            ids = _i64(block_tables)
        else:
            rows = [_i64(t) for t in block_tables]
            offsets = np.zeros(len(rows) + 1, np.int64)
            np.cumsum([r.size for r in rows], out=offsets[1:])
            ids = np.concatenate(rows) if rows else np.zeros(0, np.int64)
        lens, new = _i64(seq_lens), _i64(new_lens)
        if not offsets.size - 1 == lens.size == new.size:
            raise ValueError(f"{offsets.size - 1} block tables, {lens.size} lengths and "
                             f"{new.size} new lengths")
        lib = _lib.load()
        args = (lens.size, _p64(offsets), _p64(ids), _p64(lens), _p64(new), self.num_blocks,
                self.block_size, self.kv_heads, self.heads, self.window, self.sinks, *self._room,
                update)
        n = ctypes.c_int64(self._host.size if update else 0)
        host = self._host
        if not update:
            _lib.check(lib.aegkv_batch_plan(*args, None, ctypes.byref(n)))
            host = np.zeros(n.value, np.uint8)
        _lib.check(lib.aegkv_batch_plan(*args, host.ctypes.data, ctypes.byref(n)))
        self._host = host
        self._host_ptr = host.ctypes.data
        self.num_seqs, self.num_tokens = int(lens.size), int(new.sum())
        self.read_tokens = int(lens.sum())

    def _pinned(self) -> torch.Tensor:
        return torch.empty(self._host.size, dtype=torch.uint8, pin_memory=True)

    def _upload(self, st: torch.cuda.Stream, pinned: torch.Tensor) -> None:
        try:
            pinned.numpy()[:] = self._host
            self._plan.copy_(pinned, non_blocking=True)
            self._uploaded = torch.cuda.Event()
            self._uploaded.record(st)
        except BaseException:
            # calls go by the host's plan, kernels by the device's: now that they may
            # differ, nothing is taken over this batch any more ("no plan")
            self._host[:8] = 0
            raise
        self._home, self._stream = st, st.cuda_stream
        # BatchArgs of csrc/hostargs.cpp
        self._packed = struct.pack(
            "13q", self._host_ptr, self._plan.data_ptr(), self._stream, self.kv_heads, self.heads,
            self.block_size, self.num_blocks, self.device.index, self.num_tokens,
            self.read_tokens, *self._workspace.values())

    def update(self, block_tables, seq_lens, new_lens, *,
               stream: torch.cuda.Stream | None = None) -> None:
        """Put another batch over the same cache in this one's place. The change
        is enqueued on `stream` (default: the current one) behind every call
        made over this batch; a graph that holds such calls is replayed on that
        stream, or ordered before and behind it by the caller."""
        _require_stream(self.device, stream)
        with torch.cuda.device(self.device):
            st = stream if stream is not None else torch.cuda.current_stream()
            others = [other for other in (self._home, *self._used.values())
                      if _alive(other) and other.cuda_stream != st.cuda_stream]
            if torch.cuda.is_current_stream_capturing() or any(map(_capturing, (st, *others))):
                raise ValueError("a batch is updated outside the capture; the graph's calls "
                                 "find what it holds when they are replayed")
            with torch.cuda.stream(st):
                for other in others:
                    st.wait_event(other.record_event())
                pinned = self._pinned()
                self._make(block_tables, seq_lens, new_lens, update=1)
                self._upload(st, pinned)
                self._used.clear()

    def _enter(self, raw: int, stream: torch.cuda.Stream | None):
        """Order a call on the raw stream behind the upload. The stream, where
        the call is to be noted by _leave."""
        if raw == self._stream and _alive(self._home):
            return None     # (a new stream may have the handle of one that is closed)
        st = stream if stream is not None else torch.cuda.current_stream(self.device)
        if _capturing(st):
            return None     # capture begins behind a synchronize
        if _alive(self._home):  # a closed stream was waited for
            st.wait_event(self._uploaded)
        return st

    def _leave(self, st: torch.cuda.Stream | None) -> None:
        if st is not None:
            self._used[st.cuda_stream] = st

    def __del__(self, _finalizing=sys.is_finalizing):
        # The plan's memory goes back to the pool of the stream it was made on,
        # wherever updates have moved the batch since: that stream waits for the
        # calls on all others that read it. (Not Tensor.record_stream, which records
        # an event on them when the memory goes, when they may be closed.)
        if _finalizing() or getattr(self, "_home", None) is None:
            return
        try:
            pool = self._pool
            raw = pool.cuda_stream if _alive(pool) else None
            others = [st for st in (self._home, *self._used.values())
                      if _alive(st) and st.cuda_stream != raw]
            if not others:
                return
            if any(_capturing(st) for st in (*others, *((pool,) if raw is not None else ()))):
                _kept.append(self._plan)    # no stream may wait for a captured one
                return
            for st in others:
                if raw is not None:
                    pool.wait_event(st.record_event())
                else:
                    st.synchronize()
        except Exception:
            _kept.append(self._plan)


_kept: list = []    # plans that no stream could be ordered behind: never reused


def _alive(stream: torch.cuda.Stream) -> bool:
    """Whether a stream may still be handed to the runtime (a closed dedicated
    stream, whose work was waited for, may not)."""
    return not getattr(stream, "closed", False)


def _require_stream(device: torch.device, stream: torch.cuda.Stream | None) -> None:
    if stream is not None and stream.device != device:
        raise ValueError(f"a stream of {stream.device} for work on {device}")


def _capturing(stream: torch.cuda.Stream) -> bool:
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


def _quant_call(cache: QuantCache, batch: CacheBatch, stream: torch.cuda.Stream | None):
    if (batch.block_size, batch.kv_heads) != (cache.block_size, cache.kv_heads):
        raise ValueError(f"a batch of {batch.block_size}-token blocks and {batch.kv_heads} KV "
                         f"heads over a cache of {cache.block_size} and {cache.kv_heads}")
    if batch.num_blocks > cache.num_blocks:
        raise ValueError(f"a batch over {batch.num_blocks} blocks, a cache of {cache.num_blocks}")
    if batch.device != cache.device:
        raise ValueError(f"a batch on {batch.device}, a cache on {cache.device}")
    _require_stream(cache.device, stream)


def _here(cache: QuantCache) -> tuple:
    """(raw current stream of the cache's device, current device)."""
    return torch._C._cuda_getCurrentRawStream(cache.device.index), torch._C._cuda_getDevice()


def _answer(done):
    """What a native call gave: its result, or the status of the library."""
    if type(done) is int:
        _lib.check(done)
    return done


def _rows_arg(t: torch.Tensor, what: str, heads: int, cache: QuantCache, dtypes):
    """(pointer, token stride, head stride) of a [tokens, heads, head_dim] tensor."""
    if t.device != cache.device:
        raise ValueError(f"{what} on {t.device}, the cache on {cache.device}")
    if t.dim() != 3 or t.size(1) != heads or t.size(2) != cache.head_dim:
        raise ValueError(f"{what} must be [tokens, {heads}, {cache.head_dim}], not "
                         f"{list(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{what} of {t.dtype} is not supported")
    if t.numel() and t.stride(2) != 1:
        raise ValueError(f"{what}: the last axis must be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, which these operators do not give")
    if torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{what} carries a tangent, which these operators do not take on")
    return t.data_ptr(), t.stride(0), t.stride(1)


def _on_stream(cache: QuantCache, batch: CacheBatch, stream, fn) -> None:
    def call():
        raw = _stream_ptr(cache.device, stream)
        st = batch._enter(raw, stream)
        try:
            _lib.check(fn(raw))
        finally:
            batch._leave(st)    # of several launches the first may be on its way

    _call_on(cache.device, call)


def _empty_on(stream, *args, **kwargs) -> torch.Tensor:
    """A tensor of `stream`'s (default: the current one's) memory pool."""
    if stream is None:
        return torch.empty(*args, **kwargs)
    with torch.cuda.stream(stream):
        return torch.empty(*args, **kwargs)


def quant_write(cache: QuantCache, batch: CacheBatch, k: torch.Tensor, v: torch.Tensor, *,
                stream: torch.cuda.Stream | None = None) -> None:
    """Write the batch's new tokens into the cache (aegkv_quant_write).

    k, v: [tokens, kv_heads, head_dim] of bfloat16, float16 or float32, with any
    strides on the first two axes (slices of a fused projection, say); row i is
    the batch's i-th new token, and rows behind the last are not read. Every 32
    values share the smallest power-of-two scale under which the largest fits the format,
    and each takes its nearest code, ties to even. A group with a NaN or an
    infinity reads back as NaN.
    """
    if stream is None and _alive(batch._home):
        done = _lib.hostargs().quant_write(cache._packed, batch._packed, k, v, *_here(cache))
        if done is not None:
            _answer(done)
            return
    _quant_call(cache, batch, stream)
    kp = _rows_arg(k, "k", cache.kv_heads, cache, _DTYPES)
    vp = _rows_arg(v, "v", cache.kv_heads, cache, _DTYPES)
    if k.dtype != v.dtype or k.size(0) != v.size(0):
        raise ValueError(f"k and v differ: {k.size(0)} tokens of {k.dtype}, {v.size(0)} of "
                         f"{v.dtype}")
    lib = _lib.load()
    _on_stream(cache, batch, stream, lambda raw: lib.aegkv_quant_write(
        batch._host_ptr, batch._plan.data_ptr(), *cache._args, *kp, *vp, k.size(0),
        _DTYPES[k.dtype], raw))


def quant_read(cache: QuantCache, batch: CacheBatch, *, tokens: str = "all",
               dtype: torch.dtype = torch.bfloat16,
               out: tuple[torch.Tensor, torch.Tensor] | None = None,
               stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V of the batch's tokens as values of `dtype` (aegkv_quant_read):
    [tokens, kv_heads, head_dim] each, all tokens of the sequences one after
    another ("all"), or the new ones ("new"). `out`: two tensors to read into (their
    type counts); rows behind the last token are left as they were."""
    if tokens not in ("all", "new"):
        raise ValueError(f"tokens are 'all' or 'new', not {tokens!r}")
    if stream is None and _alive(batch._home):
        done = _lib.hostargs().quant_read(cache._packed, batch._packed, tokens == "new",
                                          _DTYPES.get(dtype) if out is None else out,
                                          *_here(cache))
        if done is not None:
            return _answer(done)
    _quant_call(cache, batch, stream)
    n = batch.read_tokens if tokens == "all" else batch.num_tokens
    if out is None:
        if dtype not in _DTYPES:
            raise ValueError(f"reading as {dtype} is not supported")
        shape = (n, cache.kv_heads, cache.head_dim)
        out = tuple(_empty_on(stream, shape, dtype=dtype, device=cache.device) for _ in range(2))
    k, v = out
    kp = _rows_arg(k, "k", cache.kv_heads, cache, _DTYPES)
    vp = _rows_arg(v, "v", cache.kv_heads, cache, _DTYPES)
    if k.dtype != v.dtype or k.size(0) != v.size(0):
        raise ValueError(f"k and v differ: {k.size(0)} tokens of {k.dtype}, {v.size(0)} of "
                         f"{v.dtype}")
    lib = _lib.load()
    _on_stream(cache, batch, stream, lambda raw: lib.aegkv_quant_read(
        batch._host_ptr, batch._plan.data_ptr(), *cache._args, 1 if tokens == "new" else 0,
        *kp, *vp, k.size(0), _DTYPES[k.dtype], raw))
    return k, v


def quant_attend(cache: QuantCache, batch: CacheBatch, q: torch.Tensor, *,
                 scale: float | None = None, out: torch.Tensor | None = None,
                 stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Attention of the batch's new tokens over the cache (aegkv_quant_attend),
    for single tokens, chunks and whole prompts alike, also side by side.

    q: [tokens, heads, head_dim] of bfloat16 or float16, row i the query of the
    batch's i-th new token, whose K and V are in the cache already (quant_write).
    scale: of the scores, head_dim ** -0.5 by default. `out` (q itself is fine, other
    overlaps are refused) takes the result; rows behind the batch's last token are left as they were.
    """
    if stream is None and _alive(batch._home):
        done = _lib.hostargs().quant_attend(cache._packed, batch._packed, q, out, scale,
                                            *_here(cache))
        if done is not None:
            return _answer(done)
    _quant_call(cache, batch, stream)
    qp = _rows_arg(q, "q", batch.heads, cache, (torch.bfloat16, torch.float16))
    if out is None:
        out = _empty_on(stream, q.shape, dtype=q.dtype, device=q.device)
    op = _rows_arg(out, "out", batch.heads, cache, (q.dtype,))
    if out.size(0) != q.size(0):
        raise ValueError(f"{q.size(0)} queries, {out.size(0)} rows of out")
    lib = _lib.load()
    d = cache.head_dim
    size = batch._workspace[d]
    work = _empty_on(stream, size, dtype=torch.uint8, device=q.device) if size else None
    _on_stream(cache, batch, stream, lambda raw: lib.aegkv_quant_attend(
        batch._host_ptr, batch._plan.data_ptr(), *cache._args, *qp, *op, q.size(0),
        _DTYPES[q.dtype], d ** -0.5 if scale is None else float(scale),
        work.data_ptr() if size else None, size, raw))
    return out
