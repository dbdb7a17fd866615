"""Torch-tensor wrappers over the C ABI (include/kvssd_b200.h).

Every function here launches CUDA kernels from libkvssd_b200 on the current CUDA stream of
the tensors' device; none has a CPU path. Tensors are passed by data pointer, so callers must
pass contiguous CUDA tensors (the wrappers check and raise otherwise).
"""

from __future__ import annotations

import ctypes
import math
import threading

import torch

from . import _native

_QUERY_DTYPES = {
    torch.float32: _native.Q_F32,
    torch.float16: _native.Q_F16,
    torch.bfloat16: _native.Q_BF16,
    torch.float64: _native.Q_F64,
}

_WORKSPACE_HEADER = 2048


class _Workspaces:
    """Per-(device, stream) decode workspaces, grown on demand and reused across calls.

    Reuse is safe because calls that share a workspace are ordered on one stream. A workspace
    is zeroed once at allocation: the header's device status word (it accumulates until read),
    the fused combine's epoch and the part words, whose epoch tags must not match a future call.
    A workspace that a larger one replaces is kept: a captured graph may hold its address, for its
    parts or for its status word. As sizes double, all of them are smaller than the one in use.
    """

    def __init__(self) -> None:
        self._lock = threading.Lock()
        self._buffers: dict[tuple[int, int], torch.Tensor] = {}
        self._replaced: dict[tuple[int, int], list[torch.Tensor]] = {}
        self._captured: set[tuple[int, int]] = set()  # zeroed by a graph, at each of its replays

    def get(self, device: torch.device, stream: torch.cuda.Stream, nbytes: int) -> torch.Tensor:
        key = (device.index, stream.cuda_stream)
        with self._lock:
            buf = self._buffers.get(key)
            if buf is None or buf.numel() < nbytes:
                size = max(nbytes, 1 << 20)
                if buf is not None:
                    size = max(size, 2 * buf.numel())
                old, buf = buf, torch.zeros(size, dtype=torch.uint8, device=device)
                capturing = torch.cuda.is_current_stream_capturing()
                if old is not None:
                    self._replaced.setdefault(key, []).append(old)
                    if not capturing:
                        buf[:4].copy_(old[:4])  # what has been flagged and not been read
                (self._captured.add if capturing else self._captured.discard)(key)
                self._buffers[key] = buf
            return buf

    def any_status_word(self, device_index: int) -> int | None:
        """Address of a status word of the device that no graph clears, for a call captured on a stream
        that has none (several streams' flags may share a word); None where nothing has run yet."""
        with self._lock:
            for key, buf in self._buffers.items():
                if key[0] == device_index and key not in self._captured:
                    return buf.data_ptr()
        return None

    def status_words(self, device_index: int, stream: int | None = None) -> list[torch.Tensor]:
        """The workspaces of one stream (None: of every stream) of a device, replaced ones included:
        a replayed graph flags what it finds in the one it was captured with."""
        with self._lock:
            return [buf for key, buf in self._buffers.items()
                    if key[0] == device_index and stream in (None, key[1])] + [
                buf for key, bufs in self._replaced.items()
                if key[0] == device_index and stream in (None, key[1]) for buf in bufs]


_workspaces = _Workspaces()


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream_handle(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _require_cuda(name: str, t: torch.Tensor, device: torch.device, dtype: torch.dtype) -> None:
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _decode_args(query, packed_k, packed_v, scales_k, scales_v, valid_tokens, bits, group_size,
                 block_table):
    """Validates decode tensors; returns (query, geometry tuple, n_sel)."""
    device = query.device
    if device.type != "cuda":
        raise RuntimeError(f"kvssd_b200 decode requires a CUDA device, got {device}")
    if query.ndim != 2:
        raise ValueError("query must be [query_heads, head_dim]")
    if query.dtype not in _QUERY_DTYPES:
        raise ValueError(f"unsupported query dtype {query.dtype}")
    if not query.is_contiguous():
        query = query.contiguous()
    if packed_k.ndim != 4 or packed_k.shape != packed_v.shape:
        raise ValueError("packed KV must match [blocks,tokens,kv_heads,packed_dim]")
    if scales_k.ndim != 4 or scales_k.shape != scales_v.shape:
        raise ValueError("KV scales must match [blocks,tokens,kv_heads,groups]")
    for name, t, dt in (("packed_k", packed_k, torch.uint8), ("packed_v", packed_v, torch.uint8),
                        ("scales_k", scales_k, torch.float16), ("scales_v", scales_v, torch.float16),
                        ("valid_tokens", valid_tokens, torch.int32)):
        _require_cuda(name, t, device, dt)
    n_pool, bt, kvh, pd = packed_k.shape
    qh, d = query.shape
    if tuple(scales_k.shape[:3]) != (n_pool, bt, kvh) or scales_k.shape[3] * group_size != d:
        raise ValueError("scale dimension mismatch")
    if valid_tokens.shape != (n_pool,):
        raise ValueError("valid_tokens must contain one count per block")
    if pd * 8 != d * bits:
        raise ValueError("packed dimension does not match query head dimension")
    if block_table is not None:
        _require_cuda("block_table", block_table, device, torch.int32)
        if block_table.ndim != 1:
            raise ValueError("block_table must be 1-D")
        n_sel = block_table.shape[0]
    else:
        n_sel = n_pool
    return query, (n_pool, n_sel, bt, qh, kvh, d, bits, group_size)


def _workspace_for(device, geometry) -> tuple[torch.Tensor, torch.cuda.Stream]:
    n_pool, n_sel, bt, qh, kvh, d, bits, group_size = geometry
    need = ctypes.c_size_t()
    _native.check(
        _native.library().kvssd_b200_decode_workspace_size(n_sel, bt, qh, kvh, d, bits,
                                                           group_size, ctypes.byref(need)),
        "kvssd_b200_decode_workspace_size",
    )
    stream = torch.cuda.current_stream(device)
    return _workspaces.get(device, stream, need.value), stream


def decode(
    query: torch.Tensor,
    packed_k: torch.Tensor,
    packed_v: torch.Tensor,
    scales_k: torch.Tensor,
    scales_v: torch.Tensor,
    valid_tokens: torch.Tensor,
    bits: int,
    group_size: int,
    sm_scale: float,
    block_table: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Fused dequantize + decode attention; returns (out fp32 [QH, D], lse fp32 [QH]).

    ``packed_*``/``scales_*``/``valid_tokens`` form a block pool; ``block_table`` (int32
    [n_sel]) selects and orders pool blocks (None = all pool blocks in order).
    """
    query, geom = _decode_args(query, packed_k, packed_v, scales_k, scales_v, valid_tokens, bits,
                               group_size, block_table)
    device = query.device
    n_pool, n_sel, bt, qh, kvh, d, _, _ = geom
    with torch.cuda.device(device):
        ws, stream = _workspace_for(device, geom)
        if out is None:
            out = torch.empty((qh, d), dtype=torch.float32, device=device)
        if lse is None:
            lse = torch.empty((qh,), dtype=torch.float32, device=device)
        _require_cuda("out", out, device, torch.float32)
        _require_cuda("lse", lse, device, torch.float32)
        status = _native.library().kvssd_b200_decode(
            _ptr(query), _QUERY_DTYPES[query.dtype],
            _ptr(packed_k), _ptr(packed_v), _ptr(scales_k), _ptr(scales_v),
            _ptr(valid_tokens), _ptr(block_table),
            n_pool, n_sel, bt, qh, kvh, d, bits, group_size,
            float(sm_scale), _ptr(out), _ptr(lse),
            _ptr(ws), ws.numel(), stream.cuda_stream,
        )
        _native.check(status, "kvssd_b200_decode")
    return out, lse


def decode_exchange(query, packed_k, packed_v, scales_k, scales_v, valid_tokens, bits: int,
                    group_size: int, sm_scale: float, rank: int, world: int,
                    buffers: list[int], block_table=None, out=None, lse=None,
                    workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """This rank's share of a multi-GPU decode (token-block-range shards) with the cross-rank
    merge fused into the kernel (kvssd_b200_decode_exchange); returns the whole context's
    (out, lse), identical on every rank. ``buffers`` are the ranks' exchange buffers as device
    addresses valid in this process (see sharding.PeerExchange)."""
    query, geom = _decode_args(query, packed_k, packed_v, scales_k, scales_v, valid_tokens, bits,
                               group_size, block_table)
    device = query.device
    n_pool, n_sel, bt, qh, kvh, d, _, _ = geom
    with torch.cuda.device(device):
        if workspace is None:
            workspace, stream = _workspace_for(device, geom)
        else:
            stream = torch.cuda.current_stream(device)
        if out is None:
            out = torch.empty((qh, d), dtype=torch.float32, device=device)
        if lse is None:
            lse = torch.empty((qh,), dtype=torch.float32, device=device)
        _require_cuda("out", out, device, torch.float32)
        _require_cuda("lse", lse, device, torch.float32)
        ptrs = (ctypes.c_void_p * len(buffers))(*buffers)
        status = _native.library().kvssd_b200_decode_exchange(
            _ptr(query), _QUERY_DTYPES[query.dtype],
            _ptr(packed_k), _ptr(packed_v), _ptr(scales_k), _ptr(scales_v),
            _ptr(valid_tokens), _ptr(block_table),
            n_pool, n_sel, bt, qh, kvh, d, bits, group_size, float(sm_scale),
            rank, world, ptrs, _ptr(out), _ptr(lse),
            _ptr(workspace), workspace.numel(), stream.cuda_stream,
        )
        _native.check(status, "kvssd_b200_decode_exchange")
    return out, lse


class BatchedDecode:
    """Several independent decodes in ONE launch (kvssd_b200_decode_batched).

    ``problems``: sequence of (query, packed_k, packed_v, scales_k, scales_v, valid_tokens,
    block_table or None) sharing the geometry (INT4, head_dim 128, group 32/64). The device
    descriptor table, the outputs and the workspace are built once, so ``run()`` is a single
    launch with no host-to-device copy: it can be captured in a CUDA graph and replayed (the
    tensors the descriptors point to may be refilled in place between replays).
    """

    def __init__(self, problems, bits: int, group_size: int, sm_scale: float,
                 out: torch.Tensor | None = None, lse: torch.Tensor | None = None):
        """``out`` fp32 [L, QH, D] / ``lse`` fp32 [L, QH] (optional): contiguous buffers the
        L problems write into (e.g. one buffer to all-gather across ranks); allocated per
        problem when absent."""
        problems = list(problems)
        if not problems:
            raise ValueError("at least one problem is required")
        self.bits, self.group_size, self.sm_scale = bits, group_size, float(sm_scale)
        checked = []
        geom0 = None
        for prob in problems:
            query, kp, vp, ks, vs, valid, table = prob
            query, geom = _decode_args(query, kp, vp, ks, vs, valid, bits, group_size, table)
            n_pool, n_sel, bt, qh, kvh, d, _, _ = geom
            if geom0 is None:
                geom0 = (bt, qh, kvh, d, query.dtype, query.device)
            elif (bt, qh, kvh, d, query.dtype, query.device) != geom0:
                raise ValueError("batched problems must share geometry, query dtype and device")
            checked.append((query, kp, vp, ks, vs, valid, table, n_pool, n_sel))
        self.geometry = geom0
        bt, qh, kvh, d, qdtype, device = geom0
        self.device = device
        self._keep = checked  # the tensors the descriptors point to
        n = len(checked)
        if (out is None) != (lse is None):
            raise ValueError("pass both out and lse, or neither")
        if out is None:
            self.outs = [(torch.empty((qh, d), dtype=torch.float32, device=device),
                          torch.empty((qh,), dtype=torch.float32, device=device))
                         for _ in checked]
        else:
            if tuple(out.shape) != (n, qh, d) or tuple(lse.shape) != (n, qh):
                raise ValueError(f"out/lse must be [{n}, {qh}, {d}] and [{n}, {qh}]")
            _require_cuda("out", out, device, torch.float32)
            _require_cuda("lse", lse, device, torch.float32)
            self.outs = [(out[i], lse[i]) for i in range(n)]
        desc = torch.empty((len(checked), 10), dtype=torch.int64, pin_memory=True)
        for i, ((query, kp, vp, ks, vs, valid, table, n_pool, n_sel), (out, lse)) in enumerate(
                zip(checked, self.outs)):
            desc[i] = torch.tensor([_ptr(query), _ptr(kp), _ptr(vp), _ptr(ks), _ptr(vs),
                                    _ptr(valid), _ptr(table) or 0, _ptr(out), _ptr(lse),
                                    (n_pool & 0xFFFFFFFF) | (n_sel << 32)], dtype=torch.int64)
        self.descriptors = desc.to(device)
        need = ctypes.c_size_t()
        with torch.cuda.device(device):
            _native.check(_native.library().kvssd_b200_decode_batched_workspace_size(
                len(checked), bt, qh, kvh, d, bits, group_size, ctypes.byref(need)),
                "kvssd_b200_decode_batched_workspace_size")
        self.workspace = torch.zeros(need.value, dtype=torch.uint8, device=device)
        torch.cuda.synchronize(device)

    def run(self) -> list[tuple[torch.Tensor, torch.Tensor]]:
        bt, qh, kvh, d, qdtype, device = self.geometry
        with torch.cuda.device(device):
            _native.check(_native.library().kvssd_b200_decode_batched(
                _ptr(self.descriptors), len(self.outs), _QUERY_DTYPES[qdtype], bt, qh, kvh, d,
                self.bits, self.group_size, self.sm_scale, _ptr(self.workspace),
                self.workspace.numel(), _stream_handle(device)),
                "kvssd_b200_decode_batched")
        return self.outs

    def read_status(self, clear: bool = True) -> int:
        """The sticky device status word of this batch's workspace (bit 16: a refused
        descriptor; see read_device_status for the others)."""
        value = ctypes.c_uint()
        with torch.cuda.device(self.device):
            status = _native.library().kvssd_b200_read_status(
                _ptr(self.workspace), 1 if clear else 0, ctypes.byref(value),
                _stream_handle(self.device))
        if status not in (_native.OK, _native.ERR_DEVICE_STATUS):
            _native.check(status, "kvssd_b200_read_status")
        return int(value.value)


def decode_batched(problems, bits: int, group_size: int, sm_scale: float):
    """One-shot BatchedDecode: builds the descriptors and launches; returns [(out, lse), ...]."""
    return BatchedDecode(problems, bits, group_size, sm_scale).run()


RECORD_BAD_HEADER, RECORD_BAD_GEOMETRY, RECORD_BAD_LENGTH, RECORD_BAD_CRC = 1, 2, 4, 8
RECORD_BAD_ID, RECORD_BAD_VALID = 16, 32


def decode_records(records: torch.Tensor, spec, layer: int | None = None,
                   block_ids: torch.Tensor | None = None):
    """Raw kvssd records on a CUDA device -> PackedBatch tensors, CRC-32 checked on the device.

    ``records`` is uint8 [n, record_bytes] (or flat, n * record_bytes), as read from the store.
    Returns (packed_k, packed_v, scales_k, scales_v, valid_tokens, status) where status is
    int32 [n] with the RECORD_BAD_* bits of each record (0 = good); see
    kvssd_b200_decode_records. Asynchronous on the current stream.
    """
    device = records.device
    if device.type != "cuda":
        raise RuntimeError(f"decode_records requires a CUDA tensor, got {device}")
    if records.dtype != torch.uint8 or not records.is_contiguous():
        raise ValueError("records must be a contiguous uint8 tensor")
    stride = spec.record_bytes
    if records.numel() % stride:
        raise ValueError(f"records must be whole records of {stride} bytes")
    n = records.numel() // stride
    bt, kvh = spec.block_tokens, spec.kv_heads
    packed_k = torch.empty((n, bt, kvh, spec.packed_dim), dtype=torch.uint8, device=device)
    packed_v = torch.empty_like(packed_k)
    scales_k = torch.empty((n, bt, kvh, spec.groups), dtype=torch.float16, device=device)
    scales_v = torch.empty_like(scales_k)
    valid = torch.empty((n,), dtype=torch.int32, device=device)
    status = torch.empty((n,), dtype=torch.int32, device=device)
    if block_ids is not None:
        block_ids = block_ids.to(device=device, dtype=torch.int32).contiguous()
        if block_ids.shape != (n,):
            raise ValueError("block_ids must name one block per record")
    with torch.cuda.device(device):
        _native.check(
            _native.library().kvssd_b200_decode_records(
                _ptr(records), stride, n, -1 if layer is None else int(layer), _ptr(block_ids),
                spec.bits, bt, kvh, spec.head_dim, spec.group_size, _ptr(packed_k),
                _ptr(packed_v), _ptr(scales_k), _ptr(scales_v), _ptr(valid), _ptr(status),
                _stream_handle(device)),
            "kvssd_b200_decode_records",
        )
    return packed_k, packed_v, scales_k, scales_v, valid, status


def decode_split(query, packed_k, packed_v, scales_k, scales_v, valid_tokens, bits: int,
                 group_size: int, sm_scale: float, block_table=None) -> tuple[int, torch.Tensor]:
    """Runs only the streaming split-KV kernel; returns (n_parts, workspace).

    The parts stay in the returned workspace until the next decode on this stream;
    decode_combine folds them into (out, lse).
    """
    query, geom = _decode_args(query, packed_k, packed_v, scales_k, scales_v, valid_tokens, bits,
                               group_size, block_table)
    device = query.device
    n_pool, n_sel, bt, qh, kvh, d, _, _ = geom
    n_parts = ctypes.c_int()
    with torch.cuda.device(device):
        ws, stream = _workspace_for(device, geom)
        status = _native.library().kvssd_b200_decode_split(
            _ptr(query), _QUERY_DTYPES[query.dtype],
            _ptr(packed_k), _ptr(packed_v), _ptr(scales_k), _ptr(scales_v),
            _ptr(valid_tokens), _ptr(block_table),
            n_pool, n_sel, bt, qh, kvh, d, bits, group_size, float(sm_scale),
            _ptr(ws), ws.numel(), ctypes.byref(n_parts), stream.cuda_stream,
        )
        _native.check(status, "kvssd_b200_decode_split")
    return n_parts.value, ws


def decode_combine(workspace: torch.Tensor, n_parts: int, query_heads: int, head_dim: int,
                   out: torch.Tensor | None = None, lse: torch.Tensor | None = None):
    device = workspace.device
    if out is None:
        out = torch.empty((query_heads, head_dim), dtype=torch.float32, device=device)
    if lse is None:
        lse = torch.empty((query_heads,), dtype=torch.float32, device=device)
    with torch.cuda.device(device):
        _native.check(
            _native.library().kvssd_b200_decode_combine(
                _ptr(workspace), n_parts, query_heads, head_dim, _ptr(out), _ptr(lse),
                _stream_handle(device)),
            "kvssd_b200_decode_combine",
        )
    return out, lse


def _indexed(device: torch.device | str | None) -> torch.device:
    """``device`` with its index: workspaces are kept by it. None, or no index: the current device."""
    device = torch.device("cuda") if device is None else torch.device(device)
    return torch.device("cuda", torch.cuda.current_device()) if device.index is None else device


def read_device_status(device: torch.device | str | None = None, clear: bool = True,
                       stream: torch.cuda.Stream | None = None) -> int:
    """Synchronously reads the sticky device status word of the current (or given) stream's
    workspace; ``clear`` zeroes the word (and the fused combine's test hook) when it is nonzero.

    Bit 1: a block-table entry was outside the pool; bit 2: a valid_tokens entry was outside
    [0, block_tokens] (such entries are skipped/clamped by the kernels, never dereferenced);
    bit 4: a fused combine, bit 8: a cross-GPU exchange, bit 32: a TMA-fed kernel's copy
    wait gave up (about a second) -- the out/lse of that call, and of later calls until the
    word is cleared, are NaN; bit 16: a batched problem descriptor was refused.
    """
    device = _indexed(device)
    stream = stream or torch.cuda.current_stream(device)
    _workspaces.get(device, stream, _WORKSPACE_HEADER)
    return _read_words(device, _workspaces.status_words(device.index, stream.cuda_stream), clear, stream)


def _read_words(device: torch.device, workspaces: list[torch.Tensor], clear: bool,
                stream: torch.cuda.Stream) -> int:
    total = 0
    with torch.cuda.device(device):
        for ws in workspaces:
            value = ctypes.c_uint()
            status = _native.library().kvssd_b200_read_status(
                _ptr(ws), 1 if clear else 0, ctypes.byref(value), stream.cuda_stream)
            if status not in (_native.OK, _native.ERR_DEVICE_STATUS):
                _native.check(status, "kvssd_b200_read_status")
            total |= int(value.value)
    return total


def read_device_status_all(device: torch.device | str | None = None, clear: bool = True) -> int:
    """OR of the status words of every decode workspace on ``device`` (one per stream that has
    decoded, graph-capture streams included), read after synchronising the device. What a replayed graph
    flags is found here: the cache-maintenance operators captured on a stream that has run nothing use
    another stream's word."""
    device = _indexed(device)
    torch.cuda.synchronize(device)
    return _read_words(device, _workspaces.status_words(device.index), clear,
                       torch.cuda.current_stream(device))


# Status bits that make a call's result invalid (the kernels then write NaN into out/lse) or
# that mean the caller passed entries the kernels had to refuse. Bit 2 (a valid_tokens entry
# outside [0, block_tokens], clamped like kvssd's CPU path clamps it by slicing) is not one.
FAILURE_BITS = (_native.DEV_BAD_BLOCK | _native.DEV_COMBINE_TIMEOUT |
                _native.DEV_EXCHANGE_TIMEOUT | _native.DEV_BAD_PROBLEM |
                _native.DEV_STREAM_TIMEOUT)

_STATUS_TEXT = {
    _native.DEV_BAD_BLOCK: "a block-table entry outside the pool",
    _native.DEV_BAD_VALID: "a valid_tokens entry outside [0, block_tokens]",
    _native.DEV_COMBINE_TIMEOUT: "the fused split-KV combine gave up waiting for parts",
    _native.DEV_EXCHANGE_TIMEOUT: "the cross-GPU exchange gave up waiting for another rank",
    _native.DEV_BAD_PROBLEM: "a batched problem descriptor was refused",
    _native.DEV_STREAM_TIMEOUT: "a TMA-fed kernel gave up waiting for its copies",
}


def describe_status(value: int) -> str:
    """Human-readable list of the conditions in a device status word."""
    parts = [text for bit, text in _STATUS_TEXT.items() if value & bit]
    return "; ".join(parts) or "none"


# Bits after which the kernels write NaN into out/lse (a wait gave up).
NAN_BITS = _native.DEV_COMBINE_TIMEOUT | _native.DEV_EXCHANGE_TIMEOUT | _native.DEV_STREAM_TIMEOUT


class DeviceFailure(RuntimeError):
    """A decode kernel flagged a failure in its workspace status word (see FAILURE_BITS)."""

    def __init__(self, status: int, where: str):
        self.status = status
        tail = ("; the out/lse of the failed call are NaN" if status & NAN_BITS else
                "; the offending entries were skipped, never dereferenced")
        super().__init__(f"{where}: device status {status:#x} ({describe_status(status)}){tail}")


class _StatusWatch:
    """Asynchronous reads of one (device, stream) workspace's status word.

    ``arm()`` enqueues, after a call's kernels, a 4-byte copy of the status word into a slot of
    pinned host memory and records an event; ``poll()`` looks at the slots whose event has
    completed (no synchronisation) and ``check()`` waits for all of them. A failure is raised
    once, as DeviceFailure, after the word has been read and cleared on the device (which
    makes the workspace usable again).
    """

    SLOTS = 4

    def __init__(self, device: torch.device, stream: torch.cuda.Stream):
        self.device, self.stream = device, stream
        self._host = list(torch.zeros(self.SLOTS, dtype=torch.int32, pin_memory=True).split(1))
        self._own_events = [torch.cuda.Event() for _ in range(self.SLOTS)]
        self._events: list[torch.cuda.Event | None] = [None] * self.SLOTS  # those of outstanding reads
        self._word: tuple[torch.Tensor, torch.Tensor] | None = None  # the workspace and its status word
        self._next = 0

    def _take(self, i: int, block: bool) -> int:
        ev = self._events[i]
        if ev is None:
            return 0
        if not ev.query():
            if not block:
                return 0
            ev.synchronize()
        self._events[i] = None
        return self._host[i].item()

    def _raise(self, value: int, where: str) -> None:
        if value & FAILURE_BITS:
            read_device_status(self.device, clear=True, stream=self.stream)
            for i in range(self.SLOTS):  # older slots hold the same sticky bits
                self._events[i] = None
            raise DeviceFailure(value, where)

    def arm(self, where: str) -> None:
        if torch.cuda.is_current_stream_capturing():
            return  # inside a graph capture the caller checks after replay (check())
        i = self._next % self.SLOTS
        self._raise(self._take(i, block=True), where)  # the slot's earlier read, long done
        ws = _workspaces.get(self.device, self.stream, _WORKSPACE_HEADER)
        if self._word is None or self._word[0] is not ws:
            self._word = ws, ws[:4].view(torch.int32)
        if _raw_stream(self.device.index) == self.stream.cuda_stream:
            self._host[i].copy_(self._word[1], non_blocking=True)
        else:
            with torch.cuda.stream(self.stream):
                self._host[i].copy_(self._word[1], non_blocking=True)
        self._own_events[i].record(self.stream)
        self._events[i] = self._own_events[i]
        self._next += 1

    def poll(self, where: str) -> None:
        if torch.cuda.is_current_stream_capturing():
            return  # an event must not be queried then; a later call outside looks
        value = 0
        for i in range(self.SLOTS):
            value |= self._take(i, block=False)
        self._raise(value, where)

    def check(self, where: str) -> None:
        value = 0
        for i in range(self.SLOTS):
            value |= self._take(i, block=True)
        self._raise(value, where)

    def discard(self) -> None:
        """Waits for the outstanding reads and drops them (the caller reads the word itself)."""
        for i in range(self.SLOTS):
            self._take(i, block=True)


_watch_lock = threading.Lock()
_watches: dict[tuple[int, int], _StatusWatch] = {}


def status_watch(device: torch.device, stream: torch.cuda.Stream | None = None) -> _StatusWatch:
    """The status watch of ``device``'s current (or given) stream workspace."""
    if device.index is None:
        device = _indexed(device)
    stream = stream or torch.cuda.current_stream(device)
    key = (device.index, stream.cuda_stream)
    with _watch_lock:
        w = _watches.get(key)
        if w is None:
            w = _watches[key] = _StatusWatch(device, stream)
        return w


def decode_path(head_dim: int, bits: int, group_size: int) -> int:
    path = ctypes.c_int()
    _native.check(
        _native.library().kvssd_b200_decode_path(head_dim, bits, group_size, ctypes.byref(path)),
        "kvssd_b200_decode_path",
    )
    return path.value


# decode_plan kernel names of the two streaming kernels (split-KV with the fused combine)
STREAMING_KERNELS = ("tensor_core_tma", "tensor_core_stream")


def decode_plan(n_sel: int, block_tokens: int, query_heads: int, kv_heads: int, head_dim: int,
                bits: int, group_size: int) -> dict:
    """Kernel choice and split count for a geometry on the current CUDA device."""
    kernel, splits, parts = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    _native.check(
        _native.library().kvssd_b200_decode_plan(
            n_sel, block_tokens, query_heads, kv_heads, head_dim, bits, group_size,
            ctypes.byref(kernel), ctypes.byref(splits), ctypes.byref(parts)),
        "kvssd_b200_decode_plan",
    )
    names = {_native.PATH_TENSOR_CORE: "tensor_core_tma",
             _native.PATH_TENSOR_CORE_CPASYNC: "tensor_core_stream",
             _native.PATH_TENSOR_CORE_REGS: "tensor_core_regs", _native.PATH_GENERIC: "generic"}
    return {"kernel": names[kernel.value], "path": kernel.value, "n_splits": splits.value,
            "n_parts": parts.value}


def set_path_override(path: int) -> None:
    _native.check(_native.library().kvssd_b200_set_path_override(path), "set_path_override")


def merge_chunks(outs: torch.Tensor, lses: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Exact N-way merge of normalised chunks: outs [N, QH, D] fp32, lses [N, QH] fp32."""
    device = outs.device
    if device.type != "cuda":
        raise RuntimeError(f"merge_chunks requires CUDA tensors, got {device}")
    if outs.ndim != 3 or lses.shape != outs.shape[:2]:
        raise ValueError("expected outs [N, QH, D] and lses [N, QH]")
    _require_cuda("outs", outs, device, torch.float32)
    _require_cuda("lses", lses, device, torch.float32)
    n, qh, d = outs.shape
    out = torch.empty((qh, d), dtype=torch.float32, device=device)
    lse = torch.empty((qh,), dtype=torch.float32, device=device)
    with torch.cuda.device(device):
        _native.check(
            _native.library().kvssd_b200_merge_chunks(
                _ptr(outs), _ptr(lses), n, qh, d, _ptr(out), _ptr(lse), _stream_handle(device)
            ),
            "kvssd_b200_merge_chunks",
        )
    return out, lse


def merge_pair(
    left_output: torch.Tensor, left_lse: torch.Tensor, right_output: torch.Tensor,
    right_lse: torch.Tensor,
) -> tuple[torch.Tensor, torch.Tensor]:
    device = left_output.device
    if device.type != "cuda":
        raise RuntimeError(f"merge_attention_chunks requires CUDA tensors, got {device}")
    if left_output.ndim != 2 or right_output.shape != left_output.shape:
        raise ValueError("chunk outputs must both be [QH, D]")
    qh, d = left_output.shape
    if left_lse.shape != (qh,) or right_lse.shape != (qh,):
        raise ValueError("chunk LSEs must be [QH]")
    tensors = [t.contiguous().float() for t in (left_output, left_lse, right_output, right_lse)]
    for name, t in zip(("left_output", "left_lse", "right_output", "right_lse"), tensors):
        _require_cuda(name, t, device, torch.float32)
    out = torch.empty((qh, d), dtype=torch.float32, device=device)
    lse = torch.empty((qh,), dtype=torch.float32, device=device)
    with torch.cuda.device(device):
        _native.check(
            _native.library().kvssd_b200_merge_pair(
                *map(_ptr, tensors), qh, d, _ptr(out), _ptr(lse), _stream_handle(device)
            ),
            "kvssd_b200_merge_pair",
        )
    return out, lse


def dequantize_packed(
    packed: torch.Tensor, scales: torch.Tensor, bits: int, group_size: int, mode: int = 0
) -> tuple[torch.Tensor, torch.Tensor]:
    """Runs the decode kernels' register unpacker over [rows, packed_dim] codes.

    Returns (codes uint8 [rows, D], values fp16 [rows, D]); used to prove bit-exactness
    against kvssd's unpack_codes / dequantize_tensor(q, torch.float16).
    """
    device = packed.device
    if device.type != "cuda":
        raise RuntimeError(f"dequantize_packed requires CUDA tensors, got {device}")
    pd = packed.shape[-1]
    d = pd * 8 // bits
    rows = packed.numel() // pd
    p2 = packed.reshape(rows, pd).contiguous()
    s2 = scales.reshape(rows, -1).contiguous()
    _require_cuda("packed", p2, device, torch.uint8)
    _require_cuda("scales", s2, device, torch.float16)
    values = torch.empty((rows, d), dtype=torch.float16, device=device)
    codes = torch.empty((rows, d), dtype=torch.uint8, device=device)
    with torch.cuda.device(device):
        _native.check(
            _native.library().kvssd_b200_dequantize(
                _ptr(p2), _ptr(s2), rows, d, bits, group_size, mode, _ptr(values), _ptr(codes),
                _stream_handle(device),
            ),
            "kvssd_b200_dequantize",
        )
    shape = (*packed.shape[:-1], d)
    return codes.reshape(shape), values.reshape(shape)


# --- cache maintenance: rotary positions, the quantizing cache write, attention weights, eviction ---

_ELEMENT_DTYPES = {torch.float32: _native.Q_F32, torch.float16: _native.Q_F16,
                   torch.bfloat16: _native.Q_BF16}
_INDEX_DTYPES = {torch.int32: 0, torch.int64: 1}


# The operators below are called once per layer and step, on tensors that differ in nothing but their
# contents, and their kernels take a few microseconds: what a call costs on the host is part of what it
# costs. Each checks its tensors in one expression and looks for the reason only when that fails.

_entry_points: dict[str, object] = {}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(index: int, name: str, *args) -> None:
    """Calls an entry point with device ``index`` current."""
    fn = _entry_points.get(name)
    if fn is None:
        fn = _entry_points[name] = getattr(_native.library(), name)
    if torch.cuda.current_device() == index:
        status = fn(*args)
    else:
        with torch.cuda.device(index):
            status = fn(*args)
    if status:
        _native.check(status, name)


def _device_index(name: str, t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise RuntimeError(f"{name} requires a CUDA device, got {t.device}")
    return t.get_device()


def _status_word(index: int, stream: int) -> int | None:
    """Address of the stream's sticky status word (read_device_status, status_watch). Creating one during a
    graph capture would be captured: another stream's serves then."""
    ws = _workspaces._buffers.get((index, stream))
    if ws is None:
        if torch.cuda.is_current_stream_capturing():
            return _workspaces.any_status_word(index)
        ws = _workspaces.get(torch.device("cuda", index), torch.cuda.current_stream(index),
                             _WORKSPACE_HEADER)
    return ws.data_ptr()


def _require_rows(name: str, t: torch.Tensor, shape, dtype, device) -> None:
    """A [tokens, heads, head_dim] tensor whose last dimension is contiguous."""
    if t.device != device or t.dtype != dtype or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)} {dtype} on {device}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    if t.stride(2) != 1 and t.shape[2] > 1:
        raise ValueError(f"{name} must be contiguous along its last dimension")


def _index_kind(name: str, t: torch.Tensor, n: int, device) -> int:
    kind = _INDEX_DTYPES.get(t.dtype)
    if kind is None or t.shape != (n,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 or int64 [{n}] on {device}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    return kind


def _check_frequencies(frequencies: torch.Tensor, head_dim: int, device) -> int:
    if (frequencies.dtype != torch.float64 or frequencies.ndim != 1
            or frequencies.device != device or not frequencies.is_contiguous()):
        raise ValueError(f"frequencies must be contiguous float64 [pairs] on {device}")
    pairs = frequencies.shape[0]
    if pairs < 1 or 2 * pairs > head_dim:
        raise ValueError("frequencies must hold 1 to head_dim / 2 pairs")
    return pairs


def rotary(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, *,
           interleaved: bool = False, magnitude: float = 1.0,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions of ``x`` [tokens, heads, head_dim] (FP32, FP16 or BF16; any token and head
    strides), in a new tensor or in ``out``, which may be ``x`` itself and else must not overlap it.

    ``positions`` int32 or int64 [tokens]; ``frequencies`` float64 [pairs], radians a position (see
    rotary.RotaryEmbedding for the usual scalings). The first 2 * pairs dims of a head are rotated
    -- pair i is dims (i, i + pairs), or (2i, 2i + 1) when ``interleaved`` --, the dims behind are
    copied. Angles are FP64; cos and sin, the ``magnitude`` that multiplies them and the products FP32,
    rounded once."""
    index = _device_index("rotary", x)
    dtype = _ELEMENT_DTYPES.get(x.dtype)
    if dtype is None:
        raise ValueError(f"unsupported element type {x.dtype}")
    if x.ndim != 3:
        raise ValueError("x must be [tokens, heads, head_dim]")
    if out is None:
        if x.stride(2) != 1:
            x = x.contiguous()
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    else:
        _require_rows("x", x, x.shape, x.dtype, x.device)
        _require_rows("out", out, x.shape, x.dtype, x.device)
        near, far = sorted(((out.stride(0), x.shape[0]), (out.stride(1), x.shape[1])))
        d = x.shape[2]
        if (near[1] > 1 and near[0] < d) or (far[1] > 1 and far[0] < near[0] * (near[1] - 1) + d):
            raise ValueError("out must not overlap itself")
    tokens, heads, d = x.shape
    kind = _INDEX_DTYPES.get(positions.dtype)
    if (kind is None or positions.shape != (tokens,) or positions.get_device() != index
            or not positions.is_contiguous()):
        _index_kind("positions", positions, tokens, x.device)
    if (frequencies.dtype is not torch.float64 or frequencies.ndim != 1
            or not 2 <= 2 * frequencies.shape[0] <= d or frequencies.get_device() != index
            or not frequencies.is_contiguous()):
        _check_frequencies(frequencies, d, x.device)
    token, head, _ = x.stride()
    out_token, out_head, _ = out.stride()
    _call(index, "kvssd_b200_rotary", x.data_ptr(), dtype, token, head, tokens, heads, d,
          positions.data_ptr(), kind, frequencies.data_ptr(), frequencies.shape[0], interleaved,
          magnitude, out.data_ptr(), out_token, out_head, _raw_stream(index))
    return out


def _check_pool(packed_k, packed_v, scales_k, scales_v, valid_tokens, bits, group_size, device):
    """Finds what is wrong with the tensors of a block pool, if anything is."""
    for name, t, dt in (("packed_k", packed_k, torch.uint8), ("packed_v", packed_v, torch.uint8),
                        ("scales_k", scales_k, torch.float16),
                        ("scales_v", scales_v, torch.float16),
                        ("valid_tokens", valid_tokens, torch.int32)):
        if t is not None:
            _require_cuda(name, t, device, dt)
    if bits not in (2, 4):
        raise ValueError("bits must be 2 or 4")
    if packed_k.ndim != 4 or (packed_v is not None and packed_v.shape != packed_k.shape):
        raise ValueError("packed KV must match [blocks,tokens,kv_heads,packed_dim]")
    n_pool, bt, kvh, pd = packed_k.shape
    d = pd * 8 // bits
    if group_size < 1 or d % group_size:
        raise ValueError("group_size must divide head_dim")
    shape = (n_pool, bt, kvh, d // group_size)
    if scales_k.shape != shape or (scales_v is not None and scales_v.shape != shape):
        raise ValueError("KV scales must match [blocks,tokens,kv_heads,groups]")
    if valid_tokens is not None and valid_tokens.shape != (n_pool,):
        raise ValueError("valid_tokens must contain one count per block")


def append(key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor, packed_k: torch.Tensor,
           packed_v: torch.Tensor, scales_k: torch.Tensor, scales_v: torch.Tensor, bits: int,
           group_size: int, *, positions: torch.Tensor | None = None,
           frequencies: torch.Tensor | None = None, interleaved: bool = False,
           magnitude: float = 1.0, valid_tokens: torch.Tensor | None = None,
           values: bool = False) -> tuple[torch.Tensor, torch.Tensor] | None:
    """Quantizes the keys and values [tokens, kv_heads, head_dim] (FP32, FP16 or BF16; any token and
    head strides) of ``tokens`` tokens into their slots of a block pool, in place.

    ``slots`` int32 or int64 [tokens]: block * block_tokens + row; a negative slot is skipped
    (padding), one behind the pool is skipped and flagged (read_device_status bit 1). The slots of
    one call must differ from each other. With ``frequencies`` and ``positions`` the keys are rotated
    first (as ``rotary``, but rounded to FP32 once instead of to their type). Codes and scales equal
    quant.quantize_tensor's bit for bit, except the codes of groups that hold a NaN or an infinity. ``valid_tokens`` (optional): the counts of the written
    blocks are raised to cover the written rows. ``values=True`` returns the FP16 keys and values that
    the cache now holds for the tokens ([tokens, kv_heads, head_dim], skipped tokens included), for a
    prompt's own attention to see what later decodes will see."""
    index = _device_index("append", key)
    dtype = _ELEMENT_DTYPES.get(key.dtype)
    if dtype is None:
        raise ValueError(f"unsupported element type {key.dtype}")
    if key.ndim != 3:
        raise ValueError("key must be [tokens, kv_heads, head_dim]")
    pool = packed_k.shape
    scales = scales_k.shape
    if (len(pool) != 4 or packed_v.shape != pool or len(scales) != 4 or scales[:3] != pool[:3]
            or scales_v.shape != scales or bits not in (2, 4) or pool[3] * 8 != scales[3] * group_size * bits
            or packed_k.dtype is not torch.uint8 or packed_v.dtype is not torch.uint8
            or scales_k.dtype is not torch.float16 or scales_v.dtype is not torch.float16
            or packed_k.get_device() != index or packed_v.get_device() != index
            or scales_k.get_device() != index or scales_v.get_device() != index
            or not packed_k.is_contiguous() or not packed_v.is_contiguous()
            or not scales_k.is_contiguous() or not scales_v.is_contiguous()
            or valid_tokens is not None and (
                valid_tokens.dtype is not torch.int32 or valid_tokens.shape != pool[:1]
                or valid_tokens.get_device() != index or not valid_tokens.is_contiguous())):
        _check_pool(packed_k, packed_v, scales_k, scales_v, valid_tokens, bits, group_size, key.device)
        raise ValueError("packed dimension does not match the scales")
    n_pool, bt, kvh, pd = pool
    tokens, d = key.shape[0], pd * 8 // bits
    shape = (tokens, kvh, d)
    if (key.shape != shape or value.shape != shape or value.dtype is not key.dtype
            or value.get_device() != index or key.stride(2) != 1 or value.stride(2) != 1):
        _require_rows("key", key, shape, key.dtype, key.device)
        _require_rows("value", value, shape, key.dtype, key.device)
    slot_kind = _INDEX_DTYPES.get(slots.dtype)
    if (slot_kind is None or slots.shape != (tokens,) or slots.get_device() != index
            or not slots.is_contiguous()):
        _index_kind("slots", slots, tokens, key.device)
    pos_ptr = freq_ptr = None
    pos_kind = pairs = 0
    if frequencies is not None:
        if positions is None:
            raise ValueError("rotated keys need positions")
        pos_kind = _INDEX_DTYPES.get(positions.dtype)
        if (pos_kind is None or positions.shape != (tokens,) or positions.get_device() != index
                or not positions.is_contiguous()):
            _index_kind("positions", positions, tokens, key.device)
        pairs = frequencies.shape[0] if frequencies.ndim == 1 else 0
        if (frequencies.dtype is not torch.float64 or not 2 <= 2 * pairs <= d
                or frequencies.get_device() != index or not frequencies.is_contiguous()):
            _check_frequencies(frequencies, d, key.device)
        pos_ptr, freq_ptr = positions.data_ptr(), frequencies.data_ptr()
    held, key_ptr, value_ptr = None, None, None
    if values:
        held = tuple(torch.empty_like(key, dtype=torch.float16, memory_format=torch.contiguous_format)
                     for _ in "kv")
        key_ptr, value_ptr = held[0].data_ptr(), held[1].data_ptr()
    stream = _raw_stream(index)
    k_token, k_head, _ = key.stride()
    v_token, v_head, _ = value.stride()
    _call(index, "kvssd_b200_append", key.data_ptr(), value.data_ptr(), dtype, k_token, k_head,
          v_token, v_head, tokens, slots.data_ptr(), slot_kind, pos_ptr, pos_kind, freq_ptr, pairs,
          interleaved, magnitude, packed_k.data_ptr(), packed_v.data_ptr(), scales_k.data_ptr(),
          scales_v.data_ptr(), None if valid_tokens is None else valid_tokens.data_ptr(), n_pool, bt,
          kvh, d, bits, group_size, key_ptr, value_ptr, _status_word(index, stream), stream)
    return held


def _check_table(block_table, n_pool: int, device) -> int:
    if block_table is None:
        return n_pool
    _require_cuda("block_table", block_table, device, torch.int32)
    if block_table.ndim != 1:
        raise ValueError("block_table must be 1-D")
    return block_table.shape[0]


def _require_stats(name: str, t: torch.Tensor, kvh: int, columns: int | None, dtype, device) -> None:
    """A [kv_heads, columns] tensor with contiguous rows."""
    if t.dtype is not dtype or t.ndim != 2 or t.shape[0] != kvh or t.device != device or (
            columns is not None and t.shape[1] != columns):
        raise ValueError(f"{name} must be [{kvh}, {columns or 'places'}] {dtype} on {device}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    if t.shape[1] > 1 and t.stride(1) != 1 or (kvh > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{name} must have contiguous rows that do not overlap")


def attention_weights(query: torch.Tensor, packed_k: torch.Tensor, scales_k: torch.Tensor,
                      valid_tokens: torch.Tensor, bits: int, group_size: int, sm_scale: float, *,
                      lse: torch.Tensor | None = None, block_table: torch.Tensor | None = None,
                      visible: torch.Tensor | None = None, previous: torch.Tensor | None = None,
                      out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The attention weight every selected place gets: returns (weights fp32
    [kv_heads, n_sel * block_tokens], lse).

    weights[h, i] = previous[h, i] + the sum over the queries t and the query heads g of KV head h of
    exp(sm_scale * q[t, g] . k[i, h] - lse[t, g]), place i being row i % block_tokens of the i //
    block_tokens-th selected block. ``query`` [query_heads, head_dim] (a decode step) or
    [queries, query_heads, head_dim] (a prompt's last queries), FP32, FP16, BF16 or FP64; a place
    counts for query t when its row lies before the block's valid count and i < ``visible``[t] (int32
    [queries]; None: all). ``lse`` fp32 [query_heads] or [queries, query_heads]: as ``decode``
    returned it for these queries, or None to compute it (a first pass over the keys). ``out`` may be
    ``previous`` and else must not overlap it. The returned lse is -inf for a query that sees nothing; it adds nothing."""
    index = _device_index("attention_weights", query)
    dtype = _QUERY_DTYPES.get(query.dtype)
    if dtype is None:
        raise ValueError(f"unsupported query dtype {query.dtype}")
    if query.ndim not in (2, 3):
        raise ValueError("query must be [query_heads, head_dim] or [queries, query_heads, head_dim]")
    if not query.is_contiguous():
        query = query.contiguous()
    pool = packed_k.shape
    scales = scales_k.shape
    if (len(pool) != 4 or len(scales) != 4 or scales[:3] != pool[:3] or bits not in (2, 4)
            or pool[3] * 8 != scales[3] * group_size * bits or packed_k.dtype is not torch.uint8
            or scales_k.dtype is not torch.float16 or valid_tokens.dtype is not torch.int32
            or valid_tokens.shape != pool[:1] or packed_k.get_device() != index
            or scales_k.get_device() != index or valid_tokens.get_device() != index
            or not packed_k.is_contiguous() or not scales_k.is_contiguous()
            or not valid_tokens.is_contiguous()):
        _check_pool(packed_k, None, scales_k, None, valid_tokens, bits, group_size, query.device)
        raise ValueError("packed dimension does not match the scales")
    n_pool, bt, kvh, pd = pool
    d = pd * 8 // bits
    rows = query.shape[:-1]
    queries = rows[0] if query.ndim == 3 else 1
    qh = rows[-1]
    if query.shape[-1] != d:
        raise ValueError("packed dimension does not match query head dimension")
    if queries < 1 or qh < 1 or qh % kvh:
        raise ValueError("query heads must be divisible by KV heads")
    table = None
    n_sel = n_pool
    if block_table is not None:
        n_sel = _check_table(block_table, n_pool, query.device)
        table = block_table.data_ptr()
    places = n_sel * bt
    seen = None
    if visible is not None:
        _require_cuda("visible", visible, query.device, torch.int32)
        if visible.shape != (queries,):
            raise ValueError("visible must hold one count per query")
        seen = visible.data_ptr()
    before, before_stride = None, 0
    if previous is not None:
        _require_stats("previous", previous, kvh, places, torch.float32, query.device)
        before, before_stride = previous.data_ptr(), previous.stride(0)
    if out is None:
        out = torch.empty((kvh, places), dtype=torch.float32, device=query.device)
    else:
        _require_stats("out", out, kvh, places, torch.float32, query.device)
    scratch, scratch_ptr, scratch_bytes, given = None, None, 0, lse is not None
    if given:
        if (lse.dtype is not torch.float32 or lse.shape != rows or lse.get_device() != index
                or not lse.is_contiguous()):
            _require_cuda("lse", lse, query.device, torch.float32)
            raise ValueError(f"lse must be {tuple(rows)}, got {tuple(lse.shape)}")
    else:
        need = ctypes.c_size_t()
        _call(index, "kvssd_b200_attention_weights_scratch_size", queries, n_sel, bt, qh, kvh, d,
              bits, group_size, ctypes.byref(need))
        scratch_bytes = need.value
        scratch = torch.empty(scratch_bytes, dtype=torch.uint8, device=query.device)
        scratch_ptr = scratch.data_ptr()
        lse = torch.empty(rows, dtype=torch.float32, device=query.device)
    stream = _raw_stream(index)
    _call(index, "kvssd_b200_attention_weights", query.data_ptr(), dtype, queries,
          packed_k.data_ptr(), scales_k.data_ptr(), valid_tokens.data_ptr(), table, seen, n_pool,
          n_sel, bt, qh, kvh, d, bits, group_size, sm_scale, given, lse.data_ptr(), before,
          before_stride, out.data_ptr(), out.stride(0), scratch_ptr, scratch_bytes,
          _status_word(index, stream), stream)
    return out, lse


def evict(weights: torch.Tensor, positions: torch.Tensor, n_tokens: int, keep: int,
          packed_k: torch.Tensor, packed_v: torch.Tensor, scales_k: torch.Tensor,
          scales_v: torch.Tensor, valid_tokens: torch.Tensor, *,
          block_table: torch.Tensor | None = None, sink: int = 0, recent: int = 0,
          next_position: int | None = None, shared: bool = False,
          out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Compacts a cache of ``n_tokens`` tokens in place to the ``keep`` tokens of the largest
    accumulated weight; returns (weights, positions) of the compacted cache, shaped as given, 0 and -1
    from ``keep`` on: in new tensors or in those of ``out`` (contiguous; they must not overlap the inputs).

    Place i of the cache is row i % block_tokens of the i // block_tokens-th selected block
    (``block_table`` entries must differ; None: the pool in order); its blocks before the last hold
    block_tokens tokens each. ``weights`` fp32 and ``positions`` int32 [kv_heads, places] say what
    each place has gathered (``attention_weights``) and which token it holds. Each KV head chooses for
    itself, or all heads together by the sum of their weights when ``shared`` (positions of head 0).
    Tokens at positions below ``sink`` or among the ``recent`` ones before ``next_position`` (None:
    n_tokens) are kept in any case; equal weights go by the lower place, a NaN ranks last. The j-th
    place below ``keep`` that is given up receives the j-th kept token from behind ``keep`` (packed
    rows, scales, weight, position); the rows from ``keep`` on stay as they were, and
    ``valid_tokens`` of the selected blocks becomes the rows they still hold."""
    index = _device_index("evict", weights)
    pool = packed_k.shape
    scales = scales_k.shape
    if (len(pool) != 4 or packed_v.shape != pool or len(scales) != 4 or scales[:3] != pool[:3]
            or scales_v.shape != scales or valid_tokens.shape != pool[:1]
            or packed_k.dtype is not torch.uint8 or packed_v.dtype is not torch.uint8
            or scales_k.dtype is not torch.float16 or scales_v.dtype is not torch.float16
            or valid_tokens.dtype is not torch.int32 or valid_tokens.get_device() != index
            or packed_k.get_device() != index or packed_v.get_device() != index
            or scales_k.get_device() != index or scales_v.get_device() != index
            or not packed_k.is_contiguous() or not packed_v.is_contiguous()
            or not scales_k.is_contiguous() or not scales_v.is_contiguous()
            or not valid_tokens.is_contiguous()):
        for name, t, dt in (("packed_k", packed_k, torch.uint8), ("packed_v", packed_v, torch.uint8),
                            ("scales_k", scales_k, torch.float16),
                            ("scales_v", scales_v, torch.float16),
                            ("valid_tokens", valid_tokens, torch.int32)):
            _require_cuda(name, t, weights.device, dt)
        raise ValueError("the pool must be [blocks,tokens,kv_heads,packed_dim] codes, "
                         "[blocks,tokens,kv_heads,groups] scales and one valid count per block")
    n_pool, bt, kvh, pd = pool
    _require_stats("weights", weights, kvh, None, torch.float32, weights.device)
    columns = weights.shape[1]
    _require_stats("positions", positions, kvh, columns, torch.int32, weights.device)
    n_sel = _check_table(block_table, n_pool, weights.device)
    if not 1 <= n_tokens <= min(columns, n_sel * bt):
        raise ValueError("n_tokens must be positive and lie in the selected blocks and in weights")
    if not 1 <= keep <= n_tokens:
        raise ValueError("keep must be 1 to n_tokens")
    if sink < 0 or recent < 0:
        raise ValueError("sink and recent counts must be non-negative")
    if sink + recent > keep:
        raise ValueError("keep must hold the sink and recent tokens")
    end = n_tokens if next_position is None else next_position
    recent_from = end - recent if recent else 1 << 40  # behind every position
    lists = 1 if shared else kvh
    if out is None:
        new_weights = torch.empty((kvh, columns), dtype=torch.float32, device=weights.device)
        new_positions = torch.empty((kvh, columns), dtype=torch.int32, device=weights.device)
    else:
        new_weights, new_positions = out
        for name, t, dtype in (("out[0]", new_weights, torch.float32), ("out[1]", new_positions, torch.int32)):
            _require_cuda(name, t, weights.device, dtype)
            if t.shape != (kvh, columns):
                raise ValueError(f"{name} must be [{kvh}, {columns}], got {tuple(t.shape)}")
            if t.data_ptr() in (weights.data_ptr(), positions.data_ptr()):
                raise ValueError("out must not overlap weights or positions")
    ints = lists * (n_tokens + 1)
    if n_tokens > 1 << 17:  # the longest caches need more
        need = ctypes.c_size_t()
        _call(index, "kvssd_b200_evict_scratch_size", n_tokens, keep, kvh, shared, ctypes.byref(need))
        ints = need.value // 4
    scratch = torch.empty(ints, dtype=torch.int32, device=weights.device)
    stream = _raw_stream(index)
    _call(index, "kvssd_b200_evict", weights.data_ptr(), weights.stride(0), positions.data_ptr(),
          positions.stride(0), n_tokens, keep, sink, recent_from, shared, new_weights.data_ptr(),
          new_positions.data_ptr(), columns, packed_k.data_ptr(), packed_v.data_ptr(),
          scales_k.data_ptr(), scales_v.data_ptr(), valid_tokens.data_ptr(), _ptr(block_table),
          n_pool, n_sel, bt, kvh, pd, scales[3], scratch.data_ptr(), 4 * ints,
          _status_word(index, stream), stream)
    return new_weights, new_positions


def default_sm_scale(head_dim: int) -> float:
    return 1.0 / math.sqrt(head_dim)
