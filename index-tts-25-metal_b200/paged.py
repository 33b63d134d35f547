"""Paged K/V cache operators (ctypes over include/itts_paged.h) on CUDA tensors.

``tables`` does a step's bookkeeping on the GPU (block tables, lengths, row
positions and slots from the requests' lengths), ``append`` writes the step's
key and value rows into the cache, ``attention`` runs the step's query rows over
it.  Every call enqueues on the current torch stream of its tensors' device and
returns at once; it can be captured into a CUDA graph.  Failures raise as in
``gpt.py`` (ValueError for arguments that the library refuses).
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import gpt

BAD_LENGTH, NO_ROWS, NO_BLOCKS, BAD_FREE, BAD_BLOCK = 1, 2, 4, 8, 16
MAX_REQUESTS = 8192

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


class Tables(C.Structure):
    """itts_paged_tables_args."""
    _fields_ = [("requests", C.c_int32), ("block_size", C.c_int32), ("blocks", C.c_int32), ("max_blocks", C.c_int32),
                ("table_stride", C.c_int64), ("rows", C.c_int32), ("cached", C.c_void_p), ("fresh", C.c_void_p),
                ("table", C.c_void_p), ("free_list", C.c_void_p), ("free_in", C.c_void_p), ("free_out", C.c_void_p),
                ("lens", C.c_void_p), ("q_start", C.c_void_p), ("positions", C.c_void_p), ("slots", C.c_void_p),
                ("status", C.c_void_p)]


class Cache(C.Structure):
    """itts_paged_cache."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("type", C.c_int32), ("blocks", C.c_int32),
                ("block_size", C.c_int32), ("heads", C.c_int32), ("head_dim", C.c_int32), ("reserved", C.c_int32),
                ("k_block_stride", C.c_int64), ("k_token_stride", C.c_int64), ("k_head_stride", C.c_int64),
                ("v_block_stride", C.c_int64), ("v_token_stride", C.c_int64), ("v_head_stride", C.c_int64)]


class Append(C.Structure):
    """itts_paged_append_args."""
    _fields_ = [("cache", Cache), ("k", C.c_void_p), ("v", C.c_void_p), ("source_type", C.c_int32),
                ("rows", C.c_int32), ("k_row_stride", C.c_int64), ("k_head_stride", C.c_int64),
                ("v_row_stride", C.c_int64), ("v_head_stride", C.c_int64), ("slots", C.c_void_p)]


class Attention(C.Structure):
    """itts_paged_attention_args."""
    _fields_ = [("cache", Cache), ("q", C.c_void_p), ("out", C.c_void_p), ("q_heads", C.c_int32), ("rows", C.c_int32),
                ("q_row_stride", C.c_int64), ("q_head_stride", C.c_int64), ("out_row_stride", C.c_int64),
                ("out_head_stride", C.c_int64), ("q_start", C.c_void_p), ("lens", C.c_void_p), ("table", C.c_void_p),
                ("table_stride", C.c_int64), ("requests", C.c_int32), ("max_blocks", C.c_int32),
                ("max_fresh", C.c_int32), ("scale", C.c_float), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_size_t)]


# The structs are packed by hand below: a ctypes.Structure costs microseconds per
# call.  Native alignment, so the layouts are those of the classes above.
_PACK_TABLES = struct.Struct("iiiiqi11P").pack
_PACK_APPEND = struct.Struct("PPiiiiii6q" "PPii4qP").pack
_PACK_ATTENTION = struct.Struct("PPiiiiii6q" "PPii4q3PqiiifPN").pack

_I32 = torch.int32
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


class _Entries:
    """The library's entry points, looked up once."""
    tables = append = attention = None
    workspace = {}  # bytes by head_dim


def _load():
    lib = gpt.load_library()
    _Entries.tables, _Entries.append, _Entries.attention = (lib.itts_paged_tables, lib.itts_paged_append,
                                                            lib.itts_paged_attention)


def _refuse(message: str):
    raise gpt.GptInvalidArgument(gpt.ERR_INVALID_ARGUMENT, message)


def _failed(rc: int):
    gpt._raise(rc, gpt.load_library().itts_paged_last_error().decode())


def _device(t, name: str) -> int:
    device = t.get_device()
    if device < 0:
        _refuse(f"{name} must be a CUDA tensor")
    return device


def _words(t, name: str, device: int, count: int) -> int:
    """Address of a contiguous int32 tensor of at least `count` entries."""
    if t.dtype is not _I32 or t.get_device() != device or t.numel() < count or not t.is_contiguous():
        _refuse(f"{name} must be a contiguous int32 tensor of {count} entries on cuda:{device}")
    return t.data_ptr()


def _table(table, requests: int, device: int):
    """Address, row stride and columns of a block table."""
    if table.dtype is not _I32 or table.get_device() != device or table.dim() != 2:
        _refuse(f"table must be an int32 matrix on cuda:{device}")
    rows, columns = table.shape
    if rows < requests:
        _refuse(f"table must have {requests} rows")
    if table.is_contiguous():
        return table.data_ptr(), columns, columns
    if columns > 1 and table.stride(1) != 1:
        _refuse("table must have contiguous columns")
    return table.data_ptr(), (table.stride(0) if rows > 1 else columns), columns


def _cache(k_cache, v_cache, device: int):
    """The fields of an itts_paged_cache."""
    kind = k_cache.dtype
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        _refuse("k_cache and v_cache must be [blocks, block_size, heads, head_dim]")
    if kind not in _TYPES or v_cache.dtype is not kind:
        _refuse("paged cache type is f32, f16 or bf16")
    if k_cache.get_device() != device or v_cache.get_device() != device:
        _refuse(f"k_cache and v_cache must be on cuda:{device}")
    kb, kt, kh, kd = k_cache.stride()
    vb, vt, vh, vd = v_cache.stride()
    if kd != 1 or vd != 1:
        _refuse("the head dimension of a paged cache must be contiguous")
    blocks, size, heads, dim = shape
    # the stride of a dimension of one is never used, and torch may give it any value
    if blocks == 1:
        kb = vb = 0
    if heads == 1:
        kh = vh = 0
    return k_cache.data_ptr(), v_cache.data_ptr(), _TYPES[kind], blocks, size, heads, dim, 0, kb, kt, kh, vb, vt, vh


def _rows(t, name: str, dtype, dim: int, device: int):
    """Address, rows, heads and row / head strides of a [rows, heads, head_dim] tensor."""
    if t.dim() != 3 or t.dtype is not dtype or t.get_device() != device:
        _refuse(f"{name} must be [rows, heads, head_dim] of {dtype} on cuda:{device}")
    rows, heads, last = t.shape
    row, head, one = t.stride()
    if last != dim or one != 1:
        _refuse(f"{name} must have a contiguous last dimension of {dim}")
    return t.data_ptr(), rows, heads, (row if rows > 1 else 0), (head if heads > 1 else 0)


def tables(cached, fresh, table, free_list, free_count, block_size: int, *, lens, q_start, positions, slots, status,
           free_out=None):
    """A step's bookkeeping (itts_paged_tables): int32 CUDA tensors throughout.

    cached, fresh [requests]; table [requests, columns] (written); free_list
    [blocks] (written); free_count [1].  Outputs: lens [requests], q_start
    [requests + 1], positions and slots [rows], status [1] and free_out [1]
    (free_count itself if not given).  ``lens`` may be ``cached``."""
    device = _device(cached, "cached")
    n, rows = fresh.numel(), slots.numel()
    address, stride, columns = _table(table, n, device)
    count = _words(free_count, "free_count", device, 1)
    try:
        args = _PACK_TABLES(n, block_size, free_list.numel(), columns, stride, rows, _words(cached, "cached", device, n),
                            _words(fresh, "fresh", device, n), address, _words(free_list, "free_list", device, 1), count,
                            count if free_out is None else _words(free_out, "free_out", device, 1),
                            _words(lens, "lens", device, n), _words(q_start, "q_start", device, n + 1),
                            _words(positions, "positions", device, rows), _words(slots, "slots", device, rows),
                            _words(status, "status", device, 1))
    except struct.error as e:
        _refuse(f"argument out of range: {e}")
    if _Entries.tables is None:
        _load()
    rc = _Entries.tables(device, args, _stream(device))
    if rc:
        _failed(rc)


def append(k, v, k_cache, v_cache, slots):
    """Writes rows k, v [rows, heads, head_dim] (the caches' type, or float32)
    into the caches [blocks, block_size, heads, head_dim] at ``slots`` [rows];
    rows with a slot outside the cache are left out (itts_paged_append)."""
    device = _device(k, "k")
    cache = _cache(k_cache, v_cache, device)
    kind = k.dtype
    if kind not in _TYPES:
        _refuse("source type is the cache's type or f32")
    kp, rows, heads, kr, kh = _rows(k, "k", kind, cache[6], device)
    vp, vrows, vheads, vr, vh = _rows(v, "v", kind, cache[6], device)
    if vrows != rows or heads != cache[5] or vheads != cache[5]:
        _refuse("k and v must have the same rows and the caches' heads")
    try:
        args = _PACK_APPEND(*cache, kp, vp, _TYPES[kind], rows, kr, kh, vr, vh, _words(slots, "slots", device, rows))
    except struct.error as e:
        _refuse(f"argument out of range: {e}")
    if _Entries.append is None:
        _load()
    rc = _Entries.append(device, args, _stream(device))
    if rc:
        _failed(rc)


def attention(q, k_cache, v_cache, table, lens, q_start, max_fresh: int, scale: float | None = None, out=None,
              workspace=None):
    """Causal attention of the fresh rows q [rows, heads, head_dim] over the
    caches (itts_paged_attention): request b owns rows q_start[b] to
    q_start[b + 1] and its last row stands at position lens[b] - 1.
    ``max_fresh`` bounds the rows of one request.  Returns ``out`` (a new
    tensor if not given; rows behind q_start[-1] are not written).
    ``workspace``: a uint8 CUDA tensor of ``workspace_bytes(head_dim)`` that no
    other call uses at the same time; by default one is taken from torch's
    allocator for the call."""
    device = _device(q, "q")
    cache = _cache(k_cache, v_cache, device)
    kind, dim = k_cache.dtype, cache[6]
    qp, rows, heads, qr, qh = _rows(q, "q", kind, dim, device)
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=kind, device=q.device)
    op, orows, oheads, orow, oh = _rows(out, "out", kind, dim, device)
    if orows != rows or oheads != heads:
        _refuse("out must have q's shape")
    requests = lens.numel()
    address, stride, columns = _table(table, requests, device)
    if workspace is None:
        need = _Entries.workspace.get(dim)
        if need is None:
            need = _Entries.workspace[dim] = workspace_bytes(dim)
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    elif workspace.get_device() != device or workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
        _refuse(f"workspace must be a contiguous uint8 tensor on cuda:{device}")
    try:
        args = _PACK_ATTENTION(*cache, qp, op, heads, rows, qr, qh, orow, oh,
                               _words(q_start, "q_start", device, requests + 1), _words(lens, "lens", device, requests),
                               address, stride, requests, columns, max_fresh, dim ** -0.5 if scale is None else scale,
                               workspace.data_ptr(), workspace.numel())
    except struct.error as e:
        _refuse(f"argument out of range: {e}")
    if _Entries.attention is None:
        _load()
    rc = _Entries.attention(device, args, _stream(device))
    if rc:
        _failed(rc)
    return out


def workspace_bytes(head_dim: int) -> int:
    """Bytes of workspace of an ``attention`` call (0: no such head_dim)."""
    return gpt.load_library().itts_paged_attention_workspace(head_dim)
