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


def _refuse(message: str):
    raise gpt.GptInvalidArgument(gpt.ERR_INVALID_ARGUMENT, message)


def _run(entry, args, device: torch.device):
    rc = entry(device.index, C.byref(args), torch._C._cuda_getCurrentRawStream(device.index))
    if rc != gpt.OK:
        gpt._raise(rc, gpt.load_library().itts_paged_last_error().decode())


def _words(t, name: str, device, count: int):
    """Address of a contiguous int32 vector of at least `count` entries."""
    if t.dtype is not torch.int32 or t.device != device or t.dim() != 1 or t.shape[0] < count or \
            (t.shape[0] > 1 and t.stride(0) != 1):
        _refuse(f"{name} must be a contiguous int32 vector of {count} entries on {device}")
    return t.data_ptr()


def _table(table, requests: int, device):
    if table.dtype is not torch.int32 or table.device != device or table.dim() != 2 or table.shape[0] < requests or \
            (table.shape[1] > 1 and table.stride(1) != 1):
        _refuse(f"table must be an int32 matrix of {requests} rows, contiguous columns, on {device}")
    return table.data_ptr(), (table.stride(0) if table.shape[0] > 1 else table.shape[1]), table.shape[1]


def _cuda(t, name: str) -> torch.device:
    if not t.is_cuda:
        _refuse(f"{name} must be a CUDA tensor")
    return t.device


def _cache(k_cache, v_cache, device) -> Cache:
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        _refuse("k_cache and v_cache must be [blocks, block_size, heads, head_dim]")
    if k_cache.dtype not in _TYPES or v_cache.dtype is not k_cache.dtype:
        _refuse("paged cache type is f32, f16 or bf16")
    if k_cache.device != device or v_cache.device != device:
        _refuse(f"k_cache and v_cache must be on {device}")
    kb, kt, kh, kd = k_cache.stride()
    vb, vt, vh, vd = v_cache.stride()
    if kd != 1 or vd != 1:
        _refuse("the head dimension of a paged cache must be contiguous")
    blocks, size, heads, dim = k_cache.shape
    # the stride of a dimension of one is never used, and torch may give it any value
    if blocks == 1:
        kb = vb = 0
    if heads == 1:
        kh = vh = 0
    return Cache(k_cache.data_ptr(), v_cache.data_ptr(), _TYPES[k_cache.dtype], blocks, size, heads, dim, 0, kb, kt,
                 kh, vb, vt, vh)


def _rows(t, name: str, dtype, heads, dim: int, device):
    """Address and row / head strides of a [rows, heads, head_dim] tensor."""
    if t.dim() != 3 or t.shape[2] != dim or (heads and t.shape[1] != heads) or t.dtype is not dtype or \
            t.device != device or t.stride(2) != 1:
        _refuse(f"{name} must be [rows, heads, {dim}] of {dtype} with a contiguous last dimension on {device}")
    return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0


def tables(cached, fresh, table, free_list, free_count, block_size: int, *, lens, q_start, positions, slots, status,
           free_out=None):
    """A step's bookkeeping (itts_paged_tables): int32 CUDA tensors throughout.

    cached, fresh [requests]; table [requests, columns] (written); free_list
    [blocks] (written); free_count [1].  Outputs: lens [requests], q_start
    [requests + 1], positions and slots [rows], status [1] and free_out [1]
    (free_count itself if not given).  ``lens`` may be ``cached``."""
    device = _cuda(cached, "cached")
    n, rows = fresh.shape[0] if fresh.dim() == 1 else -1, slots.shape[0] if slots.dim() == 1 else -1
    address, stride, columns = _table(table, n, device)
    count = _words(free_count, "free_count", device, 1)
    blocks = free_list.shape[0] if free_list.dim() == 1 else -1
    a = Tables(n, block_size, blocks, columns, stride, rows, _words(cached, "cached", device, n),
               _words(fresh, "fresh", device, n), address, _words(free_list, "free_list", device, 1), count,
               count if free_out is None else _words(free_out, "free_out", device, 1),
               _words(lens, "lens", device, n), _words(q_start, "q_start", device, n + 1),
               _words(positions, "positions", device, rows), _words(slots, "slots", device, rows),
               _words(status, "status", device, 1))
    _run(gpt.load_library().itts_paged_tables, a, device)


def append(k, v, k_cache, v_cache, slots):
    """Writes rows k, v [rows, heads, head_dim] (the caches' type, or float32)
    into the caches [blocks, block_size, heads, head_dim] at ``slots`` [rows];
    rows with a slot outside the cache are left out (itts_paged_append)."""
    device = _cuda(k, "k")
    c = _cache(k_cache, v_cache, device)
    if k.dtype not in _TYPES:
        _refuse("source type is the cache's type or f32")
    rows = k.shape[0]
    kp, kr, kh = _rows(k, "k", k.dtype, c.heads, c.head_dim, device)
    vp, vr, vh = _rows(v, "v", k.dtype, c.heads, c.head_dim, device)
    if v.shape[0] != rows:
        _refuse("k and v must have the same rows")
    a = Append(c, kp, vp, _TYPES[k.dtype], rows, kr, kh, vr, vh, _words(slots, "slots", device, rows))
    _run(gpt.load_library().itts_paged_append, a, device)


_WORKSPACE: dict = {}  # bytes by head_dim


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
    device = _cuda(q, "q")
    c = _cache(k_cache, v_cache, device)
    qp, qr, qh = _rows(q, "q", k_cache.dtype, None, c.head_dim, device)
    rows, heads = q.shape[0], q.shape[1]
    if out is None:
        out = torch.empty((rows, heads, c.head_dim), dtype=q.dtype, device=device)
    elif out.shape[0] != rows:
        _refuse("out must have q's shape")
    op, orow, oh = _rows(out, "out", k_cache.dtype, heads, c.head_dim, device)
    requests = lens.shape[0] if lens.dim() == 1 else -1
    address, stride, columns = _table(table, requests, device)
    need = _WORKSPACE.get(c.head_dim)
    if need is None:
        need = _WORKSPACE[c.head_dim] = workspace_bytes(c.head_dim)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif workspace.device != device or workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
        _refuse(f"workspace must be a contiguous uint8 tensor on {device}")
    a = Attention(c, qp, op, heads, rows, qr, qh, orow, oh, _words(q_start, "q_start", device, requests + 1),
                  _words(lens, "lens", device, requests), address, stride, requests, columns, max_fresh,
                  c.head_dim ** -0.5 if scale is None else scale, workspace.data_ptr(), workspace.numel())
    _run(gpt.load_library().itts_paged_attention, a, device)
    return out


def workspace_bytes(head_dim: int) -> int:
    """Bytes of workspace of an ``attention`` call (0: no such head_dim)."""
    return gpt.load_library().itts_paged_attention_workspace(head_dim)
