"""The 8-bit KV cache on MI355X: keys and values as int8 or e4m3 codes in pages
of a sequence's tokens, one fp32 scale per (page, kv head) for the keys and one
for the values (layout and rounding: include/sphkv.h, "8-bit KV cache").

    cache = Cache8.allocate(num_pages, num_kv, dh, page_size=16, fmt="int8")
    cache8_write(cache, k, v, table, start, cu_rows)      # a batch's new tokens
    out = cache8_prefill(cache, q, cu_rows, table, lens)  # prompts, chunks, drafted tokens
    out = cache8_decode(cache, q, table, lens)            # one query token a sequence
    k, v = cache8_read(cache, table, start, cu_rows, num_rows)

Keys are stored as given: RoPE is the caller's, as on the LayerPool path.  The
reference has no counterpart (it stores angle codes and fp16 values).

Sequence lengths, starts and page tables stay on the device: no call waits for
the GPU, and all can be captured into a graph, whose replays then follow what
those tensors hold.  Every call launches on torch's current stream of the
cache's device.  A call's workspace is its own unless one is passed in; calls
that share one must not run concurrently.  No CPU or torch fallback exists.
"""
from __future__ import annotations

import math
from functools import lru_cache
from operator import attrgetter
from typing import Optional, Tuple

import torch

import sphkv_lib
from sphkv_lib import check

_lib = sphkv_lib.load()

FORMATS = {"int8": 0, "e4m3": 1}                # SPHKV_CACHE8_*
_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_FLOAT, _INT = torch.float32, torch.int32
# torch's raw accessors where this build has them: half a microsecond a call less
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_device_index = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _need(t: torch.Tensor, dtype, name: str, device=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU device (the library has no CPU path)")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


class Cache8:
    """A layer's 8-bit cache over its three tensors:

    k_codes uint8 [num_pages, num_kv, page_size, dh], v_codes uint8 [num_pages,
    num_kv, page_size/16, dh, 16], scales fp32 [num_pages, num_kv, 2] (keys,
    values), contiguous and 16-byte aligned; fmt "int8" or "e4m3".  The tensors
    and what follows from them are read-only: a cache over others is another
    Cache8."""

    __slots__ = ("_k_codes", "_v_codes", "_scales", "_fmt", "_num_pages", "_num_kv", "_page_size", "_dh", "_device",
                 "_tail", "_index", "_sm")
    k_codes, v_codes, scales = (property(attrgetter(n)) for n in ("_k_codes", "_v_codes", "_scales"))
    fmt, device = property(attrgetter("_fmt")), property(attrgetter("_device"))
    num_pages, num_kv = property(attrgetter("_num_pages")), property(attrgetter("_num_kv"))
    page_size, dh = property(attrgetter("_page_size")), property(attrgetter("_dh"))

    def __init__(self, k_codes: torch.Tensor, v_codes: torch.Tensor, scales: torch.Tensor, fmt: str = "int8"):
        if fmt not in FORMATS:
            raise ValueError(f"fmt must be one of {sorted(FORMATS)}, got {fmt!r}")
        _need(k_codes, torch.uint8, "k_codes")
        dev = k_codes.device
        _need(v_codes, torch.uint8, "v_codes", dev)
        _need(scales, torch.float32, "scales", dev)
        if k_codes.dim() != 4:
            raise ValueError("k_codes must be [num_pages, num_kv, page_size, dh]")
        num_pages, num_kv, page_size, dh = k_codes.shape
        if not 1 <= num_kv <= 1024:
            raise ValueError(f"num_kv must be in [1, 1024], got {num_kv}")
        if page_size not in (16, 32, 64, 128):
            raise ValueError(f"page_size must be 16, 32, 64 or 128, got {page_size}")
        if dh not in (64, 128):
            raise ValueError(f"dh must be 64 or 128, got {dh}")
        if v_codes.shape != (num_pages, num_kv, page_size // 16, dh, 16):
            raise ValueError("v_codes must be [num_pages, num_kv, page_size/16, dh, 16]")
        if scales.shape != (num_pages, num_kv, 2):
            raise ValueError("scales must be [num_pages, num_kv, 2]")
        if not (k_codes.is_contiguous() and v_codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("k_codes, v_codes and scales must be contiguous")
        self._k_codes, self._v_codes, self._scales, self._fmt = k_codes, v_codes, scales, fmt
        self._num_pages, self._num_kv, self._page_size, self._dh, self._device = num_pages, num_kv, page_size, dh, dev
        self._index = dev.index
        self._tail = (dh, page_size, FORMATS[fmt])
        self._sm = 1.0 / math.sqrt(dh)

    @staticmethod
    def allocate(num_pages: int, num_kv: int, dh: int, page_size: int = 16, fmt: str = "int8",
                 device="cuda") -> "Cache8":
        """An empty cache (zeros)."""
        k = torch.zeros((num_pages, num_kv, page_size, dh), dtype=torch.uint8, device=device)
        v = torch.zeros((num_pages, num_kv, max(page_size // 16, 1), dh, 16), dtype=torch.uint8, device=device)
        return Cache8(k, v, torch.zeros((num_pages, num_kv, 2), dtype=torch.float32, device=device), fmt)

    def _ptrs(self):
        """The call's arguments from k_codes to num_kv."""
        return (self._k_codes.data_ptr(), self._v_codes.data_ptr(), self._scales.data_ptr(), self._num_pages, self._num_kv)

    def _call(self, fn, *args) -> None:
        """Launch on torch's current stream of the cache's device, that device current."""
        if _device_index() != self._index:
            with torch.cuda.device(self._device):
                return self._call(fn, *args)
        rc = fn(*args, _raw_stream(self._index) if _raw_stream else torch.cuda.current_stream(self._device).cuda_stream)
        if rc:
            check(rc, fn.__name__)


def _seq_args(cache: Cache8, table: torch.Tensor, at: torch.Tensor, cu_rows: Optional[torch.Tensor], name: str):
    """Checks of a batch's page table, per-sequence int32 values and row starts;
    (table, row stride, blocks, sequences) for the call."""
    dev = cache._device
    _need(table, _INT, "table", dev)
    _need(at, _INT, name, dev)
    if table.dim() != 2 or at.dim() != 1:
        raise ValueError(f"table must be [num_seqs, max_blocks] and {name} [num_seqs]")
    n, blocks = table.shape
    row, one = table.stride()
    if at.shape[0] != n:
        raise ValueError(f"table must be [num_seqs, max_blocks] and {name} [num_seqs]")
    if (blocks > 1 and one != 1) or (n > 1 and at.stride(0) != 1):
        raise ValueError(f"table's rows and {name} must be contiguous")
    if n > 1 and row < blocks:
        raise ValueError("table's rows must not overlap")
    if cu_rows is not None:
        _need(cu_rows, _INT, "cu_rows", dev)
        if cu_rows.dim() != 1 or cu_rows.shape[0] != n + 1 or cu_rows.stride(0) != 1:
            raise ValueError("cu_rows must be a contiguous [num_seqs + 1]")
    return table.data_ptr(), row, blocks, n


def _rows(t: torch.Tensor, name: str, heads: int, dh: int):
    """Checks of [rows, heads, dh] rows of any row and head stride; (row, head) strides."""
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dh:
        raise ValueError(f"{name} must be [rows, {heads}, {dh}], got {tuple(shape)}")
    row, head, one = t.stride()
    if one != 1:
        raise ValueError(f"the {dh} elements of a row of {name} must be contiguous")
    return row, head


def _out(t: Optional[torch.Tensor], shape, dtype, name: str, cache: Cache8) -> torch.Tensor:
    if t is None:
        return torch.empty(shape, dtype=dtype, device=cache._device)
    _need(t, dtype, name, cache._device)
    if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {tuple(shape)}")
    return t


def cache8_write(cache: Cache8, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor,
                 cu_rows: Optional[torch.Tensor] = None) -> None:
    """Quantise new tokens into their sequences' pages (sphkv_cache8_write).

    k, v [rows, num_kv, dh] fp16, bf16 or fp32, of any row and head stride:
    sequence s's tokens are rows cu_rows[s] .. cu_rows[s+1] - 1 (int32
    [num_seqs + 1]; None: row s, one token each) at positions start[s] on
    (int32 [num_seqs]), in the pages table[s] (int32 [num_seqs, max_blocks]).
    A page whose first slot is written starts over with a scale of its own;
    another page's scale grows where its new tokens need it, and the codes it
    held are rounded to the new scale.  A written page belongs to one sequence.
    Tokens past the table, of a negative start or of a page outside the cache
    are dropped."""
    tab, stride, blocks, n = _seq_args(cache, table, start, cu_rows, "start")
    if not isinstance(k, torch.Tensor) or k.dtype not in _TYPES:
        raise TypeError("k must be an fp16, bf16 or fp32 tensor")
    _need(k, k.dtype, "k", cache._device)
    _need(v, k.dtype, "v", cache._device)
    k_row, k_head = _rows(k, "k", cache._num_kv, cache._dh)
    v_row, v_head = _rows(v, "v", cache._num_kv, cache._dh)
    rows = k.shape[0]
    if v.shape[0] != rows:
        raise ValueError("k and v must have as many rows")
    if cu_rows is None and rows != n:
        raise ValueError("without cu_rows there is one row per sequence")
    cache._call(_lib.sphkv_cache8_write, k.data_ptr(), v.data_ptr(), _TYPES[k.dtype], k_row, k_head, v_row, v_head, rows,
                None if cu_rows is None else cu_rows.data_ptr(), start.data_ptr(), tab, stride, blocks, n, *cache._ptrs(),
                *cache._tail)


def cache8_read(cache: Cache8, table: torch.Tensor, start: torch.Tensor, cu_rows: Optional[torch.Tensor] = None,
                num_rows: Optional[int] = None, dtype: torch.dtype = torch.float16,
                k_out: Optional[torch.Tensor] = None, v_out: Optional[torch.Tensor] = None
                ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Tokens back as (k, v) [num_rows, num_kv, dh] of `dtype` (fp16, bf16 or
    fp32): the fp32 product code * scale, rounded to it (sphkv_cache8_read).  Rows and positions
    as in cache8_write; num_rows is cu_rows' last value, or more (None: one
    token each, num_seqs).  Rows behind the last sequence are left as they were
    in k_out and v_out.  Tokens past the table, of a negative position or of a
    page outside the cache read as zeros."""
    tab, stride, blocks, n = _seq_args(cache, table, start, cu_rows, "start")
    if dtype not in _TYPES:
        raise TypeError("dtype must be fp16, bf16 or fp32")
    if cu_rows is None:
        if num_rows is not None and num_rows != n:
            raise ValueError("without cu_rows there is one row per sequence")
        num_rows = n
    elif num_rows is None or num_rows < 0:
        raise ValueError("num_rows (cu_rows' last value, or more) is needed with cu_rows")
    shape = (int(num_rows), cache._num_kv, cache._dh)
    k_out, v_out = _out(k_out, shape, dtype, "k_out", cache), _out(v_out, shape, dtype, "v_out", cache)
    cache._call(_lib.sphkv_cache8_read, *cache._ptrs(), *cache._tail, None if cu_rows is None else cu_rows.data_ptr(),
                start.data_ptr(), tab, stride, blocks, n, shape[0], k_out.data_ptr(), v_out.data_ptr(), _TYPES[dtype])
    return k_out, v_out


def _query(cache: Cache8, q: torch.Tensor):
    """Checks of q; (shape, q heads per kv head, row stride, head stride)."""
    if not isinstance(q, torch.Tensor) or (q.dtype is not torch.float16 and q.dtype is not torch.bfloat16):
        raise TypeError("q must be an fp16 or bf16 tensor")
    _need(q, q.dtype, "q", cache._device)
    shape = q.shape
    if len(shape) != 3 or shape[1] == 0 or shape[1] % cache._num_kv:
        raise ValueError("q must be [rows, num_kv * gqa, dh]")
    return shape, shape[1] // cache._num_kv, *_rows(q, "q", shape[1], cache._dh)


def _workspace(cache: Cache8, need: int, workspace: Optional[torch.Tensor]):
    """(pointer, bytes, tensor) of a caller's workspace or of a new one."""
    if workspace is None:
        if need <= 0:
            return None, 0, None
        workspace = torch.empty(need, dtype=torch.uint8, device=cache._device)
    else:
        _need(workspace, torch.uint8, "workspace", cache._device)
        if not workspace.is_contiguous() or workspace.numel() < need:
            raise ValueError(f"workspace must be contiguous and hold {need} bytes, got {workspace.numel()}")
    return workspace.data_ptr(), workspace.numel(), workspace


@lru_cache(maxsize=256)
def _decode_bytes(num_seqs: int, num_kv: int, gqa: int, dh: int) -> int:
    return _lib.sphkv_cache8_decode_workspace_bytes(num_seqs, num_kv, gqa, dh)


@lru_cache(maxsize=256)
def _prefill_bytes(num_rows: int, num_seqs: int, num_kv: int, gqa: int, dh: int) -> int:
    return _lib.sphkv_cache8_prefill_workspace_bytes(num_rows, num_seqs, num_kv, gqa, dh)


def decode_workspace_bytes(cache: Cache8, num_seqs: int, gqa: int) -> int:
    """Bytes of a workspace for cache8_decode of num_seqs sequences."""
    n = _decode_bytes(int(num_seqs), cache._num_kv, int(gqa), cache._dh)
    if n < 0:
        raise ValueError("bad num_seqs or gqa (1..64) for the decode workspace")
    return n


def prefill_workspace_bytes(cache: Cache8, num_rows: int, num_seqs: int, gqa: int) -> int:
    """Bytes of a workspace for cache8_prefill of num_rows rows of num_seqs sequences."""
    n = _prefill_bytes(int(num_rows), int(num_seqs), cache._num_kv, int(gqa), cache._dh)
    if n < 0:
        raise ValueError("bad num_rows, num_seqs or gqa (1..64) for the prefill workspace")
    return n


def cache8_decode(cache: Cache8, q: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                  sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None, return_lse: bool = False,
                  lse: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
    """Attention of one query token per sequence over the first lens[s] tokens
    of its pages (sphkv_cache8_decode).  q [num_seqs, num_kv * gqa, dh] fp16 or
    bf16, gqa up to 64; lens int32 [num_seqs]; sm_scale 1 / sqrt(dh) unless
    given.  Returns out (q's shape and type), with return_lse (out, lse):
    lse fp32 [num_seqs, num_kv * gqa] is the natural log of the softmax's sum.
    A sequence without tokens gets zeros and -inf."""
    tab, stride, blocks, n = _seq_args(cache, table, lens, None, "lens")
    shape, gqa, q_row, q_head = _query(cache, q)
    if shape[0] != n:
        raise ValueError("q must have one row per sequence")
    out = _out(out, shape, q.dtype, "out", cache)
    if return_lse or lse is not None:
        lse = _out(lse, shape[:2], _FLOAT, "lse", cache)
    ws, nbytes, _keep = _workspace(cache, decode_workspace_bytes(cache, n, gqa), workspace)
    cache._call(_lib.sphkv_cache8_decode, q.data_ptr(), _TYPES[q.dtype], q_row, q_head, lens.data_ptr(), tab, stride, blocks,
                n, *cache._ptrs(), gqa, *cache._tail, cache._sm if sm_scale is None else float(sm_scale), out.data_ptr(),
                None if lse is None else lse.data_ptr(), ws, nbytes)
    return (out, lse) if return_lse else out


def cache8_prefill(cache: Cache8, q: torch.Tensor, cu_rows: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                   causal: bool = True, sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                   return_lse: bool = False, lse: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None):
    """Attention of several query tokens per sequence, the last ones of its
    lens[s] tokens (sphkv_cache8_prefill): row cu_rows[s] + i of q [rows, num_kv
    * gqa, dh] is at position lens[s] - n_s + i and attends the tokens up to
    its own (causal) or all lens[s].  Write the tokens first.  Rows that attend
    nothing get zeros and -inf; rows behind the last sequence are left as they
    were in out and lse.  A softmax weight meets its value with 22 bits for fp16
    q, with 11 for bf16.  Few tokens on a long context are slow beside many short
    sequences (the keys are split evenly over a batch): give them a call of their
    own.  The rest as cache8_decode."""
    if cu_rows is None:
        raise TypeError("cu_rows must be a torch.Tensor")
    tab, stride, blocks, n = _seq_args(cache, table, lens, cu_rows, "lens")
    shape, gqa, q_row, q_head = _query(cache, q)
    out = _out(out, shape, q.dtype, "out", cache)
    if return_lse or lse is not None:
        lse = _out(lse, shape[:2], _FLOAT, "lse", cache)
    ws, nbytes, _keep = _workspace(cache, prefill_workspace_bytes(cache, shape[0], n, gqa), workspace)
    cache._call(_lib.sphkv_cache8_prefill, q.data_ptr(), _TYPES[q.dtype], q_row, q_head, shape[0], cu_rows.data_ptr(),
                lens.data_ptr(), 1 if causal else 0, tab, stride, blocks, n, *cache._ptrs(), gqa, *cache._tail,
                cache._sm if sm_scale is None else float(sm_scale), out.data_ptr(),
                None if lse is None else lse.data_ptr(), ws, nbytes)
    return (out, lse) if return_lse else out
