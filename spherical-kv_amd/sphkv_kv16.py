"""The 16-bit KV cache on MI355X: keys and values as fp16 or bf16 numbers in
pages of a sequence's tokens, filled with the keys' rotation on the way and read
by attention and differential attention (include/sphkv.h, "16-bit KV cache").

    cache = Cache16.allocate(num_pages, num_kv, dh, page_size=16, dtype=torch.bfloat16)
    q = cache16_append(cache, k, v, table, start, cu_rows, inv_freq=f, q=q)   # a batch's new tokens
    out = cache16_prefill(cache, q, cu_rows, table, lens)    # prompts, chunks, drafted tokens
    out = cache16_decode(cache, q, table, lens)              # one query token a sequence
    out = cache16_diff_prefill(cache, q, lam, cu_rows, table, lens, norm_weight=w)
    out = cache16_diff_decode(cache, q, lam, table, lens, norm_weight=w)

The reference has no counterpart (it stores angle codes and fp16 values).

Sequence lengths, starts and page tables stay on the device: no call waits for
the GPU, and all can be captured into a graph, whose replays then follow what
those tensors hold.  Every call launches on torch's current stream of the
cache's device.  A call's workspace is its own unless one is passed in; calls
that share one must not run concurrently.  No CPU or torch fallback exists.
"""
from __future__ import annotations

import ctypes
import math
from functools import lru_cache
from operator import attrgetter
from typing import Optional

import torch

import sphkv_lib
from sphkv_kv8 import _FLOAT, _INT, _TYPES, _device_index, _need, _out, _raw_stream, _rows, _seq_args, _workspace
from sphkv_lib import check

_lib = sphkv_lib.load()

_Tensor = torch.Tensor
_FREQ_TYPES = {torch.float32: 2, torch.float64: 3}         # SPHKV_FP32, SPHKV_FP64


def rope_inv_freq(dim: int, theta: float = 500000.0, device="cuda") -> torch.Tensor:
    """Radians per token of the pairs of `dim` rotated elements, unscaled RoPE: theta^(-2j/dim), fp64."""
    return float(theta) ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)


class Cache16:
    """A layer's 16-bit cache over its two tensors k, v [num_pages, num_kv,
    page_size, dh], both fp16 or both bf16, 16-byte aligned, the dh elements of a
    token contiguous.  Pages, heads and tokens may lie in any order, their
    strides multiples of 8 elements: a tensor of [num_pages, page_size, num_kv,
    dh] comes in as x.transpose(1, 2), one of two as kv[:, 0] and kv[:, 1].  A
    cache whose tokens share memory (an expanded view, one tensor as k and v) is
    for attention alone, an append to it is refused.  The tensors and what follows from them are read-only: a cache over others is
    another Cache16."""

    __slots__ = ("_k", "_v", "_num_pages", "_num_kv", "_page_size", "_dh", "_device", "_dtype", "_index", "_type", "_struct",
                 "_ref", "_at", "_sm")
    k, v, dtype, device = (property(attrgetter(n)) for n in ("_k", "_v", "_dtype", "_device"))
    num_pages, num_kv = property(attrgetter("_num_pages")), property(attrgetter("_num_kv"))
    page_size, dh = property(attrgetter("_page_size")), property(attrgetter("_dh"))

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if not isinstance(k, torch.Tensor) or (k.dtype is not torch.float16 and k.dtype is not torch.bfloat16):
            raise TypeError("k must be an fp16 or bf16 tensor")
        _need(k, k.dtype, "k")
        _need(v, k.dtype, "v", k.device)
        if k.dim() != 4:
            raise ValueError("k must be [num_pages, num_kv, page_size, dh]")
        num_pages, num_kv, page_size, dh = k.shape
        if v.shape != k.shape:
            raise ValueError("v must be [num_pages, num_kv, page_size, dh] as k is")
        if not 1 <= num_kv <= 1024:
            raise ValueError(f"num_kv must be in [1, 1024], got {num_kv}")
        if page_size not in (16, 32, 64, 128):
            raise ValueError(f"page_size must be 16, 32, 64 or 128, got {page_size}")
        if dh not in (64, 128):
            raise ValueError(f"dh must be 64 or 128, got {dh}")
        strides = []
        for name, t in (("k", k), ("v", v)):
            *three, one = t.stride()
            # (a stride over one page or one head takes part in no address)
            three = [x if n > 1 else 0 for x, n in zip(three, t.shape)]
            if one != 1 or any(x % 8 for x in three) or (num_pages > 0 and t.data_ptr() % 16):
                raise ValueError(f"the {dh} elements of a token of {name} must be contiguous, its other strides multiples of 8, "
                                 "its start 16-byte aligned")
            strides += three
        self._k, self._v, self._dtype, self._device, self._index = k, v, k.dtype, k.device, k.device.index
        self._num_pages, self._num_kv, self._page_size, self._dh = num_pages, num_kv, page_size, dh
        self._type, self._sm = _TYPES[k.dtype], 1.0 / math.sqrt(dh)
        self._at = k.data_ptr(), v.data_ptr()
        self._struct = sphkv_lib.Cache16Struct(*self._at, *strides, num_pages, num_kv, dh, page_size, self._type)
        self._ref = ctypes.addressof(self._struct)

    @staticmethod
    def allocate(num_pages: int, num_kv: int, dh: int, page_size: int = 16, dtype: torch.dtype = torch.float16,
                 device="cuda") -> "Cache16":
        """An empty cache (zeros)."""
        shape = (num_pages, num_kv, page_size, dh)
        return Cache16(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))

    def _address(self) -> int:
        """The struct's address, over what the tensors are now."""
        at = self._k.data_ptr(), self._v.data_ptr()
        if at != self._at:
            self._struct.k, self._struct.v = self._at = at
        return self._ref

    def _call(self, fn, *args) -> None:
        """Launch on torch's current stream of the cache's device, that device current."""
        if _device_index() != self._index:
            with torch.cuda.device(self._device):
                return self._call(fn, *args)
        rc = fn(*args, _raw_stream(self._index) if _raw_stream else torch.cuda.current_stream(self._device).cuda_stream)
        if rc:
            check(rc, fn.__name__)


# A plain tensor of the right type on the cache's device passes by three comparisons;
# anything else goes through _need, _seq_args and _rows, which say what is wrong, or
# that nothing is (one token's append 8.9 us of the host, 10.4 with those alone).

def _seqs(cache: Cache16, table: torch.Tensor, at: torch.Tensor, cu_rows: Optional[torch.Tensor], name: str):
    """_seq_args of the ordinary case; (table, row stride, blocks, sequences) for the call."""
    index = cache._index
    if (type(table) is _Tensor and type(at) is _Tensor and table.dtype is _INT and at.dtype is _INT
            and table.get_device() == index and at.get_device() == index):
        shape = table.shape
        if len(shape) == 2 and at.shape == shape[:1]:
            n, blocks = shape
            row, one = table.stride()
            if (one == 1 or blocks <= 1) and (n == 1 or (row >= blocks and at.is_contiguous())) and (
                    cu_rows is None or (type(cu_rows) is _Tensor and cu_rows.dtype is _INT and cu_rows.get_device() == index
                                        and cu_rows.shape == (n + 1,) and cu_rows.is_contiguous())):
                return table.data_ptr(), row, blocks, n
    return _seq_args(cache, table, at, cu_rows, name)


def cache16_append(cache: Cache16, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor,
                   cu_rows: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
                   interleaved: bool = False, parts: int = 1, q: Optional[torch.Tensor] = None,
                   q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Append new tokens to their sequences' pages, the keys rotated by their
    positions, and rotate the same tokens' queries (sphkv_cache16_append).

    k, v [rows, num_kv, dh] and q [rows, num_kv * gqa, dh] all fp16, bf16 or
    fp32, of any row and head stride: sequence s's tokens are rows cu_rows[s] ..
    cu_rows[s+1] - 1 (int32 [num_seqs + 1]; None: row s, one token each) at
    positions start[s] on (int32 [num_seqs]), in the pages table[s] (int32
    [num_seqs, max_blocks]).  Keys, values and queries are rounded once, to the
    cache's type.

    inv_freq, fp32 or fp64 [n], n a multiple of 8: radians per token of the n
    pairs in the first 2n elements of each of `parts` (1 or 2) equal parts of a
    head, pair j of elements j and j + n, or 2j and 2j + 1 if interleaved; the
    rest stays (None: all).  Two parts: the two maps of differential attention.

    Returns the rotated queries [rows, num_kv * gqa, dh] of the cache's type (None
    without q), in q_out if that is given: any row and head stride, q itself too
    (other memory of q, k or v is refused).
    Keys and values past the table, of a sequence with a negative start or of a
    page outside the cache are dropped; rows behind the last sequence are left as
    they were in q_out.  A written page belongs to one sequence."""
    if parts not in (1, 2):
        raise ValueError(f"parts must be 1 or 2, got {parts}")
    tab, stride, blocks, n = _seqs(cache, table, start, cu_rows, "start")
    if not isinstance(k, _Tensor) or k.dtype not in _TYPES:
        raise TypeError("k must be an fp16, bf16 or fp32 tensor")
    dtype, dev, index, heads, dh = k.dtype, cache._device, cache._index, cache._num_kv, cache._dh
    if k.get_device() != index:
        _need(k, dtype, "k", dev)
    if type(v) is not _Tensor or v.dtype is not dtype or v.get_device() != index:
        _need(v, dtype, "v", dev)
    shape = k.shape
    rows = shape[0] if shape else 0
    k_row, k_head = _rows(k, "k", heads, dh)
    if v.shape == shape:
        v_row, v_head, one = v.stride()
        if one != 1:
            _rows(v, "v", heads, dh)
    else:
        _rows(v, "v", heads, dh)
        raise ValueError("k and v must have as many rows")
    if cu_rows is None and rows != n:
        raise ValueError("without cu_rows there is one row per sequence")
    q_ptr = o_ptr = None
    q_row = q_head = o_row = o_head = gqa = 0
    if q is not None:
        if type(q) is not _Tensor or q.dtype is not dtype or q.get_device() != index:
            _need(q, dtype, "q", dev)
        shape = q.shape
        if len(shape) != 3 or shape[0] != rows or shape[1] == 0 or shape[1] % heads:
            raise ValueError("q must be [rows, num_kv * gqa, dh], as many rows as k")
        gqa = shape[1] // heads
        q_row, q_head = _rows(q, "q", shape[1], dh)
        if q_out is None:
            q_out = _like(q, cache._dtype)
            o_row, o_head = shape[1] * dh, dh
        else:
            _need(q_out, cache._dtype, "q_out", dev)
            if q_out.shape != shape:
                raise ValueError(f"q_out must be {tuple(shape)}")
            o_row, o_head = _rows(q_out, "q_out", shape[1], dh)
            size = dh
            for st, count in sorted(x for x in ((o_row, rows), (o_head, shape[1])) if x[1] > 1):
                if st < size:
                    raise ValueError("rows and heads of q_out overlap")
                size += st * (count - 1)
        q_ptr, o_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out goes with q")
    f_ptr, f_type, freqs = None, 0, 0
    if inv_freq is not None:
        if not isinstance(inv_freq, _Tensor) or inv_freq.dtype not in _FREQ_TYPES:
            raise TypeError("inv_freq must be an fp32 or fp64 tensor")
        if inv_freq.get_device() != index:
            _need(inv_freq, inv_freq.dtype, "inv_freq", dev)
        shape = inv_freq.shape
        if len(shape) != 1 or not inv_freq.is_contiguous():
            raise ValueError("inv_freq must be a contiguous [n]")
        f_ptr, f_type, freqs = inv_freq.data_ptr(), _FREQ_TYPES[inv_freq.dtype], shape[0]
    cache._call(_lib.sphkv_cache16_append, cache._address(), k.data_ptr(), v.data_ptr(), q_ptr, _TYPES[dtype], k_row, k_head,
                v_row, v_head, q_row, q_head, gqa, o_ptr, o_row, o_head, rows, None if cu_rows is None else cu_rows.data_ptr(),
                start.data_ptr(), tab, stride, blocks, n, f_ptr, f_type, freqs, parts, 1 if interleaved else 0)
    return q_out


def _like(q: torch.Tensor, dtype) -> torch.Tensor:
    """A contiguous tensor of q's shape."""
    if q.dtype is dtype and q.is_contiguous():
        return torch.empty_like(q)
    return q.new_empty(tuple(q.shape), dtype=dtype)


def _query(cache: Cache16, q: torch.Tensor):
    """Checks of q; (shape, q heads per kv head, row stride, head stride)."""
    if type(q) is not _Tensor or q.dtype is not cache._dtype or q.get_device() != cache._index:
        _need(q, cache._dtype, "q", cache._device)
    shape = q.shape
    if len(shape) != 3 or shape[1] == 0 or shape[1] % cache._num_kv:
        raise ValueError("q must be [rows, num_kv * gqa, dh]")
    return shape, shape[1] // cache._num_kv, *_rows(q, "q", shape[1], cache._dh)


@lru_cache(maxsize=256)
def _decode_bytes(num_seqs: int, num_kv: int, gqa: int, dh: int, differential: int) -> int:
    return _lib.sphkv_cache16_decode_workspace_bytes(num_seqs, num_kv, gqa, dh, differential)


@lru_cache(maxsize=256)
def _prefill_bytes(num_rows: int, num_seqs: int, num_kv: int, gqa: int, dh: int, differential: int) -> int:
    return _lib.sphkv_cache16_prefill_workspace_bytes(num_rows, num_seqs, num_kv, gqa, dh, differential)


def decode_workspace_bytes(cache: Cache16, num_seqs: int, gqa: int, differential: bool = False) -> int:
    """Bytes of a workspace for cache16_decode (cache16_diff_decode) of num_seqs sequences."""
    n = _decode_bytes(int(num_seqs), cache._num_kv, int(gqa), cache._dh, 1 if differential else 0)
    if n < 0:
        raise ValueError("bad num_seqs or gqa (1..64, 1..32 differential) for the decode workspace")
    return n


def prefill_workspace_bytes(cache: Cache16, num_rows: int, num_seqs: int, gqa: int, differential: bool = False) -> int:
    """Bytes of a workspace for cache16_prefill (cache16_diff_prefill) of num_rows rows of num_seqs sequences."""
    n = _prefill_bytes(int(num_rows), int(num_seqs), cache._num_kv, int(gqa), cache._dh, 1 if differential else 0)
    if n < 0:
        raise ValueError("bad num_rows, num_seqs or gqa (1..64, 1..32 differential) for the prefill workspace")
    return n


def _diff_args(cache: Cache16, lam: torch.Tensor, heads: int, norm_weight: Optional[torch.Tensor], norm_eps: float):
    """Checks of differential attention's weights; their part of the call's arguments."""
    _need(lam, _FLOAT, "lam", cache._device)
    if lam.shape != (heads,) or (heads > 1 and lam.stride(0) != 1):
        raise ValueError(f"lam must be a contiguous [{heads}]")
    if norm_weight is not None:
        _need(norm_weight, _FLOAT, "norm_weight", cache._device)
        if norm_weight.shape != (cache._dh,) or norm_weight.stride(0) != 1:
            raise ValueError(f"norm_weight must be a contiguous [{cache._dh}]")
    return lam.data_ptr(), None if norm_weight is None else norm_weight.data_ptr(), float(norm_eps)


def _window(window) -> int:
    w = int(window)
    if w != window or not 0 <= w < 2 ** 31:
        raise ValueError(f"window must be a non-negative int32, got {window}")
    return w


def _decode(cache, q, table, lens, window, sm_scale, out, return_lse, lse, workspace, diff):
    tab, stride, blocks, n = _seqs(cache, table, lens, None, "lens")
    shape, gqa, q_row, q_head = _query(cache, q)
    if shape[0] != n:
        raise ValueError("q must have one row per sequence")
    if diff is None:
        fn, more, scale, maps = _lib.sphkv_cache16_decode, (), cache._sm, ()
    else:
        fn, more, scale, maps = _lib.sphkv_cache16_diff_decode, _diff_args(cache, diff[0], shape[1], *diff[1:]), math.sqrt(2.0) * cache._sm, (2,)
    out = _like(q, cache._dtype) if out is None else _out(out, shape, cache._dtype, "out", cache)
    if return_lse or lse is not None:
        lse = _out(lse, (shape[0], shape[1], *maps), _FLOAT, "lse", cache)
    need = _decode_bytes(n, cache._num_kv, gqa, cache._dh, 0 if diff is None else 1)
    if need < 0:
        decode_workspace_bytes(cache, n, gqa, diff is not None)
    ws, nbytes, _keep = _workspace(cache, need, workspace)
    cache._call(fn, cache._address(), q.data_ptr(), q_row, q_head, gqa, *more, lens.data_ptr(), _window(window), tab, stride, blocks, n,
                scale if sm_scale is None else float(sm_scale), out.data_ptr(), None if lse is None else lse.data_ptr(), ws,
                nbytes)
    return (out, lse) if return_lse else out


def _prefill(cache, q, cu_rows, table, lens, causal, window, sm_scale, out, return_lse, lse, workspace, diff):
    if cu_rows is None:
        raise TypeError("cu_rows must be a torch.Tensor")
    tab, stride, blocks, n = _seqs(cache, table, lens, cu_rows, "lens")
    shape, gqa, q_row, q_head = _query(cache, q)
    if diff is None:
        fn, more, scale, maps = _lib.sphkv_cache16_prefill, (), cache._sm, ()
    else:
        fn, more, scale, maps = _lib.sphkv_cache16_diff_prefill, _diff_args(cache, diff[0], shape[1], *diff[1:]), math.sqrt(2.0) * cache._sm, (2,)
    out = _like(q, cache._dtype) if out is None else _out(out, shape, cache._dtype, "out", cache)
    if return_lse or lse is not None:
        lse = _out(lse, (shape[0], shape[1], *maps), _FLOAT, "lse", cache)
    ws, nbytes, _keep = _workspace(cache, prefill_workspace_bytes(cache, shape[0], n, gqa, diff is not None), workspace)
    cache._call(fn, cache._address(), q.data_ptr(), q_row, q_head, gqa, *more, shape[0], cu_rows.data_ptr(), lens.data_ptr(),
                1 if causal else 0, _window(window), tab, stride, blocks, n, scale if sm_scale is None else float(sm_scale),
                out.data_ptr(), None if lse is None else lse.data_ptr(), ws, nbytes)
    return (out, lse) if return_lse else out


def cache16_decode(cache: Cache16, q: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, window: int = 0,
                   sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None, return_lse: bool = False,
                   lse: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
    """Attention of one query token per sequence over the first lens[s] tokens of
    its pages, or the last `window` of them (sphkv_cache16_decode).  q [num_seqs,
    num_kv * gqa, dh] of the cache's type, gqa up to 64; lens int32 [num_seqs];
    window 0: no window; sm_scale 1 / sqrt(dh) unless given.  A softmax weight
    meets its value with 16 bits in bf16, with 22 in fp16 (to within 2^-33 of the
    row's largest weight, if it is small beside it).  Returns out (q's shape and
    type), with return_lse (out, lse): lse fp32 [num_seqs, num_kv * gqa] is the
    natural log of the softmax's sum.  A sequence without tokens gets zeros and
    -inf."""
    return _decode(cache, q, table, lens, window, sm_scale, out, return_lse, lse, workspace, None)


def cache16_diff_decode(cache: Cache16, q: torch.Tensor, lam: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                        norm_weight: Optional[torch.Tensor] = None, norm_eps: float = 1e-5, window: int = 0,
                        sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None, return_lse: bool = False,
                        lse: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
    """Differential attention of one query token per sequence
    (sphkv_cache16_diff_decode): the first dh / 2 elements of q and k make one
    softmax map, the last dh / 2 another, and the second, times lam[head], is
    taken from the first; values have dh elements.  lam fp32 [num_kv * gqa], gqa
    up to 32.  With norm_weight (fp32 [dh], any constant factor in it) a head's
    result x becomes x / sqrt(mean(x^2) + norm_eps) * norm_weight.  sm_scale
    1 / sqrt(dh / 2) unless given; lse [num_seqs, num_kv * gqa, 2], of both maps;
    the rest as cache16_decode."""
    return _decode(cache, q, table, lens, window, sm_scale, out, return_lse, lse, workspace, (lam, norm_weight, norm_eps))


def cache16_prefill(cache: Cache16, q: torch.Tensor, cu_rows: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                    causal: bool = True, window: int = 0, sm_scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False, lse: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None):
    """Attention of several query tokens per sequence, the last ones of its
    lens[s] tokens (sphkv_cache16_prefill): row cu_rows[s] + i of q [rows, num_kv
    * gqa, dh] is at position p = lens[s] - n_s + i and attends the tokens up to
    its own (causal; with a window those after p - window) or all lens[s].  Append
    the tokens first.  Rows that attend nothing get zeros and -inf; rows behind
    the last sequence are left as they were in out and lse.  Few tokens on a long
    context are slow beside many short sequences (the keys are split evenly over a
    batch): give them a call of their own.  The rest as cache16_decode."""
    return _prefill(cache, q, cu_rows, table, lens, causal, window, sm_scale, out, return_lse, lse, workspace, None)


def cache16_diff_prefill(cache: Cache16, q: torch.Tensor, lam: torch.Tensor, cu_rows: torch.Tensor, table: torch.Tensor,
                         lens: torch.Tensor, norm_weight: Optional[torch.Tensor] = None, norm_eps: float = 1e-5,
                         causal: bool = True, window: int = 0, sm_scale: Optional[float] = None,
                         out: Optional[torch.Tensor] = None, return_lse: bool = False,
                         lse: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
    """Differential attention of several query tokens per sequence
    (sphkv_cache16_diff_prefill): rows as cache16_prefill's, maps, lam and
    norm_weight as cache16_diff_decode's, lse [rows, num_kv * gqa, 2]."""
    return _prefill(cache, q, cu_rows, table, lens, causal, window, sm_scale, out, return_lse, lse, workspace,
                    (lam, norm_weight, norm_eps))
