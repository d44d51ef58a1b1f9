"""The 16-bit KV cache in numpy, 64 bits (include/sphkv.h, "16-bit KV cache"):
what the GPU tests hold the kernels to.  No reference counterpart."""
from __future__ import annotations

import numpy as np


def rotated(x, pos, inv_freq, interleaved=False, parts=1):
    """Rows [rows, heads, dh] at positions pos [rows], turned by pos * inv_freq radians per pair."""
    y = np.array(x, np.float64)
    n, width = len(inv_freq), x.shape[-1] // parts
    a = np.asarray(pos, np.float64)[:, None, None] * np.asarray(inv_freq, np.float64)
    c, s = np.cos(a), np.sin(a)
    for p in range(parts):
        j = p * width + (2 * np.arange(n) if interleaved else np.arange(n))
        k = j + 1 if interleaved else j + n
        y[..., j], y[..., k] = x[..., j] * c - x[..., k] * s, x[..., k] * c + x[..., j] * s
    return y


class Cache:
    """k, v [num_pages, num_kv, page_size, dh] float64."""

    def __init__(self, k, v):
        self.k, self.v = np.array(k, np.float64), np.array(v, np.float64)
        self.num_pages, self.num_kv, self.ps, self.dh = self.k.shape

    def page(self, table, s, blk):
        if not 0 <= blk < table.shape[1]:
            return -1
        p = int(table[s, blk])
        return p if 0 <= p < self.num_pages else -1

    def append(self, k, v, table, start, cu_rows=None, inv_freq=(), interleaved=False, parts=1, q=None):
        """Keeps the numbers unrounded; the rotated queries (None without q), rows of no sequence as they are."""
        n = len(start)
        cu = np.arange(n + 1) if cu_rows is None else cu_rows
        out = None if q is None else np.array(q, np.float64)
        for s in range(n):
            a, b = int(cu[s]), int(cu[s + 1])
            if b <= a:
                continue
            pos = int(start[s]) + np.arange(b - a)
            if q is not None:
                out[a:b] = rotated(q[a:b], pos, inv_freq, interleaved, parts)
            if start[s] < 0:
                continue
            turned = rotated(k[a:b], pos, inv_freq, interleaved, parts)
            for i, t in enumerate(pos):
                p = self.page(table, s, int(t) // self.ps)
                if p >= 0:
                    self.k[p, :, t % self.ps], self.v[p, :, t % self.ps] = turned[i], v[a + i]
        return out

    def tokens(self, table, s, L):
        """(k, v, present) of the first L positions: [L, num_kv, dh], absent ones zeros."""
        k, v, present = np.zeros((L, self.num_kv, self.dh)), np.zeros((L, self.num_kv, self.dh)), np.zeros(L, bool)
        for blk in range(-(-L // self.ps)):
            p = self.page(table, s, blk)
            if p >= 0:
                a, b = blk * self.ps, min(L, (blk + 1) * self.ps)
                k[a:b], v[a:b] = self.k[p, :, :b - a].swapaxes(0, 1), self.v[p, :, :b - a].swapaxes(0, 1)
                present[a:b] = True
        return k, v, present

    def attend(self, q, table, lens, cu_rows=None, causal=True, window=0, sm_scale=None, dims=None):
        """(out, lse, mass, reach, under), the last three for tolerances: of each output sum_t p_t |v_t| and max_t p_t
        sum_t |v_t|, of each row the largest sum_d |q_d k_d| sm_scale.  q [rows, num_q, dh] float64; dims: the
        slice of q's and k's elements that make the scores."""
        n, H = len(lens), self.num_kv
        dims = dims or slice(0, self.dh)
        cu = np.arange(n + 1) if cu_rows is None else cu_rows
        gqa = q.shape[1] // H
        sm = 1.0 / np.sqrt(dims.stop - dims.start) if sm_scale is None else sm_scale
        out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
        mass, reach, under = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape)
        for s in range(n):
            m = int(cu[s + 1]) - int(cu[s])
            L = min(max(int(lens[s]), 0), table.shape[1] * self.ps)
            if m <= 0 or L <= 0:
                continue
            k, v, present = self.tokens(table, s, L)
            at, j = L - m + np.arange(m)[:, None], np.arange(L)[None, :]
            see = present[None, :] & ((j <= at) & ((j > at - window) if window else True) if causal else True)
            see = np.broadcast_to(see, (m, L))
            clean = np.where(present[:, None, None], v, 0.0)
            for h in range(H):
                rows = q[cu[s]:cu[s + 1], h * gqa:(h + 1) * gqa, dims]                 # [m, gqa, d]
                kh = k[:, h, dims]
                x = np.where(see[:, None], (rows.reshape(m * gqa, -1) @ kh.T).reshape(m, gqa, L) * sm, -np.inf)
                r = (np.abs(rows).reshape(m * gqa, -1) @ np.abs(kh).T).reshape(m, gqa, L) * sm
                top = x.max(-1, keepdims=True)
                p = np.exp(x - np.where(np.isfinite(top), top, 0.0))
                l = p.sum(-1, keepdims=True)
                p = np.divide(p, l, out=np.zeros_like(p), where=l > 0).reshape(m * gqa, L)
                to = (slice(int(cu[s]), int(cu[s + 1])), slice(h * gqa, (h + 1) * gqa))
                out[to] = (p @ clean[:, h]).reshape(m, gqa, -1)
                mass[to] = (p @ np.abs(clean[:, h])).reshape(m, gqa, -1)
                under[to] = p.reshape(m, gqa, L).max(-1, keepdims=True) * (see @ np.abs(clean[:, h]))[:, None]
                with np.errstate(divide="ignore"):
                    lse[to] = (np.where(np.isfinite(top), top, 0.0) + np.log(l))[..., 0]
                reach[to] = np.where(see[:, None], r, 0).max(-1)
        return out, lse, mass, reach, under

    def maps(self, q, table, lens, **more):
        """attend() of the two maps of differential attention."""
        half = self.dh // 2
        return [self.attend(q, table, lens, dims=d, **more) for d in (slice(0, half), slice(half, self.dh))]


def difference(first, second, lam, norm_weight=None, eps=1e-5):
    """(out, x, scale) of the two maps' outputs [rows, heads, dh]: x the difference, out the normalised x."""
    x = first - np.asarray(lam, np.float64)[None, :, None] * second
    if norm_weight is None:
        return x, x, np.ones(x.shape[:2] + (1,))
    scale = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return x * scale * np.asarray(norm_weight, np.float64), x, scale
