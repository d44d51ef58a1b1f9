"""The 8-bit KV cache in numpy, 64 bits (include/sphkv.h, "8-bit KV cache"):
what the GPU tests hold the kernels to.  No reference counterpart."""
from __future__ import annotations

import numpy as np

LEAST, MOST = 2.0 ** -60, 2.0 ** 60

_B = np.arange(256)
_E, _M = (_B >> 3) & 15, _B & 7
_MAG = np.where(_E > 0, (1 + _M / 8) * 2.0 ** (_E - 7.0), _M / 8 * 2.0 ** -6)
_MAG[[0x7F, 0xFF]] = np.nan
# value of each code byte
VALUES = {"int8": np.arange(256).astype(np.uint8).view(np.int8).astype(np.float64),
          "e4m3": np.where(_B >= 128, -_MAG, _MAG)}


def scale_of(a: float, fmt: str) -> float:
    """fp32 scale of a block whose largest finite magnitude is a."""
    if fmt == "int8":
        s = float(np.float32(a / 127.0))
    else:
        s = 0.0 if a == 0 else 2.0 ** float(np.ceil(np.log2(a / 448.0)))
    return min(max(s, LEAST), MOST)


def code_values(y: np.ndarray, fmt: str) -> np.ndarray:
    """y (in units of the scale) to the nearest value a code stands for, half to even."""
    y = np.where(np.isnan(y), 0.0, y)
    if fmt == "int8":
        return np.clip(np.rint(np.clip(y, -128, 128)), -127, 127)
    y = np.clip(y, -448.0, 448.0)
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
    return np.rint(y / step) * step


def codes_of(values: np.ndarray, fmt: str) -> np.ndarray:
    """The code bytes of values that codes stand for (+0 for zeros)."""
    table = VALUES[fmt]
    order = np.argsort(np.where(np.isnan(table), np.inf, table), kind="stable")
    at = np.searchsorted(table[order][:np.isfinite(table).sum()], values)
    return order[at].astype(np.uint8)


class Cache:
    """values [num_pages, num_kv, page_size, dh] (in units of the scales) and
    scales [num_pages, num_kv, 2]."""

    def __init__(self, num_pages, num_kv, dh, page_size, fmt):
        self.num_pages, self.num_kv, self.dh, self.ps, self.fmt = num_pages, num_kv, dh, page_size, fmt
        self.k = np.zeros((num_pages, num_kv, page_size, dh))
        self.v = np.zeros((num_pages, num_kv, page_size, dh))
        self.scales = np.zeros((num_pages, num_kv, 2))

    @staticmethod
    def from_bytes(k_codes, v_codes, scales, fmt):
        """From the library's tensors as numpy arrays."""
        P, H, ps, dh = k_codes.shape
        c = Cache(P, H, dh, ps, fmt)
        c.k = VALUES[fmt][k_codes]
        c.v = VALUES[fmt][v_codes].transpose(0, 1, 2, 4, 3).reshape(P, H, ps, dh)
        c.scales = scales.astype(np.float64)
        return c

    def page(self, table, s, blk):
        if not 0 <= blk < table.shape[1]:
            return -1
        p = int(table[s, blk])
        return p if 0 <= p < self.num_pages else -1

    def write(self, k, v, table, start, cu_rows=None):
        """k, v [rows, num_kv, dh] float64."""
        n = len(start)
        cu = np.arange(n + 1) if cu_rows is None else cu_rows
        ps = self.ps
        for s in range(n):
            m, a = int(cu[s + 1]) - int(cu[s]), int(start[s])
            if m <= 0 or a < 0:
                continue
            for blk in range(a // ps, (a + m - 1) // ps + 1):
                p = self.page(table, s, blk)
                if p < 0:
                    continue
                o, e = max(a - blk * ps, 0), min(a + m - blk * ps, ps)
                rows = slice(int(cu[s]) + blk * ps + o - a, int(cu[s]) + blk * ps + e - a)
                for h in range(self.num_kv):
                    for i, (x, held) in enumerate(((k, self.k), (v, self.v))):
                        x = x[rows, h]
                        fin = np.abs(x[np.isfinite(x)])
                        new = scale_of(float(fin.max()) if fin.size else 0.0, self.fmt)
                        old = self.scales[p, h, i]
                        if o > 0 and not new > old:
                            new = old
                        if o > 0 and new > old:
                            held[p, h, :o] = code_values(held[p, h, :o] * old / new, self.fmt)
                        held[p, h, o:e] = code_values(x / new, self.fmt)
                        self.scales[p, h, i] = new

    def tokens(self, table, s, a, b):
        """(k, v, present) of positions a..b: [tokens, num_kv, dh], absent ones zeros."""
        k, v = np.zeros((b - a, self.num_kv, self.dh)), np.zeros((b - a, self.num_kv, self.dh))
        present = np.zeros(b - a, bool)
        for t in range(a, b):
            p = self.page(table, s, t // self.ps) if t >= 0 else -1
            if p < 0:
                continue
            sc = self.scales[p]
            k[t - a] = self.k[p, :, t % self.ps] * sc[:, :1]
            v[t - a] = self.v[p, :, t % self.ps] * sc[:, 1:]
            present[t - a] = True
        return k, v, present

    def attend(self, q, table, lens, cu_rows=None, causal=True, sm_scale=None):
        """(out, lse, mass, reach, under), the last three for tolerances: sum_t p_t |v_t| of each output, the
        largest sum_d |q_d k_d| sm_scale of each row, and of each output max_t (p_t sv_t) sum_t |value code of t|.
        q [rows, num_q, dh] float64."""
        n = len(lens)
        cu = np.arange(n + 1) if cu_rows is None else cu_rows
        H = self.num_kv
        gqa = q.shape[1] // H
        sm = 1.0 / np.sqrt(self.dh) if sm_scale is None else sm_scale
        out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
        mass, reach, under = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape)
        for s in range(n):
            m = int(cu[s + 1]) - int(cu[s])
            L = min(max(int(lens[s]), 0), table.shape[1] * self.ps)
            if m <= 0 or L <= 0:
                continue
            k, v, present = self.tokens(table, s, 0, L)
            pages = np.repeat([max(self.page(table, s, b), 0) for b in range(-(-L // self.ps))], self.ps)[:L]
            for h in range(H):
                rows = q[cu[s]:cu[s + 1], h * gqa:(h + 1) * gqa]                       # [m, gqa, dh]
                x = np.einsum("mgd,td->mgt", rows, k[:, h]) * sm
                r = np.einsum("mgd,td->mgt", np.abs(rows), np.abs(k[:, h])) * sm
                see = present[None, :] & (np.arange(L)[None, :] < (L - m + np.arange(m)[:, None] + 1 if causal else L))
                x = np.where(see[:, None], x, -np.inf)
                top = x.max(-1, keepdims=True)
                p = np.exp(x - np.where(np.isfinite(top), top, 0.0))
                l = p.sum(-1, keepdims=True)
                p = np.divide(p, l, out=np.zeros_like(p), where=l > 0)
                at = (slice(int(cu[s]), int(cu[s + 1])), slice(h * gqa, (h + 1) * gqa))
                out[at] = p @ v[:, h]
                mass[at] = p @ np.abs(v[:, h])
                sv = self.scales[pages, h, 1]
                codes = np.abs(v[:, h]) / np.where(sv > 0, sv, 1)[:, None]
                under[at] = (p * sv).max(-1, keepdims=True) * (see[:, None] @ codes)
                with np.errstate(divide="ignore"):
                    lse[at] = (np.where(np.isfinite(top), top, 0.0) + np.log(l))[..., 0]
                reach[at] = np.where(see[:, None], r, 0).max(-1)
        return out, lse, mass, reach, under
