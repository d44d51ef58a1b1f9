"""The operators of the 16-bit KV cache, as measurable cases.

The cache holds keys and values as fp16 or bf16 numbers in pages of a
sequence's consecutive tokens, one page for each kv head:

* ``append``        new tokens' keys rotated by their positions and their values
                    into their sequences' pages, their queries rotated.
* ``decode``        attention of one query token per sequence over the cache.
* ``step``          a serving step: the token appended, then its attention.
* ``prefill``       causal attention of several query tokens per sequence, the
                    last ones of their contexts (prompts, chunks, drafted tokens).
* ``diff_decode``, ``diff_prefill``
                    the same for differential attention: a head's first and
                    second half make a softmax map each, the second, times a
                    learned weight per head, is taken from the first, and the
                    result is normalised per head.

Inputs are drawn on the GPU from the seed alone.  Shapes are those of
sphkv_synth's configurations and the tests, and generic sizes around them.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda:0"
_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spherical-kv_amd")
_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_THETA = 500000.0
_EPS = 1e-5


def _kv16():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import sphkv_kv16
    return sphkv_kv16


# ---- cases ------------------------------------------------------------------

def _case(name, kind, dh, num_kv, gqa, page, dtype, seqs, lo, hi, new_lo=1, new_hi=1, rot=0, pairs="half", parts=1,
          window=0, layout="heads", rows="same"):
    """lo..hi: tokens of a sequence, the new ones among them; new_lo..new_hi:
    its new (appended or querying) tokens.  rot: rotated elements of each of
    `parts` parts of a head, in pairs half of them apart ("half") or next to each
    other ("next").  window: tokens that a row sees at most (0: all).  layout:
    pages of [heads, tokens] or of [tokens, heads].  rows: the type of k, v and q
    ("same": the cache's)."""
    return {"name": name, "kind": kind, "dh": dh, "num_kv": num_kv, "gqa": gqa, "page": page, "dtype": dtype, "seqs": seqs,
            "lo": lo, "hi": hi, "new_lo": new_lo, "new_hi": new_hi, "rot": rot, "pairs": pairs, "parts": parts,
            "window": window, "layout": layout, "rows": rows}


def listed():
    return [
        # one conversation appends its token: the smallest call
        _case("append_1x1", "append", 128, 8, 4, 16, "fp16", 1, 4091, 4091, rot=128),
        # a full batch appends a token each, half of each head rotated
        _case("append_256x1", "append", 128, 8, 4, 32, "bf16", 256, 150, 600, rot=64, pairs="next"),
        # the prompts of a batch, of uneven length
        _case("append_16x12k", "append", 128, 8, 4, 16, "fp16", 16, 500, 12000, 500, 12000, rot=128),
        # one short conversation on a small model: token in, attention out
        _case("step_1x4k", "step", 64, 8, 4, 16, "fp16", 1, 4096, 4096, rot=64),
        # one long document on an 8B shape
        _case("decode_1x32k", "decode", 128, 8, 4, 16, "fp16", 1, 32768, 32768),
        # a full batch with long contexts, the largest read of a cache
        _case("decode_64x32k", "decode", 128, 8, 8, 64, "bf16", 64, 2048, 32768),
        # one document on a model with differential attention
        _case("diff_decode_1x16k", "diff_decode", 128, 8, 4, 16, "fp16", 1, 16384, 16384),
        # a chat server's batch on such a model: many short contexts of uneven length
        _case("diff_decode_64x2k", "diff_decode", 128, 8, 4, 32, "bf16", 64, 150, 2100, layout="tokens"),
        # prompts on such a model
        _case("diff_prefill_4x2k", "diff_prefill", 128, 8, 4, 32, "bf16", 4, 1000, 2000, 1000, 2000),
        # a few drafted tokens on long documents: many keys, few rows
        _case("prefill_4x24_32k", "prefill", 128, 8, 4, 16, "fp16", 4, 20000, 32768, 5, 24),
        # chunks of a batch's prompts on what is cached of them, a small model with a sliding window
        _case("prefill_16x700_5k", "prefill", 64, 8, 4, 16, "bf16", 16, 750, 5000, 1, 700, window=2000),
        # a whole prompt of 8K tokens, the most arithmetic
        _case("prefill_8k", "prefill", 128, 8, 4, 64, "bf16", 1, 8192, 8192, 8192, 8192),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "step", "prefill", "prefill", "diff_decode", "diff_prefill"])
    dh, num_kv, gqa = rng.choice([64, 128, 128]), rng.choice([1, 4, 8, 8]), rng.choice([1, 2, 4, 4, 7, 8])
    page, dtype = rng.choice([16, 16, 32, 64, 128]), rng.choice(["fp16", "bf16"])
    layout = rng.choice(["heads", "heads", "tokens"])
    more = {"layout": layout}
    if kind in ("append", "step"):
        parts = rng.choice([1, 1, 2])
        more.update(parts=parts, rot=16 * rng.randint(1, dh // parts // 16), pairs=rng.choice(["half", "half", "next"]))
    if kind == "append":
        more.update(rows=rng.choice(["same", "same", "fp32"]))
    if kind in ("prefill", "diff_prefill"):       # padded scores stay under those that the 8K prompt has
        seqs = _log_int(rng, 1, 32)
        most = 2 ** (30 if kind == "prefill" else 29) // (seqs * num_kv * gqa)
        new = _log_int(rng, 2, min(8192, math.isqrt(most)))
        hi = _log_int(rng, new, min(65536, most // new))
        lo, new_lo, new_hi = rng.randint(max(1, hi // 2), hi), rng.randint(1, new), new
    else:
        seqs = _log_int(rng, 1, 256)
        most = 600000 // (gqa + 2) if kind == "append" else 1000000
        hi = _log_int(rng, 20, min(131072, most // seqs))
        lo = rng.randint(max(1, hi // 16), hi)
        new_lo, new_hi = (lo, hi) if kind == "append" and rng.random() < 0.5 else (1, 1)
    if kind != "append" and rng.random() < 0.25:
        more.update(window=_log_int(rng, 1, hi))
    c = _case("", kind, dh, num_kv, gqa, page, dtype, seqs, lo, hi, new_lo, new_hi, **more)
    return {k: v for k, v in c.items() if k != "name"}


def _spread(n, lo, hi):
    return [hi if n == 1 else lo + int((hi - lo) * ((i * 0.6180339887498949 + 0.5) % 1.0)) for i in range(n)]


def _lengths(c):
    """(tokens, new tokens) of every sequence: the case's own."""
    lens, new = _spread(c["seqs"], c["lo"], c["hi"]), _spread(c["seqs"], c["new_lo"], c["new_hi"])
    return lens, [min(a, b) for a, b in zip(lens, new)]


# ---- inputs, from the seed alone --------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _channels(gen, num_kv, dh):
    """Channels of uneven size and mean, as models have them."""
    c = torch.exp(0.5 * torch.randn((num_kv, dh), generator=gen, device=DEV))
    return c, 0.2 * torch.randn((num_kv, dh), generator=gen, device=DEV)


def _starts(lens):
    return torch.tensor([0] + lens, device=DEV, dtype=torch.int64).cumsum(0).to(torch.int32)


def _inv_freq(rot):
    """Radians per token of each pair."""
    return _THETA ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)


def prepare(c, seed):
    gen = _gen(seed)
    dh, num_kv, gqa, ps, n, dt = c["dh"], c["num_kv"], c["gqa"], c["page"], c["seqs"], _TYPES[c["dtype"]]
    lens, new = _lengths(c)
    blocks = [-(-x // ps) for x in lens]
    pages = sum(blocks)
    num_pages = pages + 3
    order = torch.randperm(num_pages, generator=gen, device=DEV)[:pages].to(torch.int32)
    width = max(blocks)
    at = torch.arange(width, device=DEV)[None, :] + _starts(blocks)[:-1, None]
    held = torch.arange(width, device=DEV)[None, :] < torch.tensor(blocks, device=DEV)[:, None]
    table = torch.where(held, order[at.clamp(max=pages - 1)], -1).to(torch.int32).contiguous()
    s = {"case": c, "table": table, "lens": torch.tensor(lens, device=DEV, dtype=torch.int32),
         "start": torch.tensor([a - b for a, b in zip(lens, new)], device=DEV, dtype=torch.int32), "cu": _starts(new)}
    shape = (num_pages, num_kv, ps, dh) if c["layout"] == "heads" else (num_pages, ps, num_kv, dh)
    spread = {"k": _channels(gen, num_kv, dh), "v": _channels(gen, num_kv, dh)}
    step = max(1, (1 << 26) // (num_kv * ps * dh))
    for name, (ch, sh) in spread.items():         # what the cache holds so far
        x = torch.empty(shape, dtype=dt, device=DEV)
        x = x if c["layout"] == "heads" else x.transpose(1, 2)
        for a in range(0, num_pages, step):
            b = min(num_pages, a + step)
            x[a:b] = torch.randn((b - a, num_kv, ps, dh), generator=gen, device=DEV) * ch[:, None] + sh[:, None]
        s["cache_" + name] = x
    T, H = sum(new), num_kv
    rows = dt if c["rows"] == "same" else _TYPES[c["rows"]]
    if c["kind"] in ("append", "step"):           # one projection's output: queries, keys, values of a token in a row
        qkv = torch.randn((T, H * (gqa + 2), dh), generator=gen, device=DEV)
        qkv[:, H * gqa:H * (gqa + 1)].mul_(spread["k"][0]).add_(spread["k"][1])
        qkv[:, H * (gqa + 1):].mul_(spread["v"][0]).add_(spread["v"][1])
        qkv = qkv.to(rows)
        s["q"], s["k"], s["v"] = qkv[:, :H * gqa], qkv[:, H * gqa:H * (gqa + 1)], qkv[:, H * (gqa + 1):]
        s["inv_freq"] = _inv_freq(c["rot"])
    else:
        s["q"] = torch.randn((T, H * gqa, dh), generator=gen, device=DEV).to(dt)
    if c["kind"].startswith("diff"):
        s["lam"] = 0.2 + 0.6 * torch.rand(H * gqa, generator=gen, device=DEV)
        s["weight"] = 0.5 + 0.05 * torch.randn(dh, generator=gen, device=DEV)
    s["rows"], s["most"], s["one"] = T, max(new), c["new_hi"] == 1
    if own:                                       # the handle over the tensors, which a program keeps
        s["cache"] = _kv16().Cache16(s["cache_k"], s["cache_v"])
    return s


# ---- the plain forms ----------------------------------------------------------

def _places(s):
    """(sequence, position) of each row of a ragged batch."""
    i = torch.arange(s["rows"], device=DEV)
    seq = torch.searchsorted(s["cu"][1:].long(), i, right=True)
    return seq, s["start"].long()[seq] + i - s["cu"].long()[seq]


def _plain_rotate(x, pos, s):
    """x [rows, heads, dh] of any type, rotated, in fp32."""
    c = s["case"]
    R, rows, heads = c["rot"], x.shape[0], x.shape[1]
    angle = pos.double()[:, None] * s["inv_freq"][None, :]
    cos, sin = torch.cos(angle).float()[:, None, None, :], torch.sin(angle).float()[:, None, None, :]
    y = x.float().reshape(rows, heads, c["parts"], -1).clone()
    if c["pairs"] == "half":
        a, b = y[..., :R // 2].clone(), y[..., R // 2:R].clone()
        y[..., :R // 2], y[..., R // 2:R] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = y[..., 0:R:2].clone(), y[..., 1:R:2].clone()
        y[..., 0:R:2], y[..., 1:R:2] = a * cos - b * sin, b * cos + a * sin
    return y.reshape(rows, heads, -1)


def _plain_append(s):
    """Fills the cache; the rotated queries."""
    c = s["case"]
    dt = _TYPES[c["dtype"]]
    seq, pos = _places(s)
    page, slot = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    s["cache_k"][page, :, slot] = _plain_rotate(s["k"], pos, s).to(dt)
    s["cache_v"][page, :, slot] = s["v"].float().to(dt)
    return _plain_rotate(s["q"], pos, s).to(dt)


def _plain_map(q, k, scale, hidden):
    """(unnormalised weights, their sums, lse) of queries [n, heads, rows, d] over keys [n, heads, tokens, d]."""
    a = torch.matmul(q, k.transpose(2, 3)) * scale
    a = a.view(hidden.shape[0], a.shape[1], -1, *hidden.shape[1:]).masked_fill_(hidden[:, None, None], float("-inf"))
    top = a.amax(-1, keepdim=True)
    a = a.sub_(top).exp_()
    total = a.sum(-1, keepdim=True)
    return a, total, (top + total.log()).squeeze(-1)


def _plain_attention(s, q_rows):
    """Queries padded to [sequences, heads, most, dh], keys to whole pages of the longest."""
    c = s["case"]
    n, H, gqa, ps, dh, m = c["seqs"], c["num_kv"], c["gqa"], c["page"], c["dh"], s["most"]
    seq, _ = _places(s)
    at = torch.arange(s["rows"], device=DEV) - s["cu"].long()[seq]
    q = torch.zeros((n, m, H * gqa, dh), device=DEV)
    q[seq, at] = q_rows.float()
    q = q.view(n, m, H, gqa, dh).permute(0, 2, 3, 1, 4).reshape(n, H, gqa * m, dh)
    table = s["table"].clamp(min=0).long()
    L = table.shape[1] * ps
    k = s["cache_k"][table].transpose(1, 2).float().reshape(n, H, L, dh)
    last = (s["lens"] - (s["cu"][1:] - s["cu"][:-1]))[:, None] + torch.arange(m, device=DEV)[None, :]
    t = torch.arange(L, device=DEV)
    hidden = t > last[:, :, None]
    if c["window"]:
        hidden |= t <= last[:, :, None] - c["window"]
    rows = lambda x: x.permute(0, 3, 1, 2, *range(4, x.dim())).reshape(n, m, H * gqa, -1)[seq, at]  # noqa: E731
    if not c["kind"].startswith("diff"):
        a, total, lse = _plain_map(q, k, dh ** -0.5, hidden)
        del k
        v = s["cache_v"][table].transpose(1, 2).float().reshape(n, H, L, dh)
        o = torch.matmul(a.view(n, H, gqa * m, L), v).view(n, H, gqa, m, dh) / total
        return rows(o).to(_TYPES[c["dtype"]]), rows(lse[..., None])[..., 0]
    half, scale = dh // 2, (dh // 2) ** -0.5
    v = s["cache_v"][table].transpose(1, 2).float().reshape(n, H, L, dh)
    o, lse = None, []
    for i, (part, factor) in enumerate(((slice(0, half), 1.0), (slice(half, dh), -s["lam"].view(1, H, gqa, 1, 1)))):
        a, total, e = _plain_map(q[..., part].contiguous(), k[..., part].contiguous(), scale, hidden)
        x = factor * (torch.matmul(a.view(n, H, gqa * m, L), v).view(n, H, gqa, m, dh) / total)
        o = x if o is None else o + x
        lse.append(e)
    o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + _EPS) * s["weight"]
    return rows(o).to(_TYPES[c["dtype"]]), rows(torch.stack(lse, -1))


def run(s):
    c = s["case"]
    kind = c["kind"]
    q = s["q"]
    if own:
        kv16, cache = _kv16(), s["cache"]
        cu = None if s["one"] else s["cu"]        # None: one token of each sequence
        if kind in ("append", "step"):
            q = kv16.cache16_append(cache, s["k"], s["v"], s["table"], s["start"], cu, inv_freq=s["inv_freq"],
                                     interleaved=c["pairs"] == "next", parts=c["parts"], q=q)
        if kind in ("decode", "step"):
            out, lse = kv16.cache16_decode(cache, q, s["table"], s["lens"], window=c["window"], return_lse=True)
        elif kind == "prefill":
            out, lse = kv16.cache16_prefill(cache, q, s["cu"], s["table"], s["lens"], window=c["window"], return_lse=True)
        elif kind == "diff_decode":
            out, lse = kv16.cache16_diff_decode(cache, q, s["lam"], s["table"], s["lens"], norm_weight=s["weight"],
                                                norm_eps=_EPS, window=c["window"], return_lse=True)
        elif kind == "diff_prefill":
            out, lse = kv16.cache16_diff_prefill(cache, q, s["lam"], s["cu"], s["table"], s["lens"], norm_weight=s["weight"],
                                                 norm_eps=_EPS, window=c["window"], return_lse=True)
    else:
        if kind in ("append", "step"):
            q = _plain_append(s)
        if kind != "append":
            out, lse = _plain_attention(s, q)
    if kind == "append":
        return {"q": q, "k": s["cache_k"], "v": s["cache_v"]}
    if kind == "step":
        return {"out": out, "lse": lse, "k": s["cache_k"], "v": s["cache_v"]}
    return {"out": out, "lse": lse}


# ---- what a pass cannot do without --------------------------------------------

def work(c):
    lens, new = _lengths(c)
    H, dh, ps, gqa, w = c["num_kv"], c["dh"], c["page"], c["gqa"], c["window"]
    T = sum(new)
    nbytes = flops = 0
    if c["kind"] in ("append", "step"):           # k, v and q in and out, page ids, starts
        eb = 4 if c["rows"] == "fp32" else 2
        nbytes += T * H * (gqa + 2) * dh * (eb + 2) + 8 * len(lens)
        nbytes += 4 * sum((a - 1) // ps - (a - m) // ps + 1 for a, m in zip(lens, new))
        flops += 3 * T * H * (gqa + 1) * c["rot"] * c["parts"]
    if c["kind"] != "append":
        diff = c["kind"].startswith("diff")
        seen = reach = 0                          # (row, token) pairs, tokens that a row sees
        for a, m in zip(lens, new):
            if w == 0 or w >= a:
                seen += m * (a - m) + m * (m + 1) // 2
                reach += a
            else:
                grown = max(0, min(a - m + m, w) - (a - m))          # rows that see all before them
                seen += grown * (a - m) + grown * (grown + 1) // 2 + (m - grown) * w
                reach += min(a, w + m - 1)
        nbytes += 2 * reach * H * dh * 2 + 4 * sum(-(-min(a, w + m if w else a) // ps) for a, m in zip(lens, new)) + 8 * len(lens)
        nbytes += T * H * gqa * (2 * dh * 2 + (8 if diff else 4))
        flops += (6 if diff else 4) * seen * H * gqa * dh
    return {"bytes": nbytes, "flops": flops}


# ---- the definition in 64 bits --------------------------------------------------

def _exact_rotate(x, pos, c):
    """Rows of one sequence, [tokens, heads, dh] at positions pos, as complex numbers turned by their angles."""
    R, width = c["rot"], c["dh"] // c["parts"]
    f = _THETA ** (-2.0 * torch.arange(R // 2, dtype=torch.float64, device=DEV) / R)
    turn = torch.polar(torch.ones(len(pos), R // 2, dtype=torch.float64, device=DEV), pos.double()[:, None] * f)[:, None]
    y = x.double().clone()
    for p in range(c["parts"]):
        j = torch.arange(R // 2, device=DEV)
        a, b = (j, j + R // 2) if c["pairs"] == "half" else (2 * j, 2 * j + 1)
        a, b = a + p * width, b + p * width
        z = torch.complex(y[..., a], y[..., b]) * turn
        y[..., a], y[..., b] = z.real, z.imag
    return y


def exact(c, seed):
    s = prepare(c, seed)
    kind, ps, H, gqa, dh, w = c["kind"], c["page"], c["num_kv"], c["gqa"], c["dh"], c["window"]
    lens, new = _lengths(c)
    table = s["table"].cpu().long()
    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    K, V = s["cache_k"], s["cache_v"]
    q = s["q"].double()
    if kind in ("append", "step"):
        K, V = K.double(), V.double()
        for i, (end, m) in enumerate(zip(lens, new)):
            rows, pos = slice(cu[i], cu[i + 1]), torch.arange(end - m, end, device=DEV)
            page, slot = table[i].to(DEV)[pos // ps], pos % ps
            K[page, :, slot] = _exact_rotate(s["k"][rows], pos, c)
            V[page, :, slot] = s["v"][rows].double()
            q[rows] = _exact_rotate(s["q"][rows], pos, c)
        if kind == "append":
            return {"q": q, "k": K, "v": V}
        # a step attends to numbers of the cache's type
        q, keys, values = (x.to(_TYPES[c["dtype"]]).double() for x in (q, K, V))
    else:
        keys, values = K, V

    def tokens(i, x):
        """The tokens of sequence i: [tokens, heads, dh]."""
        pages = table[i, :-(-lens[i] // ps)].to(DEV)
        return x[pages].transpose(1, 2).reshape(-1, H, dh)[:lens[i]].double()

    diff = kind.startswith("diff")
    out = torch.zeros((s["rows"], H * gqa, dh), dtype=torch.float64, device=DEV)
    lse = torch.zeros((s["rows"], H * gqa, 2), dtype=torch.float64, device=DEV)
    maps = [(0, dh // 2, 1.0), (dh // 2, dh, -1.0)] if diff else [(0, dh, 1.0)]
    for i, (end, m) in enumerate(zip(lens, new)):
        k, v = tokens(i, keys), tokens(i, values)
        for h in range(H * gqa):
            for a in range(0, m, 1024):
                b = min(m, a + 1024)
                at = end - m + torch.arange(a, b, device=DEV)[:, None]
                first = max(0, end - m + a + 1 - w) if w else 0
                j = torch.arange(first, end - m + b, device=DEV)[None, :]
                sees = (j <= at) & (j > at - w) if w else j <= at
                for e, (lo, hi, sign) in enumerate(maps):
                    x = q[cu[i] + a:cu[i] + b, h, lo:hi] @ k[first:end - m + b, h // gqa, lo:hi].T / math.sqrt(hi - lo)
                    x = torch.where(sees, x, -math.inf)
                    l = torch.logsumexp(x, 1)
                    o = torch.exp(x - l[:, None]) @ v[first:end - m + b, h // gqa]
                    out[cu[i] + a:cu[i] + b, h] += o if sign > 0 else -s["lam"][h].double() * o
                    lse[cu[i] + a:cu[i] + b, h, e] = l
    if diff:
        out = out / torch.sqrt((out * out).mean(-1, keepdim=True) + _EPS) * s["weight"].double()
        return {"out": out, "lse": lse}
    if kind == "step":
        return {"out": out, "lse": lse[..., 0], "k": K, "v": V}
    return {"out": out, "lse": lse[..., 0]}
