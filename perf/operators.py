"""The operators of the 8-bit KV cache, as measurable cases.

The cache holds keys and values as int8 or e4m3 codes in pages of a sequence's
consecutive tokens, with one fp32 scale per (page, kv head) for the keys and
one for the values:

* ``write``    new K / V rows quantised into their sequences' pages, then what
               the touched pages hold read back: a token appended to each
               sequence, or whole prompts.
* ``read``     a batch's tokens back as K / V rows.
* ``decode``   attention of one query token per sequence over the cache.
* ``step``     a serving step: the new token written, then its attention.
* ``prefill``  causal attention of several query tokens per sequence, the last
               ones of their contexts (prompts, chunks, drafted tokens).

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
_LEAST = 2.0 ** -60      # scales lie in [2^-60, 2^60]


def _kv8():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import sphkv_kv8
    return sphkv_kv8


# ---- cases ------------------------------------------------------------------

def _case(name, kind, dh, num_kv, gqa, page, fmt, dtype, seqs, lo, hi, new_lo=1, new_hi=1):
    """lo..hi: tokens of a sequence, the new ones among them; new_lo..new_hi:
    its new (written or querying) tokens."""
    return {"name": name, "kind": kind, "dh": dh, "num_kv": num_kv, "gqa": gqa, "page": page, "fmt": fmt,
            "dtype": dtype, "seqs": seqs, "lo": lo, "hi": hi, "new_lo": new_lo, "new_hi": new_hi}


def listed():
    return [
        # one conversation appends its token: the smallest call
        _case("write_1x1", "write", 128, 8, 4, 16, "int8", "fp16", 1, 4091, 4091),
        # a full batch appends a token each
        _case("write_256x1", "write", 128, 8, 4, 32, "e4m3", "bf16", 256, 150, 2100),
        # the prompts of a batch, of uneven length
        _case("write_16x12k", "write", 128, 8, 4, 16, "int8", "fp16", 16, 500, 12000, 500, 12000),
        # a short context of a small model back in fp32
        _case("read_1x1k", "read", 64, 8, 4, 16, "e4m3", "fp32", 1, 1021, 1021, 1021, 1021),
        # a batch's contexts back as rows
        _case("read_16x12k", "read", 128, 8, 4, 64, "int8", "bf16", 16, 500, 12000, 500, 12000),
        # one short conversation on a small model: token in, attention out
        _case("step_1x4k", "step", 64, 8, 4, 16, "int8", "fp16", 1, 4096, 4096),
        # one long document on an 8B shape
        _case("decode_1x32k", "decode", 128, 8, 4, 16, "int8", "fp16", 1, 32768, 32768),
        # a chat server's batch: many short contexts of uneven length
        _case("decode_64x2k", "decode", 128, 8, 4, 32, "e4m3", "bf16", 64, 150, 2100),
        # a full batch with long contexts, the largest read of a cache
        _case("decode_64x32k", "decode", 128, 8, 8, 64, "e4m3", "bf16", 64, 2048, 32768),
        # a few drafted tokens on long documents: many keys, few rows
        _case("prefill_4x24_32k", "prefill", 128, 8, 4, 16, "int8", "fp16", 4, 20000, 32768, 5, 24),
        # chunks of a batch's prompts on what is cached of them, a small model
        _case("prefill_16x700_5k", "prefill", 64, 8, 4, 16, "e4m3", "bf16", 16, 750, 5000, 1, 700),
        # a whole prompt of 8K tokens, the most arithmetic
        _case("prefill_8k", "prefill", 128, 8, 4, 64, "int8", "bf16", 1, 8192, 8192, 8192, 8192),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "write", "read", "decode", "decode", "step", "prefill", "prefill"])
    dh, num_kv, gqa = rng.choice([64, 128, 128]), rng.choice([1, 4, 8, 8]), rng.choice([1, 2, 4, 4, 7, 8])
    page, fmt = rng.choice([16, 16, 32, 64, 128]), rng.choice(["int8", "e4m3"])
    dtype = rng.choice(["fp16", "bf16"] if kind in ("decode", "step", "prefill") else ["fp16", "bf16", "fp32"])
    if kind == "prefill":                         # padded scores stay under those of the 8K prompt
        seqs = _log_int(rng, 1, 32)
        most = 2 ** 31 // (seqs * num_kv * gqa)
        new = _log_int(rng, 2, min(8192, math.isqrt(most)))
        hi = _log_int(rng, new, min(65536, most // new))
        return {k: v for k, v in _case("", kind, dh, num_kv, gqa, page, fmt, dtype, seqs, rng.randint(max(1, hi // 2), hi),
                                       hi, rng.randint(1, new), new).items() if k != "name"}
    seqs = _log_int(rng, 1, 256 if kind != "read" else 16)
    hi = _log_int(rng, 20, min(131072, (1000000 if kind in ("decode", "step") else 100000) // seqs))
    lo = rng.randint(max(1, hi // 16), hi)
    whole = kind == "read" or (kind == "write" and rng.random() < 0.5)
    return {k: v for k, v in _case("", kind, dh, num_kv, gqa, page, fmt, dtype, seqs, lo, hi, lo if whole else 1,
                                   hi if whole else 1).items() if k != "name"}


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


def _rows(gen, n, num_kv, dh, channel, shift):
    """n rows of keys or values: channels of uneven size, as models have them."""
    return torch.randn((n, num_kv, dh), generator=gen, device=DEV) * channel + shift


def _channels(gen, num_kv, dh):
    c = torch.exp(0.5 * torch.randn((num_kv, dh), generator=gen, device=DEV))
    return c, 0.2 * torch.randn((num_kv, dh), generator=gen, device=DEV)


def _starts(lens):
    return torch.tensor([0] + lens, device=DEV, dtype=torch.int64).cumsum(0).to(torch.int32)


def prepare(c, seed):
    gen = _gen(seed)
    dh, num_kv, ps, n, dt = c["dh"], c["num_kv"], c["page"], c["seqs"], _TYPES[c["dtype"]]
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
    s["k_codes"] = torch.empty((num_pages, num_kv, ps, dh), dtype=torch.uint8, device=DEV)
    s["v_codes"] = torch.empty((num_pages, num_kv, ps // 16, dh, 16), dtype=torch.uint8, device=DEV)
    s["scales"] = torch.empty((num_pages, num_kv, 2), dtype=torch.float32, device=DEV)
    kch, ksh = _channels(gen, num_kv, dh)
    vch, vsh = _channels(gen, num_kv, dh)
    step = max(1, (1 << 26) // (num_kv * ps * dh))
    for a in range(0, num_pages, step):           # what the cache holds so far
        b = min(num_pages, a + step)
        for codes, i, ch, sh in ((s["k_codes"], 0, kch, ksh), (s["v_codes"], 1, vch, vsh)):
            x = _rows(gen, (b - a) * ps, num_kv, dh, ch, sh).view(b - a, ps, num_kv, dh).transpose(1, 2)
            sc = _scale(x.abs().amax((2, 3)), c["fmt"])
            s["scales"][a:b, :, i] = sc
            y = _quantised(x, sc[:, :, None, None], c["fmt"])
            codes[a:b] = y if i == 0 else y.reshape(b - a, num_kv, ps // 16, 16, dh).transpose(3, 4)
    T = sum(new)
    if c["kind"] in ("write", "step"):
        s["k"] = _rows(gen, T, num_kv, dh, kch, ksh).to(dt)
        s["v"] = _rows(gen, T, num_kv, dh, vch, vsh).to(dt)
    if c["kind"] == "write":                      # read back from the first slot of the first touched page
        back = [(a - b) % ps + b for a, b in zip(lens, new)]
        s["back_start"] = torch.tensor([a - b for a, b in zip(lens, back)], device=DEV, dtype=torch.int32)
        s["back_cu"], s["back_rows"] = _starts(back), sum(back)
    if c["kind"] in ("decode", "step", "prefill"):
        s["q"] = torch.randn((T, num_kv * c["gqa"], dh), generator=gen, device=DEV).to(dt)
    s["rows"], s["most"], s["one"] = T, max(new), c["new_hi"] == 1
    return s


# ---- the plain forms ----------------------------------------------------------

def _scale(amax, fmt):
    """fp32 scale of a block whose largest magnitude is amax."""
    if fmt == "int8":                             # a correctly rounded quotient
        return (amax.double() / 127.0).float().clamp(_LEAST, 1.0 / _LEAST)
    m, e = torch.frexp(amax)                      # amax = m 2^e, m in [1/2, 1): m 2^9 <= 448 for m <= 7/8
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), 0.0).clamp(_LEAST, 1.0 / _LEAST)


def _quantised(x, scale, fmt):
    """Codes (as bytes) of x over blocks of that scale: the nearest to the exact quotient."""
    if fmt == "int8":
        return (x.double() / scale.double()).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return (x.float() / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)


def _values(codes, fmt):
    return codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float()


def _places(s, start, cu, rows):
    """(page, slot) of each row of a ragged batch."""
    i = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(cu[1:].long(), i, right=True)
    pos = start.long()[seq] + i - cu.long()[seq]
    ps = s["case"]["page"]
    return s["table"][seq, pos // ps].long(), pos % ps


def _plain_write(s):
    c = s["case"]
    fmt, ps, dh, num_kv = c["fmt"], c["page"], c["dh"], c["num_kv"]
    page, slot = _places(s, s["start"], s["cu"], s["rows"])
    pages = s["scales"].shape[0]
    fresh = torch.zeros(pages, device=DEV).index_reduce_(0, page, (slot == 0).float(), "amax") > 0
    first = s["table"][torch.arange(c["seqs"], device=DEV), s["start"].long() // ps].long()
    for x, codes, i in ((s["k"], s["k_codes"], 0), (s["v"], s["v_codes"], 1)):
        x = x.float()
        top = torch.zeros((pages, num_kv), device=DEV).index_reduce_(0, page, x.abs().amax(2), "amax")
        old = s["scales"][:, :, i]
        scale = torch.where(fresh[:, None], _scale(top, fmt), torch.maximum(old, torch.where(top > 0, _scale(top, fmt), 0.0)))
        # earlier tokens of a sequence's first page, under the page's new scale
        wide = (...,) + (None,) * (codes.dim() - 2)
        was = codes[first]
        now = _quantised(_values(was, fmt).double() * old[first][wide].double(), scale[first][wide], fmt)
        grown = (scale > old)[first] & ~fresh[first][:, None]
        codes[first] = torch.where(grown[wide], now, was)
        y = _quantised(x, scale[page][:, :, None], fmt)
        if i == 0:
            codes[page, :, slot] = y
        else:
            codes[page, :, slot // 16, :, slot % 16] = y
        s["scales"][:, :, i] = scale


def _plain_read(s, start, cu, rows, dt):
    fmt = s["case"]["fmt"]
    page, slot = _places(s, start, cu, rows)
    k = _values(s["k_codes"][page, :, slot], fmt) * s["scales"][page][:, :, :1]
    v = _values(s["v_codes"][page, :, slot // 16, :, slot % 16], fmt) * s["scales"][page][:, :, 1:]
    return k.to(dt), v.to(dt)


def _plain_attention(s):
    """Queries padded to [sequences, heads, most, dh], keys to whole pages of the longest."""
    c = s["case"]
    n, num_kv, gqa, ps, dh, dt = c["seqs"], c["num_kv"], c["gqa"], c["page"], c["dh"], _TYPES[c["dtype"]]
    i = torch.arange(s["rows"], device=DEV)
    seq = torch.searchsorted(s["cu"][1:].long(), i, right=True)
    at = i - s["cu"].long()[seq]
    q = torch.zeros((n, s["most"], num_kv * gqa, dh), device=DEV)
    q[seq, at] = s["q"].float()
    table = s["table"].clamp(min=0).long()
    L = table.shape[1] * ps
    sc = s["scales"][table].transpose(1, 2)[..., None, None, :]                    # [n, H, blocks, 1, 1, 2]
    k = (_values(s["k_codes"][table], c["fmt"]).transpose(1, 2) * sc[..., 0]).reshape(n, num_kv, L, dh)
    q = q.view(n, s["most"], num_kv, gqa, dh).permute(0, 2, 3, 1, 4).reshape(n, num_kv, gqa * s["most"], dh)
    a = torch.matmul(q, k.transpose(2, 3)) * (dh ** -0.5)
    del k
    last = (s["lens"] - (s["cu"][1:] - s["cu"][:-1]))[:, None] + torch.arange(s["most"], device=DEV)[None, :]
    a = a.view(n, num_kv, gqa, s["most"], L)
    a = a.masked_fill_((torch.arange(L, device=DEV) > last[:, :, None])[:, None, None], float("-inf"))
    top = a.amax(-1, keepdim=True)
    a = a.sub_(top).exp_()
    total = a.sum(-1, keepdim=True)
    v = _values(s["v_codes"][table], c["fmt"]).transpose(4, 5).reshape(n, -1, num_kv, ps, dh)
    v = (v.transpose(1, 2) * sc[..., 1]).reshape(n, num_kv, L, dh)
    o = torch.matmul(a.view(n, num_kv, gqa * s["most"], L), v).view(n, num_kv, gqa, s["most"], dh) / total
    lse = (top + total.log()).squeeze(-1)
    out = o.permute(0, 3, 1, 2, 4).reshape(n, s["most"], num_kv * gqa, dh)[seq, at].to(dt)
    return out, lse.permute(0, 3, 1, 2).reshape(n, s["most"], num_kv * gqa)[seq, at]


def run(s):
    c = s["case"]
    kind, dt = c["kind"], _TYPES[c["dtype"]]
    if own:
        kv8 = _kv8()
        cache = kv8.Cache8(s["k_codes"], s["v_codes"], s["scales"], c["fmt"])
        cu = None if s["one"] else s["cu"]        # None: one token of each sequence
        if kind in ("write", "step"):
            kv8.cache8_write(cache, s["k"], s["v"], s["table"], s["start"], cu)
        if kind == "write":
            k, v = kv8.cache8_read(cache, s["table"], s["back_start"], s["back_cu"], s["back_rows"], dt)
            return {"k": k, "v": v, "scales": s["scales"]}
        if kind == "read":
            k, v = kv8.cache8_read(cache, s["table"], s["start"], s["cu"], s["rows"], dt)
            return {"k": k, "v": v}
        if kind == "prefill":
            out, lse = kv8.cache8_prefill(cache, s["q"], s["cu"], s["table"], s["lens"], return_lse=True)
        else:
            out, lse = kv8.cache8_decode(cache, s["q"], s["table"], s["lens"], return_lse=True)
        return {"out": out, "lse": lse, "scales": s["scales"]} if kind == "step" else {"out": out, "lse": lse}
    if kind in ("write", "step"):
        _plain_write(s)
    if kind == "write":
        k, v = _plain_read(s, s["back_start"], s["back_cu"], s["back_rows"], dt)
        return {"k": k, "v": v, "scales": s["scales"]}
    if kind == "read":
        k, v = _plain_read(s, s["start"], s["cu"], s["rows"], dt)
        return {"k": k, "v": v}
    out, lse = _plain_attention(s)
    return {"out": out, "lse": lse, "scales": s["scales"]} if kind == "step" else {"out": out, "lse": lse}


# ---- what a pass cannot do without --------------------------------------------

def work(c):
    lens, new = _lengths(c)
    H, dh, ps, gqa, eb = c["num_kv"], c["dh"], c["page"], c["gqa"], 4 if c["dtype"] == "fp32" else 2
    T = sum(new)
    pages = lambda ends, counts: sum((e - 1) // ps - (e - m) // ps + 1 for e, m in zip(ends, counts) if m)  # noqa: E731
    table = lambda ends, counts: 4 * pages(ends, counts) + 8 * len(ends)                                   # noqa: E731
    nbytes = flops = 0
    if c["kind"] in ("write", "step"):
        nbytes += 2 * T * H * dh * (eb + 1) + 8 * H * pages(lens, new) + table(lens, new)
        flops += 8 * T * H * dh
    if c["kind"] in ("write", "read"):
        m = [(a - b) % ps + b for a, b in zip(lens, new)] if c["kind"] == "write" else new
        nbytes += 2 * sum(m) * H * dh * (eb + 1) + 8 * H * pages(lens, m) + table(lens, m)
        flops += 2 * sum(m) * H * dh
    if c["kind"] in ("decode", "step", "prefill"):
        seen = sum(b * (a - b) + b * (b + 1) // 2 for a, b in zip(lens, new))
        nbytes += 2 * sum(lens) * H * dh + 8 * H * pages(lens, lens) + table(lens, lens)
        nbytes += T * H * gqa * (2 * dh * eb + 4)
        flops += 4 * seen * H * gqa * dh
    return {"bytes": nbytes, "flops": flops}


# ---- the definition in 64 bits --------------------------------------------------

def _decoded(codes, fmt):
    """The numbers that code bytes stand for, in 64 bits, by their bit fields."""
    b = torch.arange(256, dtype=torch.int64)
    if fmt == "int8":
        lut = torch.where(b < 128, b, b - 256).double()
    else:
        e, m = (b >> 3) & 15, (b & 7).double()
        lut = torch.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7).double(), m / 8 * 2.0 ** -6)
        lut = torch.where(b >= 128, -lut, lut)
    return lut.to(codes.device)[codes.long()]


def _rounded(y, fmt):
    """y (in units of the scale) to the nearest value that a code stands for."""
    if fmt == "int8":
        return torch.round(y).clamp(-127, 127)
    y = y.clamp(-448, 448)
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_scale(a, fmt):
    s = a / 127 if fmt == "int8" else 2.0 ** torch.ceil(torch.log2(a.clamp(min=1e-300) / 448))
    return s.clamp(_LEAST, 1 / _LEAST).float().double()      # a scale is an fp32 number


def exact(c, seed):
    s = prepare(c, seed)
    kind, fmt, ps, H, gqa, dh = c["kind"], c["fmt"], c["page"], c["num_kv"], c["gqa"], c["dh"]
    lens, new = _lengths(c)
    table = s["table"].cpu().long()
    cu, scales = [0], s["scales"].double()
    for m in new:
        cu.append(cu[-1] + m)

    def tokens(i, a, b, which):
        """Values of tokens a..b of sequence i: [tokens, heads, dh]."""
        if b <= a:
            return torch.zeros((0, H, dh), dtype=torch.float64, device=DEV)
        pages = table[i, a // ps:(b - 1) // ps + 1].to(DEV)
        if which == 0:
            x = _decoded(s["k_codes"][pages], fmt)
        else:
            x = _decoded(s["v_codes"][pages], fmt).transpose(3, 4).reshape(len(pages), H, ps, dh)
        x = (x * scales[pages, :, which, None, None]).transpose(1, 2).reshape(-1, H, dh)
        return x[a % ps:a % ps + b - a]

    written = {}
    if kind in ("write", "step"):
        for i, (end, m) in enumerate(zip(lens, new)):
            for which, x in ((0, s["k"]), (1, s["v"])):
                x = x[cu[i]:cu[i + 1]].double()
                begin = end - m
                base = begin - begin % ps
                before = tokens(i, base, begin, which)
                got = torch.cat([before, x])
                blocks = -(-got.shape[0] // ps)
                pad = torch.zeros((blocks * ps - got.shape[0], H, dh), dtype=torch.float64, device=DEV)
                got = torch.cat([got, pad]).view(blocks, ps, H, dh)
                fresh = got.clone()
                fresh[0, :begin % ps] = 0
                pages = table[i, base // ps:base // ps + blocks].to(DEV)
                sc = _exact_scale(fresh.abs().amax((1, 3)), fmt)
                if begin % ps:
                    sc[0] = torch.maximum(sc[0], scales[pages[0], :, which])
                scales[pages, :, which] = sc
                sc = sc[:, None, :, None]
                written[i, which] = (_rounded(got / sc, fmt) * sc).reshape(-1, H, dh)[:begin % ps + m]
    if kind == "write":
        k, v = (torch.cat([written[i, w] for i in range(c["seqs"])]) for w in (0, 1))
        return {"k": k, "v": v, "scales": scales}
    if kind == "read":
        k, v = (torch.cat([tokens(i, lens[i] - new[i], lens[i], w) for i in range(c["seqs"])]) for w in (0, 1))
        return {"k": k, "v": v}
    out = torch.zeros((s["rows"], H * gqa, dh), dtype=torch.float64, device=DEV)
    lse = torch.full((s["rows"], H * gqa), -math.inf, dtype=torch.float64, device=DEV)
    for i, (end, m) in enumerate(zip(lens, new)):
        begin = end - m
        if kind == "step":
            base = begin - begin % ps
            k, v = (torch.cat([tokens(i, 0, base, w), written[i, w]]) for w in (0, 1))
        else:
            k, v = tokens(i, 0, end, 0), tokens(i, 0, end, 1)
        q = s["q"][cu[i]:cu[i + 1]].double()
        for h in range(H * gqa):
            for a in range(0, m, 1024):
                b = min(m, a + 1024)
                seen = begin + b                  # the last row's context
                x = q[a:b, h] @ k[:seen, h // gqa].T / math.sqrt(dh)
                j = torch.arange(seen, device=DEV)
                x = torch.where(j[None, :] <= begin + torch.arange(a, b, device=DEV)[:, None], x, -math.inf)
                l = torch.logsumexp(x, 1)
                out[cu[i] + a:cu[i] + b, h] = torch.exp(x - l[:, None]) @ v[:seen, h // gqa]
                lse[cu[i] + a:cu[i] + b, h] = l
    return {"out": out, "lse": lse, "scales": scales} if kind == "step" else {"out": out, "lse": lse}
