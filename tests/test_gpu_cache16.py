"""The 16-bit KV cache on the GPU against its oracle in 64 bits: appended
numbers, attention and differential attention within derived bounds."""
import math

import numpy as np
import pytest
import torch

import sphkv_kv16 as kv16
import sphkv_lib
from gpu_helpers import log
from oracle import cache16 as o16

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
THETA = 500000.0


def i32(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=dev)


def f64(t):
    return t.detach().double().cpu().numpy()


def random_cache(dev, seed, num_pages, num_kv, dh, ps, dtype, layout="heads"):
    """A cache of normal numbers, channels of uneven size."""
    g = torch.Generator(device=dev).manual_seed(seed)
    shape = (num_pages, ps, num_kv, dh) if layout == "tokens" else (num_pages, num_kv, ps, dh)
    scale = torch.exp(0.4 * torch.randn((dh,), generator=g, device=dev))
    k, v = ((torch.randn(shape, generator=g, device=dev) * scale).to(TYPES[dtype]) for _ in range(2))
    if layout == "tokens":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    elif layout == "joined":                    # keys and values of a page behind each other
        kv = torch.stack([k, v], 1)
        k, v = kv[:, 0], kv[:, 1]
    return kv16.Cache16(k, v)


def oracle_of(cache):
    return o16.Cache(f64(cache.k), f64(cache.v))


def tables(seed, num_pages, blocks, width=None):
    """Page tables of sequences with that many blocks: distinct pages in random order, -1 behind."""
    order = np.random.default_rng(seed).permutation(num_pages)
    t = np.full((len(blocks), width or max(max(blocks), 1)), -1, np.int32)
    a = 0
    for s, n in enumerate(blocks):
        t[s, :n] = order[a:a + n]
        a += n
    assert a <= num_pages
    return t


def rounded_bound(want, reach, dtype):
    """Of a rotated number: the turns are reduced in 64 bits and rounded to fp32 (2^-26 of a turn, 2^-23 radians), sine and
    cosine are within 2^-22 of theirs, products and sum add 2^-23 of |x| + |x'| (`reach`); then one rounding to `dtype`."""
    return 2.0 ** -20.5 * reach + torch.finfo(dtype).eps / 2 * np.abs(want) * (1 + 2.0 ** -10) + (2.0 ** -25 if dtype is torch.float16 else 0)


def partner_sum(x, freqs, interleaved, parts):
    """|x| + |x'| of each element that turns, 0 of the others."""
    y, a, width = np.zeros_like(x), np.abs(x), x.shape[-1] // parts
    for p in range(parts):
        j = p * width + (2 * np.arange(freqs) if interleaved else np.arange(freqs))
        k = j + 1 if interleaved else j + freqs
        y[..., j] = y[..., k] = a[..., j] + a[..., k]
    return y


# ---- append --------------------------------------------------------------------

APPENDS = [
    # (in, cache, dh, page, num_kv, gqa, freqs, interleaved, parts, layout, [(start, new)])
    ("fp16", "fp16", 128, 16, 8, 4, 64, False, 1, "heads", [(0, 1), (15, 1), (5, 3), (16, 16), (0, 0), (7, 60)]),
    ("bf16", "bf16", 64, 16, 3, 1, 32, True, 1, "tokens", [(0, 33), (31, 2), (16, 0), (3, 13), (0, 16)]),
    ("fp32", "fp16", 64, 32, 1, 7, 16, False, 2, "joined", [(33, 64), (0, 31), (31, 1), (32, 32), (1, 7)]),
    ("fp32", "bf16", 128, 64, 2, 2, 16, True, 2, "heads", [(63, 2), (0, 64), (10, 130), (64, 1)]),
    ("bf16", "fp16", 128, 128, 4, 0, 8, False, 1, "tokens", [(0, 200), (127, 1), (100, 28), (17, 16)]),
    ("fp16", "bf16", 128, 32, 8, 8, 32, False, 2, "heads", [(0, 0), (40, 9), (0, 0)]),
    ("fp16", "fp16", 64, 64, 5, 3, 24, True, 1, "heads", [(i, 1) for i in range(0, 140, 7)]),
    ("bf16", "bf16", 128, 16, 2, 16, 64, False, 1, "heads", [(3, 1)] + [(0, 5)] * 70),         # more than 64 sequences
    ("fp16", "fp16", 64, 16, 1, 2, 0, False, 1, "heads", [(i % 23, i % 4) for i in range(5000)]),   # more than 64 * 64, no rotation
]


@pytest.mark.parametrize("dtype, ctype, dh, ps, num_kv, gqa, freqs, inter, parts, layout, seqs", APPENDS)
def test_append(gpu, dtype, ctype, dh, ps, num_kv, gqa, freqs, inter, parts, layout, seqs):
    rng = np.random.default_rng(3)
    blocks = [-(-(a + m) // ps) for a, m in seqs]
    num_pages = sum(blocks) + 2
    cache = random_cache(gpu, 4, num_pages, num_kv, dh, ps, ctype, layout)
    want, before = oracle_of(cache), oracle_of(cache)
    table = tables(5, num_pages, blocks)
    cu = np.cumsum([0] + [m for _, m in seqs])
    T = int(cu[-1])
    x = torch.from_numpy(rng.standard_normal((T + 3, num_kv * (gqa + 2), dh))).to(gpu).to(TYPES[dtype])
    x[T:] = float("nan")                                                 # rows behind the last sequence
    q, k, v = x[:, :num_kv * gqa], x[:, num_kv * gqa:num_kv * (gqa + 1)], x[:, num_kv * (gqa + 1):]
    f = kv16.rope_inv_freq(2 * freqs, THETA, gpu) if freqs else None
    log(f"append {dtype} into {ctype} dh {dh} page {ps}")
    q_out = torch.full((T + 3, num_kv * gqa, dh), 7.0, dtype=TYPES[ctype], device=gpu)
    start = [a for a, _ in seqs]
    got = kv16.cache16_append(cache, k, v, i32(table, gpu), i32(start, gpu), i32(cu, gpu), inv_freq=f, interleaved=inter,
                              parts=parts, q=q if gqa else None, q_out=q_out if gqa else None)
    assert got is (q_out if gqa else None)
    kk, vv, qq = f64(k), f64(v), f64(q)
    freq = f64(f) if freqs else np.zeros(0)
    rq = want.append(kk, vv, table, start, cu, freq, inter, parts, qq)
    reach = oracle_of(cache)
    reach.k[:], reach.v[:] = 0, 0
    reach.append(partner_sum(kk, freqs, inter, parts), 0 * vv, table, start, cu)
    have = oracle_of(cache)
    ct = TYPES[ctype]
    for name, near in (("k", reach.k), ("v", 0 * reach.v)):
        a, b, old = getattr(have, name), getattr(want, name), getattr(before, name)
        tol = rounded_bound(b, near, ct)
        assert (np.abs(a - b) <= tol).all(), f"{name}: {(np.abs(a - b) > tol).sum()} off"
        same = b == old
        assert np.array_equal(a[same], old[same]), f"{name}: numbers that no token has changed"
    if dtype == ctype:
        assert np.array_equal(have.v, want.v)
    if gqa:
        a, b = f64(q_out)[:T], rq[:T]
        assert (np.abs(a - b) <= rounded_bound(b, partner_sum(qq[:T], freqs, inter, parts), ct)).all()
        assert (q_out[T:] == 7.0).all()


@pytest.mark.parametrize("ftype", [torch.float32, torch.float64])
def test_append_far_positions(gpu, ftype):
    """Angles of positions up to 2^20 are those of 64 bits, by the frequencies as they are given."""
    dh, H, ps = 128, 2, 128
    pos = [2 ** 20 - 1, 999_999, 131_071, 2 ** 19 + 3]
    cache = random_cache(gpu, 1, 4, H, dh, ps, "fp16")
    want = oracle_of(cache)
    blocks = 2 ** 20 // ps
    table = np.full((4, blocks), -1, np.int32)
    for s, p in enumerate(pos):
        table[s, p // ps] = s
    g = torch.Generator(device=gpu).manual_seed(2)
    k, v, q = (torch.randn((4, h, dh), generator=g, device=gpu) for h in (H, H, 3 * H))
    f = kv16.rope_inv_freq(dh, 10000.0, gpu).to(ftype)
    got = kv16.cache16_append(cache, k, v, i32(table, gpu), i32(pos, gpu), inv_freq=f, q=q)
    rq = want.append(f64(k), f64(v), table, pos, None, f64(f), q=f64(q))
    have = oracle_of(cache)
    top = 2.0 ** -20.5 * 16 + 2.0 ** -11 * np.abs(want.k) * 1.001 + 2.0 ** -25
    assert (np.abs(have.k - want.k) <= top).all()
    assert (np.abs(f64(got) - rq) <= rounded_bound(rq, partner_sum(f64(q), dh // 2, False, 1), torch.float16)).all()


def test_append_keeps_bits_and_special_values(gpu):
    """Values and elements that do not turn are copied bit for bit, infinities and NaN among them; one in a pair that turns
    stays in its pair."""
    dh, H, ps = 64, 2, 16
    cache = kv16.Cache16.allocate(2, H, dh, ps, torch.bfloat16, gpu)
    k = torch.randn((1, H, dh), device=gpu).bfloat16()
    v = torch.randn((1, H, dh), device=gpu).bfloat16()
    v[0, 0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), -0.0])
    k[0, 1, 50], k[0, 1, 3] = float("inf"), float("nan")
    f = kv16.rope_inv_freq(32, device=gpu)
    kv16.cache16_append(cache, k, v, i32([[1]], gpu), i32([5], gpu), inv_freq=f)
    assert torch.equal(cache.v[1, :, 5].view(torch.int16), v[0].view(torch.int16))
    assert torch.equal(cache.k[1, :, 5, 32:].view(torch.int16), k[0, :, 32:].view(torch.int16))
    nan = cache.k[1, 1, 5].isnan()
    assert nan[3] and nan[19] and nan.sum() == 2


def test_append_drops_what_has_no_page(gpu):
    """Past the table, a negative start, a page outside the cache: nothing is written, queries are rotated all the same."""
    dh, H, ps = 64, 1, 16
    cache = random_cache(gpu, 3, 6, H, dh, ps, "fp16")
    before = [cache.k.clone(), cache.v.clone()]
    table = np.array([[0, 1], [2, 99], [-5, 3], [4, 5]], np.int32)
    start, new = [30, 14, 0, -3], [5, 4, 20, 6]
    cu = np.cumsum([0] + new)
    g = torch.Generator(device=gpu).manual_seed(2)
    k, v, q = (torch.randn((cu[-1], h, dh), generator=g, device=gpu).half() for h in (H, H, 2 * H))
    want = oracle_of(cache)
    f = kv16.rope_inv_freq(dh, device=gpu)
    got = kv16.cache16_append(cache, k, v, i32(table, gpu), i32(start, gpu), i32(cu, gpu), inv_freq=f, q=q)
    rq = want.append(f64(k), f64(v), table, start, cu, f64(f), q=f64(q))
    have = oracle_of(cache)
    assert (np.abs(have.k - want.k) <= 2.0 ** -20.5 * 16 + 2.0 ** -11 * np.abs(want.k) * 1.001 + 2.0 ** -25).all()
    assert np.array_equal(have.v, want.v)
    for p in (4, 5):                                                     # of the negative start
        assert torch.equal(cache.k[p], before[0][p]) and torch.equal(cache.v[p], before[1][p])
    assert (np.abs(f64(got) - rq) <= rounded_bound(rq, partner_sum(f64(q), dh // 2, False, 1), torch.float16)).all()


def test_append_strides_alignment_and_queries_in_place(gpu):
    dh, H, gqa, ps, T = 128, 2, 3, 16, 21
    raw = torch.randn(T * 1600 + 1, device=gpu).half()
    x = raw[1:].view(T, 1600)                                            # rows 2 bytes off any vector
    q = x[:, :gqa * H * 132].unflatten(1, (gqa * H, 132))[..., :dh]
    k = x[:, 800:800 + 2 * dh].unflatten(1, (2, dh))
    v = x[:, 1100:1100 + 2 * 130].unflatten(1, (2, 130))[..., :dh]
    cache = random_cache(gpu, 3, 4, H, dh, ps, "fp16", "tokens")
    want = oracle_of(cache)
    f = kv16.rope_inv_freq(64, device=gpu)
    args = dict(inv_freq=f, parts=2)
    rq = want.append(f64(k), f64(v), np.array([[2, 0]], np.int32), [3], [0, T], f64(f), parts=2, q=f64(q))
    bound = rounded_bound(rq, partner_sum(f64(q), 32, False, 2), torch.float16)
    copy = q.clone()
    table, start, cu = i32([[2, 0]], gpu), i32([3], gpu), i32([0, T], gpu)
    one = kv16.cache16_append(cache, k.clone(), v.clone(), table, start, cu, q=copy, **args)
    first = [cache.k.clone(), cache.v.clone()]
    cache.k.zero_(), cache.v.zero_()
    two = kv16.cache16_append(cache, k, v, table, start, cu, q=q, q_out=q, **args)
    assert two is q and torch.equal(one, q)
    assert (np.abs(f64(q) - rq) <= bound).all()
    for s in range(T):
        p, i = [2, 0][(3 + s) // ps], (3 + s) % ps
        assert torch.equal(first[0][p, :, i], cache.k[p, :, i]) and torch.equal(first[1][p, :, i], cache.v[p, :, i])


def test_memory_that_tensors_share(gpu):
    """Keys and values, queries and outputs beside each other in one buffer are appended as into buffers of their own; over
    each other they are refused, and attention reads such a cache."""
    P, H, ps, dh, T = 4, 3, 16, 64, 40
    g = torch.Generator(device=gpu).manual_seed(3)
    k, v, q = (torch.randn((T, h, dh), generator=g, device=gpu).half() for h in (H, H, 2 * H))
    args = (i32([[2, 0, 3]], gpu), i32([5], gpu), i32([0, T], gpu))
    f = kv16.rope_inv_freq(dh, device=gpu)
    own = kv16.Cache16.allocate(P, H, dh, ps, device=gpu)
    ref = kv16.cache16_append(own, k, v, *args, inv_freq=f, q=q)
    pair = torch.zeros((P, ps, H, 2, dh), dtype=torch.float16, device=gpu).transpose(1, 2)           # a token's keys, then its values
    mixed = torch.zeros((P, 2, H * ps * dh), dtype=torch.float16, device=gpu)                         # heads first, tokens first
    both = torch.empty((T, 2, 2 * H, dh), dtype=torch.float16, device=gpu)
    both[:, 0] = q
    for cache in (kv16.Cache16(pair[..., 0, :], pair[..., 1, :]),
                  kv16.Cache16(mixed[:, 0].unflatten(1, (H, ps, dh)), mixed[:, 1].unflatten(1, (ps, H, dh)).transpose(1, 2))):
        got = kv16.cache16_append(cache, k, v, *args, inv_freq=f, q=both[:, 0], q_out=both[:, 1])
        assert torch.equal(got, ref) and torch.equal(cache.k, own.k) and torch.equal(cache.v, own.v)
    assert torch.equal(both[:, 0], q)
    lens = i32([45], gpu)
    tied, alike = kv16.Cache16(own.k, own.k), kv16.Cache16(own.k, own.k.clone())
    views = kv16.Cache16(own.k[:1].expand(P, -1, -1, -1), own.v[:, :1].expand(-1, H, -1, -1))
    copies = kv16.Cache16(views.k.contiguous(), views.v.contiguous())
    for x, y in ((tied, alike), (views, copies)):
        before = x.k.clone()
        with pytest.raises(sphkv_lib.SphkvError, match="share memory"):
            kv16.cache16_append(x, k, v, *args, inv_freq=f)
        assert torch.equal(x.k, before)
        assert torch.equal(kv16.cache16_decode(x, q[:1], args[0], lens), kv16.cache16_decode(y, q[:1], args[0], lens))
        assert torch.equal(kv16.cache16_prefill(x, q, args[2], args[0], lens), kv16.cache16_prefill(y, q, args[2], args[0], lens))
    flat = torch.zeros(T * 2 * H * dh + 8, dtype=torch.float16, device=gpu)
    over = [flat[a:a + T * 2 * H * dh].view(T, 2 * H, dh) for a in (0, 8)]
    with pytest.raises(sphkv_lib.SphkvError, match="q_out must be q itself"):
        kv16.cache16_append(own, k, v, *args, inv_freq=f, q=over[0], q_out=over[1])


# ---- attention -------------------------------------------------------------------

def score_bound(reach, dh):
    """How far a weight may be off by its score: a sum of dh products, its scaling and its exponent in fp32."""
    return 2.0 ** -24 * (dh + 24) * reach + 2.0 ** -21


def x_bound(parts, lens, dtype, dh, bits):
    """|out - want| before the last rounding.  A weight is off by `delta` (its score) and by 2^-bits of it as a matrix
    operand, fp16 ones by 2^-25 at least, where the largest is 2^8 or more: 2^-33 max p sum |v| (`under`).  Sums of
    products and of weights in fp32 in which a term passes n additions are off by n steps of 2^-23 and 2^-24; `lens`: the
    tokens of the sequences, or n itself."""
    _, _, mass, reach, under = parts
    n = lens if isinstance(lens, int) else max(max(lens), 1)
    rel = 2.0 ** -bits + 2.2 * score_bound(reach, dh) + (n + 64) * 1.5 * 2.0 ** -23
    return rel[..., None] * mass + (2.0 ** -33 * under if dtype is torch.float16 else 0)


def last_rounding(want, dtype):
    return torch.finfo(dtype).eps / 2 * np.abs(want) + (2.0 ** -25 if dtype is torch.float16 else 0)


def check_lse(lse, want, reach, dh, what):
    lse, dead = f64(lse), np.isneginf(want)
    assert np.array_equal(np.isneginf(lse), dead), what
    tol = score_bound(reach, dh) + 2.0 ** -19 + 2.0 ** -21 * np.abs(want, where=~dead, out=np.zeros_like(want))
    assert (np.abs(np.where(dead, 0, lse) - np.where(dead, 0, want)) <= tol).all(), f"{what}: lse"


def check(out, lse, parts, lens, dh, bits, what):
    want, want_lse, _, reach, _ = parts
    dtype = out.dtype
    tol = x_bound(parts, lens, dtype, dh, bits)
    tol = tol * (1 + torch.finfo(dtype).eps) + last_rounding(want, dtype)
    err = np.abs(f64(out) - want)
    log(f"  {what}: max err {err.max(initial=0):.3g}, {(err / np.maximum(tol, 1e-300)).max(initial=0):.3f} of the bound")
    assert (err <= tol).all(), f"{what}: {(err > tol).sum()} outputs off"
    assert (f64(out)[np.isneginf(want_lse)] == 0).all(), what
    check_lse(lse, want_lse, reach, dh, what)


def check_diff(out, lse, maps, lam, weight, eps, lens, dh, bits, what):
    """x = a - lam b, each within its bound, the rounding of the product and the difference 2^-23; normalised, an error dx
    moves x by |dx| and the norm by |dx|_2 / |x|_2 of it."""
    lam = f64(lam)
    w = None if weight is None else f64(weight)
    want, x, scale = o16.difference(maps[0][0], maps[1][0], lam, w, eps)
    dtype = out.dtype
    tol = [x_bound(m, lens, dtype, dh, bits) for m in maps]
    tol = tol[0] + np.abs(lam)[None, :, None] * tol[1]
    tol += 2.0 ** -22 * (np.abs(maps[0][0]) + np.abs(lam)[None, :, None] * np.abs(maps[1][0]))
    if w is not None:
        # sqrt(sum x^2 + dh eps) is what the norm divides by
        size = np.sqrt((x * x).sum(-1, keepdims=True) + dh * eps)
        moved = np.sqrt((tol * tol).sum(-1, keepdims=True)) / size
        assert (moved < 0.5).all()
        # |(x + dx) / size' - x / size| <= (|dx| + |x| moved) / size', size' >= size (1 - moved)
        tol = np.maximum(1.2, 1 / (1 - moved)) * scale * np.abs(w) * (tol + np.abs(x) * moved) + 2.0 ** -20 * np.abs(want)
    tol = tol * (1 + torch.finfo(dtype).eps) + last_rounding(want, dtype)
    err = np.abs(f64(out) - want)
    log(f"  {what}: max err {err.max(initial=0):.3g}, {(err / np.maximum(tol, 1e-300)).max(initial=0):.3f} of the bound")
    assert (err <= tol).all(), f"{what}: {(err > tol).sum()} outputs off"
    assert (f64(out)[np.isneginf(maps[0][1])] == 0).all(), what
    for i in (0, 1):
        check_lse(lse[..., i], maps[i][1], maps[i][3], dh, f"{what} map {i}")


def weight_bits(dtype, prefill, diff):
    """Bits of a weight as it meets its value."""
    two = diff or not prefill or dtype == "fp16"
    return (22 if two else 11) if dtype == "fp16" else (16 if two else 8)


def diff_weights(dev, seed, heads, dh):
    g = torch.Generator(device=dev).manual_seed(seed)
    return 0.2 + 0.6 * torch.rand(heads, generator=g, device=dev), 0.5 + 0.1 * torch.randn(dh, generator=g, device=dev)


def setup(dev, seed, dtype, dh, ps, num_kv, lens, layout="heads", width=0):
    """(cache, oracle, table): numbers that no sequence holds are NaN in the cache."""
    blocks = [-(-max(x, 0) // ps) for x in lens]
    num_pages = sum(blocks) + 2
    cache = random_cache(dev, seed, num_pages, num_kv, dh, ps, dtype, layout)
    table = tables(seed + 1, num_pages, blocks, max(max(blocks), 1) + width)
    want = oracle_of(cache)
    held = np.zeros((num_pages, ps), bool)
    for s, n in enumerate(lens):
        for t in range(max(n, 0)):
            held[table[s, t // ps], t % ps] = True
    gone = torch.from_numpy(~held).to(dev)[:, None, :, None]
    cache.k.masked_fill_(gone, float("nan"))
    cache.v.masked_fill_(gone, float("nan"))
    return cache, want, table


DECODES = [
    # (dtype, dh, page, num_kv, gqa, layout, window, lens)
    ("fp16", 128, 16, 2, 4, "heads", 0, [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0, 300]),
    ("bf16", 128, 32, 2, 8, "tokens", 0, [1, 0, 700, 33, 5, 0]),
    ("fp16", 64, 64, 3, 1, "joined", 0, [200, 1, 64]),
    ("bf16", 64, 128, 1, 7, "heads", 0, [513, 127, 128, 129]),
    ("fp16", 128, 16, 1, 16, "heads", 0, [77, 600]),
    ("bf16", 64, 16, 2, 17, "heads", 0, [50, 3, 333]),
    ("fp16", 64, 32, 1, 64, "heads", 0, [100, 31]),
    ("bf16", 128, 16, 1, 33, "heads", 40, [100, 31, 41, 40]),
    ("fp16", 128, 16, 4, 2, "heads", 1, [1, 2, 33, 500, 0]),
    ("bf16", 128, 64, 2, 4, "tokens", 100, [99, 100, 101, 131, 132, 700]),
    ("fp16", 64, 16, 2, 4, "heads", 2 ** 31 - 1, [64, 5]),
    ("bf16", 64, 16, 1, 3, "heads", 37, [(i * 37) % 150 for i in range(90)]),      # more than 64 sequences
]


@pytest.mark.parametrize("dtype, dh, ps, num_kv, gqa, layout, window, lens", DECODES)
def test_decode(gpu, dtype, dh, ps, num_kv, gqa, layout, window, lens):
    cache, want, table = setup(gpu, 11, dtype, dh, ps, num_kv, lens, layout)
    q = torch.randn((len(lens), num_kv * gqa, dh), device=gpu, generator=torch.Generator(device=gpu).manual_seed(9)).to(TYPES[dtype])
    out, lse = kv16.cache16_decode(cache, q, i32(table, gpu), i32(lens, gpu), window=window, return_lse=True)
    parts = want.attend(f64(q), table, lens, window=window)
    check(out, lse, parts, lens, dh, weight_bits(dtype, False, False), f"decode {dtype} dh {dh} gqa {gqa} window {window}")


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype, dh, ps, num_kv, gqa, layout, window, lens", [c for c in DECODES if c[4] <= 32])
def test_diff_decode(gpu, dtype, dh, ps, num_kv, gqa, layout, window, lens, norm):
    cache, want, table = setup(gpu, 12, dtype, dh, ps, num_kv, lens, layout)
    q = torch.randn((len(lens), num_kv * gqa, dh), device=gpu, generator=torch.Generator(device=gpu).manual_seed(9)).to(TYPES[dtype])
    lam, weight = diff_weights(gpu, 5, num_kv * gqa, dh)
    out, lse = kv16.cache16_diff_decode(cache, q, lam, i32(table, gpu), i32(lens, gpu), norm_weight=weight if norm else None,
                                        norm_eps=1e-3, window=window, return_lse=True)
    maps = want.maps(f64(q), table, lens, window=window)
    check_diff(out, lse, maps, lam, weight if norm else None, 1e-3, lens, dh, weight_bits(dtype, False, True),
               f"diff decode {dtype} dh {dh} gqa {gqa} window {window} norm {norm}")


# more tiles than workgroups can hold at once; pairs cut by workgroups; one long context among short ones
LONG = [
    ("fp16", 128, 16, 8, 4, [30000]),
    ("bf16", 64, 16, 8, 8, [9000, 1, 300, 4000]),
    ("bf16", 128, 128, 4, 4, [2500] * 7 + [11]),
    ("fp16", 64, 32, 2, 20, [12345, 77]),
]


def on_gpu(cache, q, table, lens, window=0, dims=None):
    """One query token a sequence in 64 bits on the GPU: attend()'s five."""
    dh, H, ps = cache.dh, cache.num_kv, cache.page_size
    dims = dims or slice(0, dh)
    gqa = q.shape[1] // H
    res = [np.zeros(q.shape), np.full(q.shape[:2], -np.inf), np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape)]
    for s, n in enumerate(lens):
        a = max(0, n - window) if window else 0
        if n <= 0:
            continue
        pages = torch.as_tensor(table[s, :-(-n // ps)].astype(np.int64), device=q.device)
        k, v = (x[pages].transpose(1, 2).reshape(-1, H, dh)[a:n].double() for x in (cache.k, cache.v))
        for h in range(H):
            rows = q[s, h * gqa:(h + 1) * gqa, dims].double()
            sm = 1 / math.sqrt(dims.stop - dims.start)
            x = rows @ k[:, h, dims].T * sm
            l = torch.logsumexp(x, 1)
            p = torch.exp(x - l[:, None])
            to = (s, slice(h * gqa, (h + 1) * gqa))
            res[0][to], res[1][to], res[2][to] = f64(p @ v[:, h]), f64(l), f64(p @ v[:, h].abs())
            res[3][to] = f64((rows.abs() @ k[:, h, dims].abs().T * sm).amax(1))
            res[4][to] = f64(p.amax(1)[:, None] * v[:, h].abs().sum(0)[None])
    return res


@pytest.mark.parametrize("dtype, dh, ps, num_kv, gqa, lens", LONG)
def test_decode_many_tiles_a_wave(gpu, dtype, dh, ps, num_kv, gqa, lens):
    cache, _, table = setup(gpu, 13, dtype, dh, ps, num_kv, lens)
    # additions that a term passes: the tiles of 32 tokens are spread over 2,048 waves, each adds its own, four waves and
    # the workgroups of a pair join theirs (as many as there are tiles at most)
    tiles = sum(-(-n // 32) for n in lens) * num_kv * 4
    depth = 32 * -(-tiles // 2048) + 4 + min(512, -(-max(lens) // 32))
    q = torch.randn((len(lens), num_kv * gqa, dh), device=gpu, generator=torch.Generator(device=gpu).manual_seed(9)).to(TYPES[dtype])
    lam, weight = diff_weights(gpu, 5, num_kv * gqa, dh)
    for window in (0, 777):
        out, lse = kv16.cache16_decode(cache, q, i32(table, gpu), i32(lens, gpu), window=window, return_lse=True)
        check(out, lse, on_gpu(cache, q, table, lens, window), depth, dh, weight_bits(dtype, False, False), f"decode {lens} {window}")
        out, lse = kv16.cache16_diff_decode(cache, q, lam, i32(table, gpu), i32(lens, gpu), norm_weight=weight, window=window,
                                            return_lse=True)
        maps = [on_gpu(cache, q, table, lens, window, d) for d in (slice(0, dh // 2), slice(dh // 2, dh))]
        check_diff(out, lse, maps, lam, weight, 1e-5, depth, dh, weight_bits(dtype, False, True), f"diff decode {lens} {window}")


def test_decode_lengths_beyond_the_table_and_negative(gpu):
    cache, want, table = setup(gpu, 14, "fp16", 64, 16, 2, [48, 48, 48, 48])
    lens = [1000, 2 ** 31 - 1, -5, -2 ** 31]
    q = torch.randn((4, 4, 64), device=gpu).half()
    out, lse = kv16.cache16_decode(cache, q, i32(table, gpu), i32(lens, gpu), return_lse=True)
    check(out, lse, want.attend(f64(q), table, lens), [48], 64, 22, "lengths")


def test_absent_pages(gpu):
    """Pages outside the cache hold no token, inside a context, at its start and its end, and altogether."""
    lens = [100, 100, 64, 33]
    cache, want, table = setup(gpu, 15, "bf16", 128, 16, 2, lens)
    table[0, [1, 6]] = [-1, 10 ** 6]
    table[1, 0:5] = -7
    table[2, :] = -1
    table[3, 2] = 2 ** 31 - 1
    q = torch.randn((4, 8, 128), device=gpu).bfloat16()
    lam, weight = diff_weights(gpu, 1, 8, 128)
    t, n = i32(table, gpu), i32(lens, gpu)
    out, lse = kv16.cache16_decode(cache, q, t, n, return_lse=True)
    check(out, lse, want.attend(f64(q), table, lens), lens, 128, 16, "decode")
    out, lse = kv16.cache16_diff_decode(cache, q, lam, t, n, norm_weight=weight, return_lse=True)
    check_diff(out, lse, want.maps(f64(q), table, lens), lam, weight, 1e-5, lens, 128, 16, "diff decode")
    cu = np.array([0, 30, 60, 90, 120])
    q = torch.randn((120, 8, 128), device=gpu).bfloat16()
    for window in (0, 20):
        more = dict(cu_rows=cu, window=window)
        out, lse = kv16.cache16_prefill(cache, q, i32(cu, gpu), t, n, window=window, return_lse=True)
        check(out, lse, want.attend(f64(q), table, lens, **more), lens, 128, 8, "prefill")
        out, lse = kv16.cache16_diff_prefill(cache, q, lam, i32(cu, gpu), t, n, norm_weight=weight, window=window, return_lse=True)
        check_diff(out, lse, want.maps(f64(q), table, lens, **more), lam, weight, 1e-5, lens, 128, 16, "diff prefill")


PREFILLS = [
    # (dtype, dh, page, num_kv, gqa, layout, causal, window, [(len, new)])
    ("fp16", 128, 16, 2, 4, "heads", True, 0, [(1, 1), (40, 40), (100, 33), (64, 64), (65, 1), (0, 0), (200, 7)]),
    ("bf16", 128, 32, 1, 8, "tokens", True, 0, [(300, 300), (70, 64)]),
    ("bf16", 64, 64, 2, 1, "heads", True, 0, [(333, 333), (5, 5), (128, 100)]),
    ("fp16", 64, 16, 1, 7, "joined", True, 0, [(90, 50), (64, 63)]),
    ("fp16", 128, 128, 1, 1, "heads", False, 0, [(200, 130), (7, 7), (0, 3)]),
    ("bf16", 64, 16, 2, 3, "heads", False, 0, [(100, 20), (64, 64)]),
    ("fp16", 128, 16, 1, 4, "heads", True, 1, [(100, 100), (33, 9)]),
    ("bf16", 128, 16, 2, 2, "tokens", True, 50, [(300, 300), (200, 3), (49, 49), (129, 80)]),
    ("fp16", 64, 32, 1, 8, "heads", True, 64, [(256, 200), (130, 130)]),
    ("bf16", 64, 64, 1, 4, "heads", True, 100, [(700, 300), (99, 5)]),
    ("bf16", 128, 16, 1, 64, "heads", True, 0, [(40, 20)]),
    ("fp16", 64, 16, 1, 32, "heads", True, 9, [(40, 20), (3, 3)]),
    ("bf16", 128, 16, 1, 4, "heads", True, 0, [(10, 20), (30, 64)]),               # rows before the first token
    ("fp16", 64, 16, 2, 2, "heads", True, 5, [(i % 40, i % 7) for i in range(80)]),  # more than 64 sequences
]


@pytest.mark.parametrize("dtype, dh, ps, num_kv, gqa, layout, causal, window, seqs", PREFILLS)
def test_prefill(gpu, dtype, dh, ps, num_kv, gqa, layout, causal, window, seqs):
    lens, new = [a for a, _ in seqs], [b for _, b in seqs]
    cache, want, table = setup(gpu, 16, dtype, dh, ps, num_kv, lens, layout)
    cu = np.cumsum([0] + new)
    T = int(cu[-1])
    q = torch.randn((T + 2, num_kv * gqa, dh), device=gpu, generator=torch.Generator(device=gpu).manual_seed(9)).to(TYPES[dtype])
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=gpu)
    kv16.cache16_prefill(cache, q, i32(cu, gpu), i32(table, gpu), i32(lens, gpu), causal=causal, window=window, out=out, lse=lse)
    parts = want.attend(f64(q[:T]), table, lens, cu, causal, window)
    check(out[:T], lse[:T], parts, lens, dh, weight_bits(dtype, True, False), f"prefill {dtype} dh {dh} gqa {gqa} window {window}")
    assert (out[T:] == 7.0).all() and (lse[T:] == 7.0).all()


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype, dh, ps, num_kv, gqa, layout, causal, window, seqs", [c for c in PREFILLS if c[4] <= 32])
def test_diff_prefill(gpu, dtype, dh, ps, num_kv, gqa, layout, causal, window, seqs, norm):
    lens, new = [a for a, _ in seqs], [b for _, b in seqs]
    cache, want, table = setup(gpu, 17, dtype, dh, ps, num_kv, lens, layout)
    cu = np.cumsum([0] + new)
    T = int(cu[-1])
    q = torch.randn((T + 2, num_kv * gqa, dh), device=gpu, generator=torch.Generator(device=gpu).manual_seed(9)).to(TYPES[dtype])
    out, lse = torch.full_like(q, 7.0), torch.full((*q.shape[:2], 2), 7.0, device=gpu)
    lam, weight = diff_weights(gpu, 5, num_kv * gqa, dh)
    kv16.cache16_diff_prefill(cache, q, lam, i32(cu, gpu), i32(table, gpu), i32(lens, gpu), norm_weight=weight if norm else None,
                              norm_eps=1e-3, causal=causal, window=window, out=out, lse=lse)
    maps = want.maps(f64(q[:T]), table, lens, cu_rows=cu, causal=causal, window=window)
    check_diff(out[:T], lse[:T], maps, lam, weight if norm else None, 1e-3, lens, dh, weight_bits(dtype, True, True),
               f"diff prefill {dtype} dh {dh} gqa {gqa} window {window} norm {norm}")
    assert (out[T:] == 7.0).all() and (lse[T:] == 7.0).all()


# few rows on long contexts: keys split over workgroups, tiles taken in turn
SPLITS = [
    ("fp16", 128, 16, 2, 4, [(3000, 9), (2000, 20)], 0),
    ("bf16", 128, 64, 4, 8, [(4097, 3)], 1500),
    ("bf16", 64, 16, 2, 4, [(3000, 33), (700, 2)], 0),
    ("fp16", 64, 32, 1, 2, [(2500, 100)], 1000),
    ("bf16", 128, 16, 1, 4, [(1500, 300)], 0),
]


@pytest.mark.parametrize("dtype, dh, ps, num_kv, gqa, seqs, window", SPLITS)
def test_prefill_splits(gpu, dtype, dh, ps, num_kv, gqa, seqs, window):
    lens, new = [a for a, _ in seqs], [b for _, b in seqs]
    cache, want, table = setup(gpu, 18, dtype, dh, ps, num_kv, lens)
    cu = np.cumsum([0] + new)
    q = torch.randn((int(cu[-1]), num_kv * gqa, dh), device=gpu, generator=torch.Generator(device=gpu).manual_seed(9)).to(TYPES[dtype])
    args = (i32(cu, gpu), i32(table, gpu), i32(lens, gpu))
    assert kv16.prefill_workspace_bytes(cache, int(cu[-1]), len(seqs), gqa) > 0
    out, lse = kv16.cache16_prefill(cache, q, *args, window=window, return_lse=True)
    check(out, lse, want.attend(f64(q), table, lens, cu, True, window), lens, dh, weight_bits(dtype, True, False), f"splits {seqs}")
    lam, weight = diff_weights(gpu, 5, num_kv * gqa, dh)
    for w in (weight, None):
        out, lse = kv16.cache16_diff_prefill(cache, q, lam, *args, norm_weight=w, window=window, return_lse=True)
        maps = want.maps(f64(q), table, lens, cu_rows=cu, window=window)
        check_diff(out, lse, maps, lam, w, 1e-5, lens, dh, weight_bits(dtype, True, True), f"diff splits {seqs}")


# more tiles in a workgroup than it looks up at once, unsplit: row tiles of 256 and 128 rows; a few rows each of many
# sequences, tiles taken in turn; windows, so that the first tile is not tile 0
LONG_PREFILLS = [
    ("bf16", 128, 16, 8, 4, [(9000, 1100)], 0),
    ("fp16", 128, 64, 8, 4, [(4200, 300), (8300, 800)], 5000),
    ("bf16", 64, 32, 8, 4, [(9000, 1600)], 0),
    ("fp16", 64, 16, 8, 4, [(6000, 1600)], 4500),
    ("fp16", 128, 128, 8, 4, [(9000, 3), (20, 3), (5000, 4)] + [(100, 1)] * 29, 0),
    ("bf16", 128, 32, 8, 8, [(12500, 2), (20, 3), (9000, 4)] + [(70, 1)] * 29, 10000),
]


def rows_on_gpu(cache, q, table, lens, cu, window, dims=None):
    """Causal rows in 64 bits on the GPU: attend()'s five."""
    dh, H, ps = cache.dh, cache.num_kv, cache.page_size
    dims = dims or slice(0, dh)
    gqa, sm = q.shape[1] // H, 1 / math.sqrt(dims.stop - dims.start)
    res = [np.zeros(q.shape), np.full(q.shape[:2], -np.inf), np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape)]
    for s, n in enumerate(lens):
        ids = table[s, :-(-n // ps)].astype(np.int64)
        there = (ids >= 0) & (ids < cache.num_pages)
        pages = torch.as_tensor(np.where(there, ids, 0), device=q.device)
        there = torch.as_tensor(there, device=q.device).repeat_interleave(ps)[:n]
        k, v = (torch.where(there[:, None, None], x[pages].transpose(1, 2).reshape(-1, H, dh)[:n], 0).double() for x in (cache.k, cache.v))
        a, b = int(cu[s]), int(cu[s + 1])
        if n <= 0 or a == b:
            continue
        pos = torch.arange(n - (b - a), n, device=q.device)[:, None]
        t = torch.arange(n, device=q.device)[None]
        sees = (t <= pos) & there[None] & ((t > pos - window) if window else True)
        for h in range(H):
            for g in range(h * gqa, (h + 1) * gqa):
                rows = q[a:b, g, dims].double()
                x = (rows @ k[:, h, dims].T * sm).masked_fill(~sees, -math.inf)
                l = torch.logsumexp(x, 1)
                p = torch.exp(x - l[:, None]).masked_fill(~sees, 0)
                reach = (rows.abs() @ k[:, h, dims].abs().T * sm).masked_fill(~sees, 0).amax(1)
                under = p.amax(1)[:, None] * (sees.double() @ v[:, h].abs())
                for to, x in zip(res, (p @ v[:, h], l, p @ v[:, h].abs(), reach, under)):
                    to[a:b, g] = f64(x)
    return res


@pytest.mark.parametrize("dtype, dh, ps, num_kv, gqa, seqs, window", LONG_PREFILLS)
def test_prefill_many_tiles(gpu, dtype, dh, ps, num_kv, gqa, seqs, window):
    lens, new = [a for a, _ in seqs], [b for _, b in seqs]
    cache, _, table = setup(gpu, 28, dtype, dh, ps, num_kv, lens)
    for token in (1000, lens[0] - new[0] + 1, lens[0] - 40):             # pages that are not there, early and late
        table[0, token // ps] = -1
    cu = np.cumsum([0] + new)
    rows = int(cu[-1])
    q = torch.randn((rows, num_kv * gqa, dh), device=gpu, generator=torch.Generator(device=gpu).manual_seed(9)).to(TYPES[dtype])
    args = (i32(cu, gpu), i32(table, gpu), i32(lens, gpu))
    lam, weight = diff_weights(gpu, 5, num_kv * gqa, dh)
    for diff in (False, True):
        assert kv16.prefill_workspace_bytes(cache, rows, len(lens), gqa, diff) == 0
    out, lse = kv16.cache16_prefill(cache, q, *args, window=window, return_lse=True)
    check(out, lse, rows_on_gpu(cache, q, table, lens, cu, window), lens, dh, weight_bits(dtype, True, False), f"many tiles {dtype} {dh}")
    out, lse = kv16.cache16_diff_prefill(cache, q, lam, *args, norm_weight=weight, window=window, return_lse=True)
    maps = [rows_on_gpu(cache, q, table, lens, cu, window, d) for d in (slice(0, dh // 2), slice(dh // 2, dh))]
    check_diff(out, lse, maps, lam, weight, 1e-5, lens, dh, weight_bits(dtype, True, True), f"diff many tiles {dtype} {dh}")


# more row tiles than run at once, of 2 to 9 sequences (up to 8 are taken by how far their tiles reach): equal ones, empty
# ones, ones without rows, rows before the first token, a tile that two share the reach of, one reach of its own
ORDERS = [
    [(1024, 1024)] * 2,
    [(700, 600), (0, 0), (300, 300), (1200, 37), (90, 500), (64, 64), (2000, 256), (1, 1)],
    [(0, 0), (900, 0), (1500, 1500), (40000, 70), (0, 90)],
    [(5, 5), (1337, 1337), (257, 257), (3, 3)],
    [(600, 300)] * 7 + [(1, 1)] * 2,
]


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("dtype, dh, gqa", [("bf16", 128, 4), ("fp16", 64, 7), ("fp16", 128, 3)])
@pytest.mark.parametrize("seqs", ORDERS)
def test_prefill_order(gpu, dtype, dh, gqa, seqs, window):
    lens, new, H = [a for a, _ in seqs], [b for _, b in seqs], 8
    cache, _, table = setup(gpu, 33, dtype, dh, 32, H, lens)
    cu = np.cumsum([0] + new)
    rows = int(cu[-1])
    q = torch.randn((rows + 3, H * gqa, dh), device=gpu, generator=torch.Generator(device=gpu).manual_seed(9)).to(TYPES[dtype])
    args = (i32(cu, gpu), i32(table, gpu), i32(lens, gpu))
    lam, _ = diff_weights(gpu, 5, H * gqa, dh)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=gpu)
    kv16.cache16_prefill(cache, q, *args, window=window, out=out, lse=lse)
    check(out[:rows], lse[:rows], rows_on_gpu(cache, q[:rows], table, lens, cu, window), lens, dh, weight_bits(dtype, True, False), f"order {seqs}")
    assert (out[rows:] == 7.0).all() and (lse[rows:] == 7.0).all()
    out, lse = kv16.cache16_diff_prefill(cache, q, lam, *args, window=window, return_lse=True)
    maps = [rows_on_gpu(cache, q[:rows], table, lens, cu, window, d) for d in (slice(0, dh // 2), slice(dh // 2, dh))]
    check_diff(out[:rows], lse[:rows], maps, lam, None, 1e-5, lens, dh, weight_bits(dtype, True, True), f"diff order {seqs}")


# contexts of up to 625 tiles: row tiles of 256 and 128 rows, tiles in turn, splits
EACH_TILE = [
    ("bf16", 128, 16, 8, 4, [(9000, 1100)]),
    ("fp16", 128, 32, 8, 3, [(0, 0), (900, 0), (1500, 1500), (40000, 70), (0, 90)]),
    ("bf16", 64, 32, 8, 4, [(9000, 1600)]),
    ("fp16", 128, 128, 8, 4, [(9000, 3), (20, 3), (5000, 4)] + [(100, 1)] * 29),
    ("bf16", 128, 16, 2, 4, [(30000, 9)]),
    ("fp16", 64, 16, 2, 4, [(30000, 33), (3000, 2)]),
]


@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("dtype, dh, ps, num_kv, gqa, seqs", EACH_TILE)
def test_every_tile_of_a_long_context_counts(gpu, dtype, dh, ps, num_kv, gqa, seqs, diff):
    """A tile's values lie in one element, so that an output is the sum of a few tiles: keys or values of one of hundreds
    taken from another tile are far past the bound, as the oracle with such a tile in it shows."""
    lens, new = [a for a, _ in seqs], [b for _, b in seqs]
    cache, _, table = setup(gpu, 35, dtype, dh, ps, num_kv, lens)
    long = int(np.argmax(lens))
    v = torch.zeros_like(cache.v)
    for s, n in enumerate(lens):
        token = torch.arange(n, device=gpu)
        page = torch.as_tensor(table[s].astype(np.int64), device=gpu)[token // ps]
        d = (token // 64) % dh
        v[page, :, token % ps, d] = cache.v[page, :, token % ps, d].abs() + 1
    cache = kv16.Cache16(cache.k, v)
    bad = kv16.Cache16(cache.k.clone(), v.clone())                        # a late tile's keys and values are the next one's
    tile = lens[long] // 64 - 3
    at = [[(int(table[long, t // ps]), t % ps) for t in range(64 * i, 64 * i + 64)] for i in (tile, tile + 1)]
    to, of = (torch.as_tensor(x, device=gpu).T for x in at)
    bad.k[to[0], :, to[1]], bad.v[to[0], :, to[1]] = cache.k[of[0], :, of[1]], cache.v[of[0], :, of[1]]
    bits = 22 if dtype == "fp16" else 16
    cu = np.cumsum([0] + new)
    rows = int(cu[-1])
    q = (0.5 * torch.randn((rows, num_kv * gqa, dh), device=gpu, generator=torch.Generator(device=gpu).manual_seed(9))).to(TYPES[dtype])
    args = (i32(cu, gpu), i32(table, gpu), i32(lens, gpu))
    last = slice(int(cu[long + 1]) - 1, int(cu[long + 1]))
    few = [0] * long + [lens[long]] + [0] * (len(lens) - long - 1)        # the last row of the long context alone
    one = [0] * (long + 1) + [1] * (len(lens) - long)
    if diff:
        lam = torch.full((num_kv * gqa,), 0.5, device=gpu)
        out, lse = kv16.cache16_diff_prefill(cache, q, lam, *args, return_lse=True)
        halves = (slice(0, dh // 2), slice(dh // 2, dh))
        maps = [rows_on_gpu(cache, q, table, lens, cu, 0, d) for d in halves]
        for s, n in enumerate(lens):                                      # (each by its own length)
            of = slice(int(cu[s]), int(cu[s + 1]))
            check_diff(out[of], lse[of], [[x[of] for x in m] for m in maps], lam, None, 0, [n], dh, bits, f"each tile {dtype} {dh} {n}")
        wrong = [rows_on_gpu(bad, q[last], table, few, one, 0, d) for d in halves]
        tol = x_bound([x[last] for x in maps[0]], lens, TYPES[dtype], dh, bits) + 0.5 * x_bound([x[last] for x in maps[1]], lens, TYPES[dtype], dh, bits)
        want, other = maps[0][0][last] - 0.5 * maps[1][0][last], wrong[0][0] - 0.5 * wrong[1][0]
    else:
        out, lse = kv16.cache16_prefill(cache, q, *args, return_lse=True)
        parts = rows_on_gpu(cache, q, table, lens, cu, 0)
        for s, n in enumerate(lens):
            of = slice(int(cu[s]), int(cu[s + 1]))
            check(out[of], lse[of], [x[of] for x in parts], [n], dh, bits, f"each tile {dtype} {dh} {n}")
        other = rows_on_gpu(bad, q[last], table, few, one, 0)[0]
        want, tol = parts[0][last], x_bound([x[last] for x in parts], lens, TYPES[dtype], dh, bits)
    assert (np.abs(other - want) > 4 * (tol + last_rounding(want, TYPES[dtype]))).any(-1).all()


@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dh", [64, 128])
def test_prefill_values_that_are_not_finite(gpu, dtype, dh, diff):
    """An infinity or NaN among the values reaches the rows that see its token, and no other, whatever the tile."""
    L, gqa = 200, 2
    cache, _, table = setup(gpu, 19, dtype, dh, 16, 1, [L])
    clean = kv16.Cache16(cache.k.clone(), cache.v.clone())
    put = {30: (3, float("inf")), 64: (dh - 1, float("-inf")), 100: (0, float("nan")), 150: (3, float("-inf"))}
    for t, (d, x) in put.items():
        cache.v[int(table[0, t // 16]), 0, t % 16, d] = x
    q = (0.1 * torch.randn((L, gqa, dh), device=gpu)).to(TYPES[dtype])
    args = (i32([0, L], gpu), i32(table, gpu), i32([L], gpu))
    lam = torch.full((gqa,), 0.5, device=gpu)
    run = (lambda c, **kw: kv16.cache16_diff_prefill(c, q, lam, *args, **kw)) if diff else (lambda c, **kw: kv16.cache16_prefill(c, q, *args, **kw))
    for window in (0, 40):
        got, base = run(cache, window=window), run(clean, window=window)
        pos = torch.arange(L, device=gpu)
        for d in range(dh):
            sees = {t: (pos >= t) & ((pos - t < window) if window else True) for t, (at, _) in put.items() if at == d}
            hit = torch.zeros(L, dtype=torch.bool, device=gpu)
            for m in sees.values():
                hit |= m
            assert torch.equal(got[~hit][:, :, d], base[~hit][:, :, d]), (window, d)
            for t, m in sees.items():
                only = m.clone()
                for u, o in sees.items():
                    if u != t:
                        only &= ~o
                # (an infinity times a weight's second number, which may be 0 or negative, is NaN beside the first's)
                assert not got[only][:, :, d].isfinite().any(), (window, d, t)


@pytest.mark.parametrize("dh", [64, 128])
def test_scores_of_any_size(gpu, dh):
    """Scores of magnitude 2^30 and beyond: the largest takes all, no overflow; equal ones share."""
    ps, n = 16, 40
    for scale in (1.0, 2.0 ** 9, 2.0 ** 15):
        cache = kv16.Cache16.allocate(4, 1, dh, ps, torch.float16, gpu)
        g = torch.Generator(device=gpu).manual_seed(3)
        k = torch.randint(-1, 2, (n, dh), generator=g, device=gpu).half() * scale
        k[7], k[25] = scale, scale
        v = torch.randn((n, dh), generator=g, device=gpu).half()
        table = i32([[2, 0, 1]], gpu)
        kv16.cache16_append(cache, k[:, None], v[:, None], table, i32([0], gpu), i32([0, n], gpu))
        q = torch.full((1, 2, dh), scale, dtype=torch.float16, device=gpu)
        want = o16.Cache(f64(cache.k), f64(cache.v)).attend(f64(q), table.cpu().numpy(), [n])
        for out, lse in (kv16.cache16_decode(cache, q, table, i32([n], gpu), return_lse=True),
                         kv16.cache16_prefill(cache, q, i32([0, 1], gpu), table, i32([n], gpu), return_lse=True)):
            err = np.abs(f64(out) - want[0])
            # scores are whole multiples of scale^2 and exact in fp32; times sm_scale log2(e) equal ones stay equal, others
            # differ by at least scale^2 / 16; at scale 1 the bounds of check() hold as they are
            if scale == 1.0:
                check(out, lse, want, [n], dh, 22, "scores")
            else:
                assert (err <= 2.0 ** -10 * np.abs(want[0]) + 2.0 ** -20).all(), (scale, err.max())
            assert (np.abs(f64(lse) - want[1]) <= 2.0 ** -21 * np.abs(want[1]) + 2.0 ** -18).all()


def cancelling(dev, dtype, dh, n, num_kv, gqa, ps=16):
    """Values that cancel: token 2 i has +b, token 2 i + 1 -b, on scores that differ a little, so that an output is what is
    left of sums hundreds of times its size."""
    g = torch.Generator(device=dev).manual_seed(21)
    blocks = -(-n // ps)
    k = 0.3 * torch.randn((n, num_kv, dh), generator=g, device=dev)
    v = 8.0 + torch.randn((n // 2, num_kv, dh), generator=g, device=dev)
    v = torch.stack([v, -v], 1).reshape(n, num_kv, dh)
    cache = kv16.Cache16.allocate(blocks, num_kv, dh, ps, TYPES[dtype], dev)
    table = i32([list(range(blocks))], dev)
    kv16.cache16_append(cache, k.to(TYPES[dtype]), v.to(TYPES[dtype]), table, i32([0], dev), i32([0, n], dev))
    q = 0.3 * torch.randn((1, num_kv * gqa, dh), generator=g, device=dev)
    return cache, table, q.to(TYPES[dtype])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dh, num_kv, gqa", [(128, 2, 1), (64, 1, 4), (128, 1, 8), (64, 1, 16), (128, 1, 40)])
def test_decode_weights_are_two_numbers(gpu, dtype, dh, num_kv, gqa):
    """Outputs far below their terms: within the bound of two numbers a weight, 2^-11 or 2^-8 of the mass would be far off."""
    cache, table, q = cancelling(gpu, dtype, dh, 64, num_kv, gqa)
    out, lse = kv16.cache16_decode(cache, q, table, i32([64], gpu), return_lse=True)
    parts = oracle_of(cache).attend(f64(q), table.cpu().numpy(), [64])
    check(out, lse, parts, [64], dh, weight_bits(dtype, False, False), "decode")


@pytest.mark.parametrize("dtype, diff", [("fp16", False), ("fp16", True), ("bf16", True)])
@pytest.mark.parametrize("dh", [64, 128])
def test_prefill_weights_are_two_numbers(gpu, dtype, dh, diff):
    cache, table, q = cancelling(gpu, dtype, dh, 64, 1, 8)
    args = (i32([0, 1], gpu), table, i32([64], gpu))
    if diff:
        lam = torch.full((8,), 0.5, device=gpu)
        out, lse = kv16.cache16_diff_prefill(cache, q, lam, *args, return_lse=True)
        maps = oracle_of(cache).maps(f64(q), table.cpu().numpy(), [64])
        check_diff(out, lse, maps, lam, None, 0, [64], dh, weight_bits(dtype, True, True), "diff prefill")
    else:
        out, lse = kv16.cache16_prefill(cache, q, *args, return_lse=True)
        check(out, lse, oracle_of(cache).attend(f64(q), table.cpu().numpy(), [64]), [64], dh, 22, "prefill")


@pytest.mark.parametrize("dh, rows, gqa", [(128, 1, 8), (128, 40, 4), (64, 40, 4)])
def test_prefill_bf16_weights_are_two_numbers(gpu, dh, rows, gqa):
    """Tiles taken in turn and by row tiles: outputs far below their terms, to which a weight of 8 bits would show."""
    n = 128
    cache, table, _ = cancelling(gpu, "bf16", dh, n, 1, gqa)
    q = (0.3 * torch.randn((rows, gqa, dh), generator=torch.Generator(device=gpu).manual_seed(4), device=gpu)).bfloat16()
    cu = [0, rows]
    out, lse = kv16.cache16_prefill(cache, q, i32(cu, gpu), table, i32([n], gpu), causal=False, return_lse=True)
    parts = oracle_of(cache).attend(f64(q), table.cpu().numpy(), [n], cu, causal=False)
    check(out, lse, parts, [n], dh, 16, f"bf16 prefill dh {dh} rows {rows}")


# rows of a call and kv heads: decode; prefill's tiles in turn, split and not; row tiles, split and not
SHAPES = [("decode", 1, 4), ("decode", 1, 300), ("prefill", 2, 2), ("prefill", 2, 400), ("prefill", 140, 2), ("prefill", 140, 400)]


@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("late", [False, True])
@pytest.mark.parametrize("dtype, dh", [("fp16", 128), ("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("kind, rows, H", SHAPES)
def test_equal_scores_share_in_any_tile(gpu, kind, rows, H, dtype, dh, late, diff):
    """A few equal keys far above all others, in different tiles (late: larger ones behind them): their values' mean, at any
    magnitude of the scores.  Equal numbers meet the same roundings, so an output is off by the weights' bits, a few fp32
    sums and its own rounding alone; 3,600 makes scores whose fp32 step is 16 in the exponent of two."""
    n, ps = 1000, 16
    first, behind = [5, 70, 333, 400], [600, 990]
    top = behind if late else first
    table = np.random.default_rng(5).permutation(-(-n // ps))[None].astype(np.int32)
    pages = torch.as_tensor(table[0].astype(np.int64), device=gpu)
    for size in (6.0, 64.0, 512.0, 3600.0):
        g = torch.Generator(device=gpu).manual_seed(7)
        key = size * torch.exp(0.2 * torch.randn((H, dh), generator=g, device=gpu))          # (all positive)
        k = 0.25 * size * torch.randn((n, H, dh), generator=g, device=gpu)
        k[first] = key
        if late:
            k[behind] = 1.5 * key
        v = torch.randn((n, H, dh), generator=g, device=gpu)
        cache = kv16.Cache16.allocate(table.size, H, dh, ps, TYPES[dtype], gpu)
        k, v = (torch.cat([x, x.new_zeros((table.size * ps - n, H, dh))]).to(TYPES[dtype]).view(-1, ps, H, dh).transpose(1, 2) for x in (k, v))
        cache.k[pages], cache.v[pages] = k, v
        q = (size * torch.exp(0.2 * torch.randn((rows, H, dh), generator=g, device=gpu))).to(TYPES[dtype])
        lam = torch.full((H,), 0.5, device=gpu)
        args = (i32(table, gpu), i32([n], gpu))
        if kind == "decode":
            out, lse = kv16.cache16_diff_decode(cache, q, lam, *args, return_lse=True) if diff else kv16.cache16_decode(cache, q, *args, return_lse=True)
        else:
            cu, more = i32([0, rows], gpu), dict(causal=False, return_lse=True)
            out, lse = kv16.cache16_diff_prefill(cache, q, lam, cu, *args, **more) if diff else kv16.cache16_prefill(cache, q, cu, *args, **more)
        kk, vv = (x.transpose(1, 2).reshape(-1, H, dh)[:n].double() for x in (k, v))
        for i, d in enumerate((slice(0, dh // 2), slice(dh // 2, dh)) if diff else (slice(0, dh),)):
            s = torch.bmm(q[..., d].double().transpose(0, 1).contiguous(), kk[..., d].permute(1, 2, 0).contiguous())
            s = s.transpose(0, 1) / math.sqrt(d.stop - d.start)
            others = s.clone()
            others[..., top] = -math.inf
            most = s[..., top[0]]
            assert (most - others.amax(-1) > 40).all()                   # (e^-40 of the others)
            want = f64(most) + math.log(len(top))
            check_lse(lse[..., i] if diff else lse, want, f64(q[..., d].double().mul(kk[top[0], :, d]).sum(-1) / math.sqrt(d.stop - d.start)), dh, f"size {size}")
        want = vv[top].mean(0)[None].expand(rows, -1, -1) * (0.5 if diff else 1.0)
        mass = vv[top].abs().mean(0)[None] * (1.5 if diff else 1.0)
        tol = (2.0 ** (-22 if dtype == "fp16" else -16) + 2.0 ** -19) * f64(mass) + last_rounding(f64(want), TYPES[dtype]) * 1.01
        err = np.abs(f64(out) - f64(want))
        log(f"  {kind} {rows} x {H} {dtype} dh {dh} size {size}: {np.nan_to_num(err / tol, nan=9e9).max():.3f} of the bound")
        assert (err <= tol).all(), f"size {size}: {(~(err <= tol)).sum()} outputs off"


def test_nan_query_and_key_stay_in_their_rows(gpu):
    lens = [50, 70]
    cache, want, table = setup(gpu, 22, "fp16", 128, 16, 2, lens)
    q = torch.randn((2, 8, 128), device=gpu).half()
    q[0, 3, 5] = float("nan")
    args = (i32(table, gpu), i32(lens, gpu))
    base = torch.nan_to_num(q)
    out, ref = kv16.cache16_decode(cache, q, *args), kv16.cache16_decode(cache, base, *args)
    assert out[0, 3].isnan().all()
    mask = torch.ones((2, 8), dtype=torch.bool, device=gpu)
    mask[0, 3] = False
    assert torch.equal(out[mask], ref[mask])
    cache.k[int(table[1, 1]), 1, 4, 0] = float("nan")                    # token 20 of the second, its second kv head
    out = kv16.cache16_decode(cache, base, *args)
    assert out[1, 4:].isnan().all() and torch.equal(out[0], ref[0]) and torch.equal(out[1, :4], ref[1, :4])
    rows = base.repeat(20, 1, 1)[:40]
    cu = i32([0, 0, 40], gpu)
    out = kv16.cache16_prefill(cache, rows, cu, *args)                   # rows at positions 30 .. 69 of the second: all see token 20
    assert out[:, 4:].isnan().all() and out[:, :4].isfinite().all()


def test_query_strides(gpu):
    lens = [50, 70, 9]
    cache, want, table = setup(gpu, 23, "bf16", 64, 16, 2, lens)
    raw = torch.randn(3 * 700 + 1, device=gpu).bfloat16()
    q = raw[1:].view(3, 700)[:, 8:8 + 6 * 70].unflatten(1, (6, 70))[..., 3:67]
    args = (i32(table, gpu), i32(lens, gpu))
    assert torch.equal(kv16.cache16_decode(cache, q, *args), kv16.cache16_decode(cache, q.contiguous(), *args))
    cu = i32([0, 1, 1, 3], gpu)
    assert torch.equal(kv16.cache16_prefill(cache, q, cu, *args), kv16.cache16_prefill(cache, q.contiguous(), cu, *args))


@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("dtype, dh", [("fp16", 128), ("bf16", 128), ("bf16", 64)])
def test_late_values_that_are_not_finite(gpu, dtype, dh, diff):
    """Values that are not finite in tiles past the first 64 that a workgroup looks up."""
    L, n, H, gqa = 5000, 1600, 8, 4
    cache, _, table = setup(gpu, 30, dtype, dh, 16, H, [L])
    clean = kv16.Cache16(cache.k.clone(), cache.v.clone())
    put = {4500: (3, float("inf")), 4990: (5, float("nan"))}
    for t, (d, x) in put.items():
        cache.v[int(table[0, t // 16]), 2, t % 16, d] = x
    q = (0.1 * torch.randn((n, H * gqa, dh), device=gpu)).to(TYPES[dtype])
    args = (i32([0, n], gpu), i32(table, gpu), i32([L], gpu))
    lam = torch.full((H * gqa,), 0.5, device=gpu)
    run = (lambda c: kv16.cache16_diff_prefill(c, q, lam, *args)) if diff else (lambda c: kv16.cache16_prefill(c, q, *args))
    assert kv16.prefill_workspace_bytes(cache, n, 1, gqa, diff) == 0
    got, base = run(cache), run(clean)
    hit = torch.zeros_like(got, dtype=torch.bool)
    for t, (d, _) in put.items():
        hit[t - (L - n):, 2 * gqa:3 * gqa, d] = True
    assert not got[hit].isfinite().any()
    assert torch.equal(got[~hit], base[~hit])


def test_outputs_over_their_queries(gpu):
    """out may be q: each row's queries are read before its output is written."""
    lens = [5000, 70, 300, 1] + [40] * 60
    for dtype, dh, gqa in (("fp16", 128, 4), ("bf16", 64, 20), ("bf16", 128, 2)):
        cache, want, table = setup(gpu, 29, dtype, dh, 16, 4, lens)
        lam, weight = diff_weights(gpu, 5, 4 * gqa, dh)
        args = (i32(table, gpu), i32(lens, gpu))
        q = torch.randn((len(lens), 4 * gqa, dh), device=gpu).to(TYPES[dtype])
        cu = i32([0] + [len(lens) - 5] * 2 + [len(lens)] * (len(lens) - 2), gpu)
        for run in (lambda x, **kw: kv16.cache16_decode(cache, x, *args, **kw),
                    lambda x, **kw: kv16.cache16_diff_decode(cache, x, lam, *args, norm_weight=weight, **kw),
                    lambda x, **kw: kv16.cache16_prefill(cache, x, cu, *args, **kw),
                    lambda x, **kw: kv16.cache16_diff_prefill(cache, x, lam, cu, *args, **kw)):
            ref, x = run(q), q.clone()
            assert run(x, out=x) is x and torch.equal(x, ref)


def test_outputs_beside_their_queries(gpu):
    """Queries and outputs in one buffer without a common byte, as in buffers of their own; a shifted output is refused."""
    lens = [70, 300, 1]
    cache, want, table = setup(gpu, 36, "fp16", 64, 16, 2, lens)
    flat = torch.randn(2 * 3 * 8 * 64 + 64, device=gpu).half()
    q, out = flat[:3 * 8 * 64].view(3, 8, 64), flat[3 * 8 * 64:2 * 3 * 8 * 64].view(3, 8, 64)
    near = flat[64:3 * 8 * 64 + 64].view(3, 8, 64)
    lam = torch.full((8,), 0.5, device=gpu)
    args, cu = (i32(table, gpu), i32(lens, gpu)), i32([0, 1, 2, 3], gpu)
    for run in (lambda **kw: kv16.cache16_decode(cache, q, *args, **kw), lambda **kw: kv16.cache16_diff_decode(cache, q, lam, *args, **kw),
                lambda **kw: kv16.cache16_prefill(cache, q, cu, *args, **kw), lambda **kw: kv16.cache16_diff_prefill(cache, q, lam, cu, *args, **kw)):
        ref = run()
        assert torch.equal(run(out=out), ref)
        with pytest.raises(sphkv_lib.SphkvError, match="out must be q itself"):
            run(out=near)


def test_graphs_that_share_a_workspace(gpu):
    """Two captured graphs over one workspace, replayed in turn with eager calls between."""
    lens = [900, 70, 4000]
    cache, want, table = setup(gpu, 31, "bf16", 128, 16, 2, lens)
    t, n, cu = i32(table, gpu), i32(lens, gpu), i32([0, 1, 2, 3], gpu)
    lam, weight = diff_weights(gpu, 5, 8, 128)
    need = max(kv16.decode_workspace_bytes(cache, 3, 4, True), kv16.prefill_workspace_bytes(cache, 3, 3, 4))
    ws = torch.empty(need, dtype=torch.uint8, device=gpu)
    q = [torch.empty((3, 8, 128), dtype=torch.bfloat16, device=gpu) for _ in range(2)]

    def one(w):
        return kv16.cache16_decode(cache, q[0], t, n, workspace=w), kv16.cache16_prefill(cache, q[0], cu, t, n, workspace=w)

    def two(w):
        return (kv16.cache16_diff_decode(cache, q[1], lam, t, n, norm_weight=weight, window=1000, workspace=w),)

    for x in q:
        x.normal_()
    one(ws), two(ws)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for f in (one, two):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(f(ws))
    for i in range(4):
        for x in q:
            x.normal_()
        n.copy_(i32([900 - 200 * i, 70, 4000 - 1200 * i], gpu))
        for g in (graphs if i % 2 else graphs[::-1]):
            g.replay()
            two(ws)
        torch.cuda.synchronize()
        for got, f in zip(outs, (one, two)):
            for a, b in zip(got, f(None)):
                assert torch.equal(a, b)


def test_given_outputs_and_workspace(gpu):
    lens = [500, 70, 0]
    cache, want, table = setup(gpu, 24, "fp16", 128, 16, 2, lens)
    q = torch.randn((3, 8, 128), device=gpu).half()
    lam, weight = diff_weights(gpu, 5, 8, 128)
    args = (i32(table, gpu), i32(lens, gpu))
    ref, rlse = kv16.cache16_decode(cache, q, *args, return_lse=True)
    dref, dlse = kv16.cache16_diff_decode(cache, q, lam, *args, norm_weight=weight, return_lse=True)
    for diff in (False, True):
        need = kv16.decode_workspace_bytes(cache, 3, 4, diff)
        ws = torch.full((need,), 255, dtype=torch.uint8, device=gpu)      # NaN in every number it may hold
        buf = torch.full((3 * 8 * 128 + 1,), 3.0, dtype=torch.float16, device=gpu)
        out = buf[1:].view(3, 8, 128)                                     # 2 bytes off any vector
        lse = torch.empty((3, 8, 2) if diff else (3, 8), device=gpu)
        if diff:
            got = kv16.cache16_diff_decode(cache, q, lam, *args, norm_weight=weight, out=out, lse=lse, workspace=ws)
        else:
            got = kv16.cache16_decode(cache, q, *args, out=out, lse=lse, workspace=ws)
        assert got is out and torch.equal(out, dref if diff else ref) and torch.equal(lse, dlse if diff else rlse)
        assert buf[0] == 3.0
        with pytest.raises(ValueError):
            kv16.cache16_decode(cache, q, *args, workspace=ws[:kv16.decode_workspace_bytes(cache, 3, 4) - 1])
    cu = i32([0, 1, 2, 3], gpu)
    ref = kv16.cache16_prefill(cache, q, cu, *args)
    ws = torch.full((kv16.prefill_workspace_bytes(cache, 3, 3, 4),), 255, dtype=torch.uint8, device=gpu)
    buf = torch.empty(3 * 8 * 128 + 1, dtype=torch.float16, device=gpu)
    out = buf[1:].view(3, 8, 128)
    kv16.cache16_prefill(cache, q, cu, *args, out=out, workspace=ws)
    assert torch.equal(out, ref)


@pytest.mark.parametrize("dtype, dh, ps, parts, diff", [("fp16", 128, 16, 1, False), ("bf16", 64, 64, 1, False),
                                                        ("bf16", 128, 32, 2, True), ("fp16", 64, 16, 2, True)])
def test_prompts_then_decode_steps(gpu, dtype, dh, ps, parts, diff):
    """The calls as a server makes them: prompts in and attended, then tokens one at a time; the cache and the rotated
    queries as the calls left them are what attention is held to."""
    H, gqa, prompts, steps = 2, 4, [37, 1, 90], 4
    n, dt = len(prompts), TYPES[dtype]
    g = torch.Generator(device=gpu).manual_seed(31)
    blocks = [-(-(p + steps) // ps) for p in prompts]
    cache = kv16.Cache16.allocate(sum(blocks), H, dh, ps, dt, gpu)
    cache.k.fill_(float("nan")), cache.v.fill_(float("nan"))
    table = tables(1, sum(blocks), blocks)
    t = i32(table, gpu)
    f = kv16.rope_inv_freq(dh // parts, device=gpu)
    lam, weight = diff_weights(gpu, 5, H * gqa, dh)
    lens = i32(prompts, gpu)
    cu = np.cumsum([0] + prompts)

    def rows(m):
        x = torch.randn((m, H * (gqa + 2), dh), generator=g, device=gpu).to(dt)
        return x[:, :H * gqa], x[:, H * gqa:H * (gqa + 1)], x[:, H * (gqa + 1):]

    q, k, v = rows(int(cu[-1]))
    q = kv16.cache16_append(cache, k, v, t, i32([0] * n, gpu), i32(cu, gpu), inv_freq=f, parts=parts, q=q)
    want = oracle_of(cache)
    if diff:
        out, lse = kv16.cache16_diff_prefill(cache, q, lam, i32(cu, gpu), t, lens, norm_weight=weight, return_lse=True)
        check_diff(out, lse, want.maps(f64(q), table, prompts, cu_rows=cu), lam, weight, 1e-5, prompts, dh, weight_bits(dtype, True, True), "prompts")
    else:
        out, lse = kv16.cache16_prefill(cache, q, i32(cu, gpu), t, lens, return_lse=True)
        check(out, lse, want.attend(f64(q), table, prompts, cu), prompts, dh, weight_bits(dtype, True, False), "prompts")
    for step in range(steps):
        q, k, v = rows(n)
        q = kv16.cache16_append(cache, k, v, t, lens, inv_freq=f, parts=parts, q=q)
        lens += 1
        now = [p + step + 1 for p in prompts]
        want = oracle_of(cache)
        if diff:
            out, lse = kv16.cache16_diff_decode(cache, q, lam, t, lens, norm_weight=weight, return_lse=True)
            check_diff(out, lse, want.maps(f64(q), table, now), lam, weight, 1e-5, now, dh, weight_bits(dtype, False, True), f"step {step}")
        else:
            out, lse = kv16.cache16_decode(cache, q, t, lens, return_lse=True)
            check(out, lse, want.attend(f64(q), table, now), now, dh, weight_bits(dtype, False, False), f"step {step}")


def test_captured_step_follows_its_tensors(gpu):
    """Append, decode and differential decode captured once and replayed as the sequences grow, eager work between."""
    H, gqa, dh, ps, n = 2, 4, 128, 16, 3
    g = torch.Generator(device=gpu).manual_seed(3)
    caches = [kv16.Cache16.allocate(24, H, dh, ps, torch.float16, gpu) for _ in range(2)]
    table = i32(tables(1, 24, [8, 8, 8]), gpu)
    lam, weight = diff_weights(gpu, 5, H * gqa, dh)
    f = kv16.rope_inv_freq(dh, device=gpu)
    lens = [i32([5, 100, 0], gpu) for _ in range(2)]
    for c in caches:
        c.k.normal_(generator=torch.Generator(device=gpu).manual_seed(1))
        c.v.normal_(generator=torch.Generator(device=gpu).manual_seed(2))
    x = torch.empty((n, H * (gqa + 2), dh), dtype=torch.float16, device=gpu)

    def step(c, lens):
        q, k, v = x[:, :H * gqa], x[:, H * gqa:H * (gqa + 1)], x[:, H * (gqa + 1):]
        q = kv16.cache16_append(c, k, v, table, lens, inv_freq=f, q=q)
        lens += 1
        return (q, kv16.cache16_decode(c, q, table, lens, return_lse=True),
                kv16.cache16_diff_decode(c, q, lam, table, lens, norm_weight=weight, window=50, return_lse=True))

    x.normal_(generator=g)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(caches[0], lens[0].clone())                                  # warm
    torch.cuda.synchronize()
    caches[0].k.copy_(caches[1].k), caches[0].v.copy_(caches[1].v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0], lens[0])
    for _ in range(6):
        x.normal_(generator=g)
        want = step(caches[1], lens[1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0])
        for a, b in zip(got[1] + got[2], want[1] + want[2]):
            assert torch.equal(a, b)
        assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)


def test_captured_prefill(gpu):
    lens = [300, 70]
    cache, want, table = setup(gpu, 25, "bf16", 128, 16, 2, lens)
    q = torch.empty((120, 8, 128), dtype=torch.bfloat16, device=gpu)
    lam, weight = diff_weights(gpu, 5, 8, 128)
    n, cu, t = i32(lens, gpu), i32([0, 100, 120], gpu), i32(table, gpu)

    def both():
        return (kv16.cache16_prefill(cache, q, cu, t, n, return_lse=True) +
                kv16.cache16_diff_prefill(cache, q, lam, cu, t, n, norm_weight=weight, return_lse=True))

    q.normal_()
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for i in range(5):
        q.normal_()
        n.copy_(i32([300 - 13 * i, 70 - 20 * i], gpu))
        ref = both()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, ref):
            assert torch.equal(a, b)


def test_two_streams(gpu):
    """Calls on two streams at once, each with its own workspace, give what they give alone."""
    lens = [3000, 70, 900]
    cache, want, table = setup(gpu, 26, "bf16", 128, 16, 4, lens)
    q = [torch.randn((3, 16, 128), device=gpu).bfloat16() for _ in range(2)]
    t, n = i32(table, gpu), i32(lens, gpu)
    ref = [kv16.cache16_decode(cache, x, t, n) for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(kv16.cache16_decode(cache, q[i], t, n))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, ref[i]) for o in outs[i])


def test_offsets_past_32_bits(gpu):
    """Pages far past 2^32 bytes (and 2^31 elements) of the cache."""
    H, dh, ps = 8, 128, 128
    page = H * dh * ps
    num_pages = (2 ** 32 // 2) // page + 40                               # > 2^31 elements each
    k = torch.empty((num_pages, H, ps, dh), dtype=torch.float16, device=gpu)
    v = torch.empty_like(k)
    cache = kv16.Cache16(k, v)
    n = 300
    ids = [num_pages - 1, 0, num_pages - 7]
    small = kv16.Cache16.allocate(3, H, dh, ps, torch.float16, gpu)
    g = torch.Generator(device=gpu).manual_seed(3)
    kk, vv = (torch.randn((n, H, dh), generator=g, device=gpu).half() for _ in range(2))
    q = torch.randn((n, 2 * H, dh), generator=g, device=gpu).half()
    f = kv16.rope_inv_freq(dh, device=gpu)
    res = []
    for c, t in ((cache, ids), (small, [0, 1, 2])):
        t = i32([t], gpu)
        qq = kv16.cache16_append(c, kk, vv, t, i32([0], gpu), i32([0, n], gpu), inv_freq=f, q=q)
        res.append((qq, kv16.cache16_decode(c, qq[-1:], t, i32([n], gpu)), kv16.cache16_prefill(c, qq, i32([0, n], gpu), t, i32([n], gpu))))
    for a, b in zip(*res):
        assert torch.equal(a, b)
    assert torch.equal(cache.k[ids[2], :, :44], small.k[2, :, :44])


@pytest.mark.parametrize("cu", [[0, 40, 10, 60], [50, 0, 60, 20], [-5, 1000, 3, 60], [60, 40, 20, 0], [2 ** 31 - 1, -2 ** 31, 30, 31]])
def test_row_starts_out_of_order(gpu, cu):
    """Row starts that break the rules stay within the tensors: rows outside the batch and their neighbours keep their
    contents, the cache's pages that no table names too."""
    H, dh, ps, T = 1, 64, 16, 60
    cache = random_cache(gpu, 27, 16, H, dh, ps, "fp16")
    table = i32(np.arange(12).reshape(3, 4), gpu)
    spare = [cache.k[12:].clone(), cache.v[12:].clone()]
    buf = torch.full((T + 20, 2, dh), 7.0, dtype=torch.float16, device=gpu)
    q = torch.randn((T, 2, dh), device=gpu).half()
    k, v = (torch.randn((T, H, dh), device=gpu).half() for _ in range(2))
    starts = i32(cu, gpu)
    kv16.cache16_append(cache, k, v, table, i32([0, 3, 30], gpu), starts, inv_freq=kv16.rope_inv_freq(dh, device=gpu), q=q, q_out=buf[10:-10])
    kv16.cache16_prefill(cache, q, starts, table, i32([64, 20, 5], gpu), out=buf[10:-10])
    kv16.cache16_diff_prefill(cache, q, torch.ones(2, device=gpu), starts, table, i32([64, 20, 5], gpu), out=buf[10:-10])
    torch.cuda.synchronize()
    assert (buf[:10] == 7.0).all() and (buf[-10:] == 7.0).all()
    assert torch.equal(cache.k[12:], spare[0]) and torch.equal(cache.v[12:], spare[1])


def test_empty_caches_tables_and_batches(gpu):
    dh = 64
    q = torch.randn((2, 2, dh), device=gpu).half()
    empty = kv16.Cache16.allocate(0, 1, dh, 16, torch.float16, gpu)
    one = kv16.Cache16.allocate(1, 1, dh, 16, torch.float16, gpu)
    lam = torch.ones(2, device=gpu)
    for cache, table in ((empty, [[0, 1], [2, 3]]), (one, [[], []])):
        t = i32(np.asarray(table, np.int32).reshape(2, -1), gpu)
        n = i32([20, 5], gpu)
        for out, lse in (kv16.cache16_decode(cache, q, t, n, return_lse=True),
                         kv16.cache16_diff_decode(cache, q, lam, t, n, norm_weight=torch.ones(dh, device=gpu), norm_eps=0.0, return_lse=True),
                         kv16.cache16_prefill(cache, q, i32([0, 1, 2], gpu), t, n, return_lse=True),
                         kv16.cache16_diff_prefill(cache, q, lam, i32([0, 1, 2], gpu), t, n, norm_weight=torch.ones(dh, device=gpu), norm_eps=0.0, return_lse=True)):
            assert (out == 0).all() and torch.isneginf(lse).all()
        kv16.cache16_append(cache, q[:, :1], q[:, :1], t, n)
    t = torch.zeros((0, 2), dtype=torch.int32, device=gpu)
    none = torch.empty((0, 2, dh), dtype=torch.float16, device=gpu)
    assert kv16.cache16_decode(one, none, t, i32([], gpu)).shape == (0, 2, dh)
    assert kv16.cache16_prefill(one, none, i32([0], gpu), t, i32([], gpu)).shape == (0, 2, dh)
    assert kv16.cache16_append(one, none[:, :1], none[:, :1], t, i32([], gpu), q=none).shape == (0, 2, dh)
