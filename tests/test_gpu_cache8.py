"""The 8-bit KV cache on the GPU against its oracle in 64 bits: written codes
and scales bit for bit, reads bit for bit, attention within derived bounds."""
import math

import numpy as np
import pytest
import torch

import sphkv_kv8 as kv8
from gpu_helpers import log
from oracle import cache8 as o8

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def i32(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=dev)


def rows_np(t):
    return t.double().cpu().numpy()


def random_cache(dev, seed, num_pages, num_kv, dh, ps, fmt, spread=2.0):
    """A cache of random codes (no e4m3 NaN) and scales over a range of 2^+-spread."""
    rng = np.random.default_rng(seed)
    b = rng.integers(0, 256, (2, num_pages, num_kv, ps, dh)).astype(np.uint8)
    if fmt == "e4m3":
        b[(b & 0x7F) == 0x7F] = 0x7E
    else:
        b[b == 0x80] = 0x81
    sc = 2.0 ** rng.uniform(-spread, spread, (num_pages, num_kv, 2)) * (1 / 100 if fmt == "int8" else 1 / 32)
    k = torch.from_numpy(b[0]).to(dev)
    v = torch.from_numpy(np.ascontiguousarray(b[1].reshape(num_pages, num_kv, ps // 16, 16, dh).swapaxes(3, 4))).to(dev)
    return kv8.Cache8(k, v, torch.from_numpy(sc.astype(np.float32)).to(dev), fmt)


def oracle_of(cache):
    return o8.Cache.from_bytes(cache.k_codes.cpu().numpy(), cache.v_codes.cpu().numpy(), cache.scales.cpu().numpy(),
                               cache.fmt)


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


def same_cache(cache, want, what):
    """Codes (as the values they stand for) and scales equal the oracle's bit for bit."""
    got = oracle_of(cache)
    assert np.array_equal(got.scales, want.scales), f"{what}: scales differ"
    for name in ("k", "v"):
        a, b = getattr(got, name), getattr(want, name)
        assert np.array_equal(a, b, equal_nan=True), f"{what}: {(a != b).sum()} {name} codes differ"


def check_attention(out, lse, want, want_lse, mass, reach, under, dtype, dh, what):
    """|out - want| against the roundings that the operator makes.  A score's sum
    of dh products, its scaling and its exponent in fp32 are off by at most
    delta = 2^-24 ((dh + 16) sum|q k| + 8 |score|) + 2^-21 (|score| is at most
    sum|q k|), which moves a weight by that factor, above and below the
    division.  A weight w_t ~ p_t sv_t is rounded to fp16: by 2^-11 of it, or by
    2^-25, half of the smallest fp16 step.  The largest weight is at least 2^8
    then, so w = 1 is at most 2^-8 max(p sv), and 2^-25 for every token and its
    code moves an output by at most 2^-33 max_t(p_t sv_t) sum_t |code_t|
    (`under`).  The output is rounded once more, by half a step (2^-25 at least
    in fp16)."""
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    delta = 2.0 ** -24 * (dh + 24) * reach + 2.0 ** -21
    tol = (2.0 ** -11 + 2.2 * delta)[..., None] * mass + 2.0 ** -33 * under \
        + torch.finfo(dtype).eps / 2 * np.abs(want) + 2.0 ** -25
    err = np.abs(out - want)
    log(f"  {what}: max err {err.max(initial=0):.3g}, {(err / tol).max(initial=0):.3f} of the bound")
    assert (err <= tol).all(), f"{what}: {(err > tol).sum()} outputs off"
    dead = np.isneginf(want_lse)
    assert np.array_equal(np.isneginf(lse), dead), what
    assert (out[dead] == 0).all(), what
    tol = delta + 2.0 ** -21 * np.abs(want_lse, where=~dead, out=np.zeros_like(want_lse))
    assert (np.abs(np.where(dead, 0, lse) - np.where(dead, 0, want_lse)) <= tol).all(), f"{what}: lse"


# ---- write ---------------------------------------------------------------------

WRITES = [
    # (fmt, dtype, dh, page, num_kv, [(start, new)]): partial first and last pages, empty sequences, one token
    ("int8", "fp16", 128, 16, 8, [(0, 1), (15, 1), (5, 3), (16, 16), (0, 0), (7, 60)]),
    ("e4m3", "bf16", 64, 16, 3, [(0, 33), (31, 2), (16, 0), (3, 13), (0, 16)]),
    ("int8", "fp32", 64, 32, 1, [(33, 64), (0, 31), (31, 1), (32, 32), (1, 7)]),
    ("e4m3", "fp32", 128, 64, 2, [(63, 2), (0, 64), (10, 130), (64, 1)]),
    ("int8", "bf16", 128, 128, 4, [(0, 200), (127, 1), (100, 28), (17, 16)]),
    ("e4m3", "fp16", 128, 32, 8, [(0, 0), (40, 9), (0, 0)]),
    ("int8", "fp16", 64, 64, 5, [(i, 1) for i in range(0, 140, 7)]),
    ("int8", "fp32", 128, 16, 2, [(3, 1)] * 1 + [(0, 5)] * 70),          # more than 64 sequences
    ("e4m3", "bf16", 64, 16, 1, [(i % 23, i % 4) for i in range(5000)]), # more than 64 * 64
]


@pytest.mark.parametrize("fmt, dtype, dh, ps, num_kv, seqs", WRITES)
def test_write(gpu, fmt, dtype, dh, ps, num_kv, seqs):
    rng = np.random.default_rng(3)
    blocks = [-(-(a + m) // ps) for a, m in seqs]
    num_pages = sum(blocks) + 2
    cache = random_cache(gpu, 4, num_pages, num_kv, dh, ps, fmt, spread=6.0)
    want = oracle_of(cache)
    table = tables(5, num_pages, blocks)
    cu = np.cumsum([0] + [m for _, m in seqs])
    T = int(cu[-1])
    x = rng.standard_normal((2, T + 3, num_kv, dh)) * 2.0 ** rng.uniform(-8, 8, (2, T + 3, 1, 1))
    k, v = (torch.from_numpy(a).to(gpu).to(TYPES[dtype]) for a in x)
    k[T:], v[T:] = float("nan"), float("inf")                            # rows behind the last sequence
    log(f"write {fmt} {dtype} dh {dh} page {ps}")
    kv8.cache8_write(cache, k, v, i32(table, gpu), i32([a for a, _ in seqs], gpu), i32(cu, gpu))
    want.write(rows_np(k), rows_np(v), table, [a for a, _ in seqs], cu)
    same_cache(cache, want, "write")


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("ps", [16, 128])
def test_write_token_by_token(gpu, fmt, ps):
    """The form of one token a sequence, growing each page's scales again and again."""
    rng = np.random.default_rng(6)
    n, num_kv, dh = 3, 2, 64
    cache = random_cache(gpu, 7, 12, num_kv, dh, ps, fmt)
    want = oracle_of(cache)
    table = tables(8, 12, [3, 3, 3])
    starts = np.array([0, 9, 20])
    for t in range(20):
        x = rng.standard_normal((2, n, num_kv, dh)) * 2.0 ** (t / 4 + rng.uniform(-3, 1, (2, n, 1, 1)))
        k, v = (torch.from_numpy(a).to(gpu).half() for a in x)
        kv8.cache8_write(cache, k, v, i32(table, gpu), i32(starts + t, gpu))
        want.write(rows_np(k), rows_np(v), table, starts + t)
        same_cache(cache, want, f"token {t}")


@pytest.mark.parametrize("fmt, dtype", [("int8", "fp16"), ("e4m3", "bf16"), ("int8", "fp32"), ("e4m3", "fp32")])
def test_write_special_values(gpu, fmt, dtype):
    """Zeros, NaN, infinities, the type's largest and smallest, ties, -0."""
    dh, num_kv, ps = 64, 2, 16
    t = TYPES[dtype]
    info = torch.finfo(t)
    x = torch.randn(2, 48, num_kv, dh, device=gpu, generator=torch.Generator(gpu).manual_seed(9)).to(t)
    x[0, 0] = 0
    x[0, 1, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), -0.0])
    x[1, :16] = 0                                       # a page of zeros
    x[1, 16:32] = float("nan")                          # a page of NaN
    x[0, 16:32] = float("inf")                          # a page without a finite value
    x[0, 32:] = info.max                                # the largest finite value
    x[1, 32:] = info.smallest_normal
    x[1, 33, 0] = info.tiny / 4                         # a denormal (0 where the type has none)
    grid = torch.arange(dh, device=gpu).float() - dh // 2 + 0.5
    x[0, 2:16, 1] = grid.to(t)                          # ties once the page's largest is 127
    x[0, 2, 1, 0] = 127.0
    cache = random_cache(gpu, 10, 4, num_kv, dh, ps, fmt)
    want = oracle_of(cache)
    table = np.array([[3, 0, 2]], np.int32)
    kv8.cache8_write(cache, x[0], x[1], i32(table, gpu), i32([0], gpu), i32([0, 48], gpu))
    want.write(rows_np(x[0]), rows_np(x[1]), table, [0], [0, 48])
    same_cache(cache, want, "special values")
    assert torch.isfinite(cache.scales).all()


def test_write_strides_and_alignment(gpu):
    """k and v as slices of one fused projection, off 16-byte alignment, and broadcast heads."""
    rng = np.random.default_rng(11)
    num_kv, dh, T = 4, 128, 21
    fused = torch.from_numpy(rng.standard_normal((T, 3 * num_kv * dh + 1))).to(gpu).to(torch.bfloat16)
    views = [fused[:, 1 + i * num_kv * dh:1 + (i + 1) * num_kv * dh].view(T, num_kv, dh) for i in (1, 2)]
    heads_first = [torch.from_numpy(rng.standard_normal((num_kv, T, dh))).to(gpu).half().transpose(0, 1) for _ in range(2)]
    broadcast = [torch.from_numpy(rng.standard_normal((T, 1, dh))).to(gpu).float().expand(T, num_kv, dh) for _ in range(2)]
    for k, v in (views, heads_first, broadcast):
        cache = random_cache(gpu, 12, 4, num_kv, dh, 16, "int8")
        want = oracle_of(cache)
        table = np.array([[1, 3, -5], [0, 9, 2]], np.int32)             # -5 and 9: no such pages
        wide = torch.full((2, 7), 99, dtype=torch.int32, device=gpu)    # rows apart by more than their length
        wide[:, :3] = i32(table, gpu)
        kv8.cache8_write(cache, k, v, wide[:, :3], i32([2, 30], gpu), i32([0, 17, T], gpu))
        want.write(rows_np(k), rows_np(v), table, [2, 30], [0, 17, T])
        same_cache(cache, want, "strides")


def test_write_drops_what_has_no_page(gpu):
    num_kv, dh = 2, 64
    cache = random_cache(gpu, 13, 5, num_kv, dh, 16, "e4m3")
    want = oracle_of(cache)
    k = torch.randn(60, num_kv, dh, device=gpu)
    table = np.array([[0, -1, 4], [1, 2, 3], [-1, -1, -1]], np.int32)
    start, cu = [10, 40, 0], [0, 30, 50, 60]                             # past the table; absent pages
    kv8.cache8_write(cache, k, k, i32(table, gpu), i32(start, gpu), i32(cu, gpu))
    want.write(rows_np(k), rows_np(k), table, start, cu)
    same_cache(cache, want, "absent pages")
    kv8.cache8_write(cache, k[:3], k[:3], i32(table, gpu), i32([-1, 48, 2 ** 31 - 1], gpu))
    same_cache(cache, want, "starts outside the table")
    kv8.cache8_write(cache, k[:0], k[:0], i32(table, gpu), i32([0, 0, 0], gpu), i32([0, 0, 0, 0], gpu))
    kv8.cache8_write(cache, k[:2], k[:2], i32(table, gpu), i32([0, 0, 0], gpu), i32([0, 0, 0, 0], gpu))
    same_cache(cache, want, "no new token")


# ---- read ------------------------------------------------------------------------

@pytest.mark.parametrize("fmt, dtype, dh, ps, num_kv, seqs", [
    ("int8", "fp16", 128, 16, 8, [(0, 1), (15, 2), (0, 0), (3, 100)]),
    ("e4m3", "fp32", 64, 32, 3, [(31, 33), (0, 64), (5, 1)]),
    ("int8", "fp32", 64, 128, 2, [(120, 20), (0, 128), (16, 16)]),
    ("e4m3", "bf16", 128, 64, 1, [(0, 65), (63, 1)] + [(1, 2)] * 70),
])
def test_read(gpu, fmt, dtype, dh, ps, num_kv, seqs):
    blocks = [-(-(a + m) // ps) for a, m in seqs]
    cache = random_cache(gpu, 14, sum(blocks) + 1, num_kv, dh, ps, fmt)
    table = tables(15, sum(blocks) + 1, blocks)
    table[-1, 0] = -1                                                    # an absent page: zeros
    cu = np.cumsum([0] + [m for _, m in seqs])
    T = int(cu[-1])
    k, v = (torch.full((T + 5, num_kv, dh), 7.0, dtype=TYPES[dtype], device=gpu) for _ in range(2))
    got = kv8.cache8_read(cache, i32(table, gpu), i32([a for a, _ in seqs], gpu), i32(cu, gpu), T + 5, TYPES[dtype], k, v)
    assert got[0] is k and got[1] is v
    o = oracle_of(cache)
    for s, (a, m) in enumerate(seqs):
        wk, wv, _ = o.tokens(table, s, a, a + m)
        for t, w in ((k, wk), (v, wv)):                                  # the fp32 product, then one rounding
            w = torch.from_numpy(w.astype(np.float32)).to(TYPES[dtype])
            assert torch.equal(t[cu[s]:cu[s + 1]].cpu(), w), f"sequence {s}"
    assert (k[T:] == 7).all() and (v[T:] == 7).all()


def test_read_one_token_a_sequence(gpu):
    cache = random_cache(gpu, 16, 6, 2, 64, 16, "int8")
    table = tables(17, 6, [2, 2, 2])
    start = [0, 17, 40]                                                  # the last is past its table
    k, v = kv8.cache8_read(cache, i32(table, gpu), i32(start, gpu))
    o = oracle_of(cache)
    for s in range(3):
        wk, wv, _ = o.tokens(table, s, start[s], start[s] + 1)
        assert torch.equal(k[s:s + 1].cpu(), torch.from_numpy(wk.astype(np.float32)).half())
        assert torch.equal(v[s:s + 1].cpu(), torch.from_numpy(wv.astype(np.float32)).half())
    k, v = kv8.cache8_read(cache, i32(table, gpu), i32([-1, -40, 2 ** 31 - 1], gpu))
    assert (k == 0).all() and (v == 0).all()


# ---- decode ------------------------------------------------------------------------

DECODES = [
    # (fmt, dtype, dh, page, num_kv, gqa, lens)
    ("int8", "fp16", 128, 16, 8, 4, [0, 1, 15, 16, 17, 63, 64, 65, 255, 256, 257, 1000]),
    ("e4m3", "bf16", 128, 16, 8, 8, [4097, 1, 700, 0, 33]),
    ("int8", "bf16", 64, 32, 4, 1, [31, 32, 33, 512, 100, 0]),
    ("e4m3", "fp16", 64, 64, 2, 2, [63, 64, 65, 129, 2000]),
    ("int8", "fp16", 128, 128, 1, 16, [127, 128, 129, 1500]),
    ("e4m3", "bf16", 64, 128, 3, 7, [1, 5, 300]),
    ("int8", "bf16", 128, 64, 2, 17, [70, 640, 3]),
    ("e4m3", "fp16", 128, 16, 1, 64, [900, 2]),
    ("int8", "fp16", 64, 16, 2, 33, [50, 0, 1]),
    ("int8", "fp16", 128, 16, 2, 3, [(i * 37) % 200 for i in range(150)]),
    ("e4m3", "bf16", 128, 32, 8, 5, [12000]),
    ("int8", "fp16", 64, 16, 1, 1, [20000, 1]),
    ("e4m3", "fp16", 64, 16, 1, 2, [(i * 7) % 40 for i in range(3000)]),
]


def poison(cache, table, lens):
    """Bytes of every slot behind its sequence's length: NaN codes of e4m3, -128 of int8; scales of pages no token is in: NaN."""
    ps = cache.page_size
    bad = 0x7F if cache.fmt == "e4m3" else 0x80
    used = np.zeros(cache.num_pages, bool)
    kc, vc = cache.k_codes.cpu().numpy(), cache.v_codes.cpu().numpy()
    for s, n in enumerate(lens):
        for blk in range(-(-n // ps)):
            p = int(table[s, blk])
            if not 0 <= p < cache.num_pages:
                continue
            used[p] = True
            for t in range(min(max(n - blk * ps, 0), ps), ps):
                kc[p, :, t] = bad
                vc[p, :, t // 16, :, t % 16] = bad
    kc[~used], vc[~used] = bad, bad
    cache.k_codes.copy_(torch.from_numpy(kc))
    cache.v_codes.copy_(torch.from_numpy(vc))
    cache.scales[torch.from_numpy(~used).to(cache.device)] = float("nan")


def clean(o):
    """An oracle whose poisoned slots hold zeros (attention does not see them)."""
    o.k, o.v, o.scales = (np.nan_to_num(x) for x in (o.k, o.v, o.scales))
    return o


def attention_case(gpu, seed, fmt, dtype, dh, ps, num_kv, gqa, lens, rows, spread=2.0, absent=True):
    blocks = [-(-n // ps) for n in lens]
    num_pages = sum(blocks) + 2
    cache = random_cache(gpu, seed, num_pages, num_kv, dh, ps, fmt, spread)
    table = tables(seed + 1, num_pages, blocks, max(blocks) + 1)
    if absent and len(lens) > 2 and blocks[2] > 1:
        table[2, 1] = -1                                                 # a page that is not there
    if absent and len(lens) > 1 and blocks[-1] > 2:
        table[-1, 0] = num_pages + 7
    poison(cache, table, lens)
    q = torch.randn(rows, num_kv * gqa, dh, device=gpu, generator=torch.Generator(gpu).manual_seed(seed)).to(TYPES[dtype])
    return cache, table, q


@pytest.mark.parametrize("fmt, dtype, dh, ps, num_kv, gqa, lens", DECODES)
def test_decode(gpu, fmt, dtype, dh, ps, num_kv, gqa, lens):
    cache, table, q = attention_case(gpu, 20, fmt, dtype, dh, ps, num_kv, gqa, lens, len(lens))
    log(f"decode {fmt} {dtype} dh {dh} page {ps} gqa {gqa} lens {lens[:12]}")
    out, lse = kv8.cache8_decode(cache, q, i32(table, gpu), i32(lens, gpu), return_lse=True)
    want = clean(oracle_of(cache)).attend(rows_np(q), table, lens)
    check_attention(out, lse, *want, TYPES[dtype], dh, "decode")
    again = kv8.cache8_decode(cache, q, i32(table, gpu), i32(lens, gpu))
    assert torch.equal(again, out)                                       # the same bits each time


def test_decode_lengths_beyond_the_table(gpu):
    cache, table, q = attention_case(gpu, 22, "int8", "fp16", 64, 16, 2, 4, [48, 48, 48], 3, absent=False)
    table = table[:, :3]
    lens = [49, 2 ** 31 - 1, -3]
    out, lse = kv8.cache8_decode(cache, q, i32(table, gpu), i32(lens, gpu), return_lse=True)
    want = clean(oracle_of(cache)).attend(rows_np(q), table, [48, 48, 0])
    check_attention(out, lse, *want, torch.float16, 64, "beyond the table")


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_decode_scales_far_apart(gpu, fmt):
    """Value scales from 2^-60 to 2^40 in one sequence: tokens of small values and much weight next to large
    ones of little, and pages that hold nothing but zeros."""
    lens, dh, ps = [400, 300], 64, 16
    cache, table, q = attention_case(gpu, 24, fmt, "bf16", dh, ps, 2, 4, lens, 2, absent=False)
    g = np.random.default_rng(25)
    sc = cache.scales.cpu().numpy()
    sc[..., 1] = 2.0 ** g.uniform(-60, 40, sc.shape[:2])
    sc[table[0, :20], 0, 1] = 2.0 ** -60                                 # one head: all but a few pages tiny
    cache.scales.copy_(torch.from_numpy(sc))
    p = int(table[1, 3])
    cache.v_codes[p] = 0
    out, lse = kv8.cache8_decode(cache, q, i32(table, gpu), i32(lens, gpu), return_lse=True)
    want = oracle_of(cache)
    want = clean(want).attend(rows_np(q), table, lens)
    check_attention(out, lse, *want, torch.bfloat16, dh, "scales far apart")


def test_decode_peaked_and_flat_softmax(gpu):
    """Scores of +-1e3 (one token takes all), equal scores, and a large sm_scale."""
    lens, dh = [700, 64, 129], 128
    cache, table, q = attention_case(gpu, 26, "int8", "fp16", dh, 16, 2, 4, lens, 3, absent=False)
    q[1] = 0
    for sm in (1.0, 1e-6, 30.0):
        out, lse = kv8.cache8_decode(cache, q, i32(table, gpu), i32(lens, gpu), sm, return_lse=True)
        want = clean(oracle_of(cache)).attend(rows_np(q), table, lens, sm_scale=sm)
        if sm < 30:
            check_attention(out, lse, *want, torch.float16, dh, f"sm_scale {sm}")
        else:                # scores pass 1e3: their fp32 errors move weights by whole factors.  The lse is off by a
            # score's error (1e-5 of sum|q k| covers (dh + 24) 2^-24) and, as the row of zero queries shows, whose
            # sum|q k| is 0 and lse ln 64, by the fp32 roundings of the lse itself: up to 8 half steps of 2^-24 of it
            tol = 1e-5 * want[3] + 2.0 ** -21 * np.abs(want[1])
            assert torch.isfinite(out).all() and (np.abs(rows_np(lse) - want[1]) <= tol).all()


@pytest.mark.parametrize("dh", [64, 128])
def test_scores_of_any_size(gpu, dh):
    """Scores up to 2^36, whose fp32 spacing is 2^13: the largest takes all, and its weight is exactly its own."""
    n, ps = 100, 16
    k = torch.zeros(8, 1, ps, dh, dtype=torch.uint8, device=gpu)
    table = tables(70, 8, [7])
    for t in range(n):
        k[int(table[0, t // ps]), 0, t % ps, 0] = t + 1
    cache = random_cache(gpu, 71, 8, 1, dh, ps, "int8")
    cache.k_codes.copy_(k)
    cache.scales[..., 0] = 512.0
    q = torch.zeros(3, 2, dh, dtype=torch.float16, device=gpu)
    q[:, 0, 0], q[:, 1, 0] = 65504.0, -65504.0
    o = oracle_of(cache)
    _, v, _ = o.tokens(table, 0, 0, n)
    td, lens = i32(table, gpu), i32([n], gpu)
    outs = [kv8.cache8_decode(cache, q[:1], td, lens, return_lse=True),
            kv8.cache8_prefill(cache, q, i32([0, 3], gpu), td, lens, False, return_lse=True)]
    for out, lse in outs:
        for row in range(out.shape[0]):
            for head, token in ((0, n - 1), (1, 0)):
                want = v[token, 0]
                got = out[row, head].double().cpu().numpy()
                # one weight: rounded to fp16 in the product and not in the sum, and the output's own rounding
                assert (np.abs(got - want) <= 2.0 ** -10 * np.abs(want) + 2.0 ** -25).all()
                score = (1 if head == 0 else -1) * 65504.0 * 512.0 * (token + 1) / math.sqrt(dh)
                assert abs(lse[row, head].item() - score) <= 2.0 ** -21 * abs(score)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dh", [64, 128])
def test_scores_whose_step_is_sixteen(gpu, dh, dtype):
    """Exponents of two from 2^27 to 2^28, where 8 below a number is a tie between it and 16 below: the largest takes all."""
    n, ps, heads = 100, 16, 16
    table = tables(70, 8, [7])
    cache = random_cache(gpu, 71, 8, 1, dh, ps, "int8")
    cache.k_codes.zero_()
    for t in range(n):
        cache.k_codes[int(table[0, t // ps]), 0, t % ps, 0] = t + 1
    cache.scales[..., 0] = 512.0
    q = torch.zeros(1, heads, dh, dtype=TYPES[dtype], device=gpu)
    q[0, :, 0] = torch.linspace(2.0 ** 27.1, 2.0 ** 27.9, heads) * (math.sqrt(dh) * math.log(2) / 512 / n)
    score = rows_np(q)[0, :, 0] * 512 * n / math.sqrt(dh)
    assert (score / math.log(2) > 2 ** 27).all() and (score / math.log(2) < 2 ** 28).all()
    _, v, _ = oracle_of(cache).tokens(table, 0, 0, n)
    td, lens = i32(table, gpu), i32([n], gpu)
    for out, lse in (kv8.cache8_decode(cache, q, td, lens, return_lse=True),
                     kv8.cache8_prefill(cache, q, i32([0, 1], gpu), td, lens, return_lse=True)):
        got = rows_np(out)[0]
        # one weight, rounded in the product and not in the sum (2^-11), and the output's own rounding
        tol = 2.0 ** -11 + torch.finfo(TYPES[dtype]).eps / 2 * 1.001
        assert (np.abs(got - v[n - 1, 0]) <= tol * np.abs(v[n - 1, 0]) + 2.0 ** -24).all()
        assert (np.abs(rows_np(lse)[0] - score) <= 2.0 ** -21 * score).all()


def test_empty_caches_and_tables(gpu):
    """A cache of no page, tables of no block, no sequence at all: zeros and -inf, and nothing written."""
    q = torch.randn(2, 4, 64, device=gpu).half()
    cu = i32([0, 1, 2], gpu)
    for cache, table in ((kv8.Cache8.allocate(0, 2, 64, 16, "int8", gpu), i32([[0, 1], [5, -1]], gpu)),
                         (random_cache(gpu, 72, 3, 2, 64, 16, "int8"), torch.empty(2, 0, dtype=torch.int32, device=gpu))):
        lens = i32([5, 20], gpu)
        before = cache.k_codes.clone()
        kv8.cache8_write(cache, q[:, :2], q[:, :2], table, i32([0, 3], gpu))
        assert torch.equal(cache.k_codes, before)
        k, v = kv8.cache8_read(cache, table, i32([0, 3], gpu))
        assert (k == 0).all() and (v == 0).all()
        for out, lse in (kv8.cache8_decode(cache, q, table, lens, return_lse=True),
                         kv8.cache8_prefill(cache, q, cu, table, lens, return_lse=True)):
            assert (out == 0).all() and torch.isneginf(lse).all()
    none = torch.empty(0, 2, dtype=torch.int32, device=gpu)
    assert kv8.cache8_decode(cache, q[:0], none, i32([], gpu)).shape == (0, 4, 64)
    assert kv8.cache8_prefill(cache, q[:0], i32([0], gpu), none, i32([], gpu)).shape == (0, 4, 64)
    kv8.cache8_write(cache, q[:0, :2], q[:0, :2], none, i32([], gpu))
    assert kv8.cache8_read(cache, none, i32([], gpu))[0].shape == (0, 2, 64)


def test_tokens_never_written(gpu):
    """A new cache holds zeros under scales of zero: they count as tokens of zeros."""
    cache = kv8.Cache8.allocate(3, 2, 64, 16, "e4m3", gpu)
    q = torch.randn(4, 4, 64, device=gpu).bfloat16()
    table, lens = i32([[2, 0]], gpu), i32([20], gpu)
    for out, lse in (kv8.cache8_decode(cache, q[:1], table, lens, return_lse=True),
                     kv8.cache8_prefill(cache, q, i32([0, 4], gpu), table, lens, False, return_lse=True)):
        assert (out == 0).all()
        # Scores of zero, ln 20.  A value scale below 2^-60 counts as that: the reference is -60 - 8 and the sum
        # 20 * 2^68, whose log2 is 72.3, with an fp32 spacing of 2^-17: one spacing for the logarithm (1 ulp) and
        # half of one for the addition, times ln 2
        assert (lse - math.log(20)).abs().max().item() <= 1.5 * 2.0 ** -17 * math.log(2)


def test_decode_nan_query_stays_in_its_row(gpu):
    lens = [300, 300]
    cache, table, q = attention_case(gpu, 28, "e4m3", "bf16", 128, 16, 2, 4, lens, 2, absent=False)
    clean_out = kv8.cache8_decode(cache, q, i32(table, gpu), i32(lens, gpu))
    q2 = q.clone()
    q2[0, 5, 17] = float("nan")
    out = kv8.cache8_decode(cache, q2, i32(table, gpu), i32(lens, gpu))
    assert torch.isnan(out[0, 5]).all()
    out[0, 5] = clean_out[0, 5]
    assert torch.equal(out, clean_out)


def test_decode_query_strides(gpu):
    lens, H, gqa, dh = [100, 333, 20], 2, 4, 128
    cache, table, q = attention_case(gpu, 30, "int8", "bf16", dh, 16, H, gqa, lens, 3)
    want = kv8.cache8_decode(cache, q, i32(table, gpu), i32(lens, gpu))
    fused = torch.zeros(3, H * gqa * dh + 3 + 64, dtype=q.dtype, device=gpu)
    a = fused[:, 3:3 + H * gqa * dh].view(3, H * gqa, dh)
    a.copy_(q)
    b = q.transpose(0, 1).contiguous().transpose(0, 1)
    for x in (a, b):
        assert torch.equal(kv8.cache8_decode(cache, x, i32(table, gpu), i32(lens, gpu)), want)


def test_decode_given_outputs_and_workspace(gpu):
    lens = [100, 2000]
    cache, table, q = attention_case(gpu, 32, "int8", "fp16", 64, 32, 2, 2, lens, 2, absent=False)
    t, n = i32(table, gpu), i32(lens, gpu)
    want, wl = kv8.cache8_decode(cache, q, t, n, return_lse=True)
    ws = torch.full((kv8.decode_workspace_bytes(cache, 2, 2) + 16,), 0xFF, dtype=torch.uint8, device=gpu)
    out, lse = torch.empty_like(q), torch.empty(2, 4, device=gpu)
    got = kv8.cache8_decode(cache, q, t, n, out=out, lse=lse, workspace=ws)
    assert got is out and torch.equal(out, want) and torch.equal(lse, wl)
    with pytest.raises(ValueError, match="out must be"):
        kv8.cache8_decode(cache, q, t, n, out=out[:1])
    with pytest.raises(ValueError, match="one row per sequence"):
        kv8.cache8_decode(cache, q[:1], t, n)
    with pytest.raises(TypeError, match="fp16 or bf16"):
        kv8.cache8_decode(cache, q.float(), t, n)
    with pytest.raises(ValueError, match="num_kv \\* gqa"):
        kv8.cache8_decode(cache, q[:, :3], t, n)
    with pytest.raises(TypeError, match="torch.int32"):
        kv8.cache8_decode(cache, q, t, n.long())
    with pytest.raises(ValueError, match="must be contiguous"):
        kv8.cache8_decode(cache, q.transpose(1, 2).contiguous().transpose(1, 2), t, n)
    with pytest.raises(ValueError, match="GPU device"):
        kv8.cache8_decode(cache, q.cpu(), t, n)


# ---- prefill -----------------------------------------------------------------------

PREFILLS = [
    # (fmt, dtype, dh, page, num_kv, gqa, [(len, new)], causal)
    ("int8", "fp16", 128, 16, 2, 4, [(200, 200), (0, 0), (65, 1), (300, 37), (16, 16)], True),
    ("e4m3", "bf16", 128, 64, 2, 8, [(1000, 5), (64, 64), (129, 128)], True),
    ("int8", "bf16", 64, 32, 4, 1, [(500, 260), (33, 33), (70, 3)], True),
    ("e4m3", "fp16", 64, 16, 1, 7, [(100, 50), (257, 256), (3, 3)], True),
    ("int8", "fp16", 128, 128, 1, 33, [(140, 20), (9, 9)], True),
    ("e4m3", "bf16", 64, 128, 1, 64, [(300, 9), (5, 4)], False),
    ("int8", "fp16", 128, 16, 2, 3, [(150, 50), (0, 4), (64, 64)], False),
    ("int8", "bf16", 128, 16, 2, 2, [(5, 9), (30, 30), (-4, 3), (17, 20)], True),      # more rows than tokens
    ("e4m3", "fp16", 128, 32, 1, 4, [(3 * i, i) for i in range(70)], True),
    ("int8", "fp16", 128, 16, 1, 4, [(6000, 3), (4000, 24)], True),                    # few rows, many keys
    ("e4m3", "bf16", 128, 16, 1, 4, [(3000, 100)], True),                              # split, more rows than a tile
    ("int8", "bf16", 64, 16, 1, 4, [(2500, 20), (40, 40)], True),
    ("e4m3", "fp16", 128, 64, 8, 4, [(1100, 1100)], True),                             # whole tiles, no split
]


@pytest.mark.parametrize("fmt, dtype, dh, ps, num_kv, gqa, seqs, causal", PREFILLS)
def test_prefill(gpu, fmt, dtype, dh, ps, num_kv, gqa, seqs, causal):
    lens, new = [max(a, 0) for a, _ in seqs], [m for _, m in seqs]
    cu = np.cumsum([0] + new)
    T = int(cu[-1])
    cache, table, q = attention_case(gpu, 40, fmt, dtype, dh, ps, num_kv, gqa, lens, T + 3)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=gpu)
    lse = torch.full(q.shape[:2], 7.0, device=gpu)
    log(f"prefill {fmt} {dtype} dh {dh} page {ps} gqa {gqa} {seqs[:5]} causal {causal}")
    kv8.cache8_prefill(cache, q, i32(cu, gpu), i32(table, gpu), i32([a for a, _ in seqs], gpu), causal, out=out, lse=lse)
    assert (out[T:] == 7).all() and (lse[T:] == 7).all()
    want = clean(oracle_of(cache)).attend(rows_np(q[:T]), table, lens, cu, causal)
    check_attention(out[:T], lse[:T], *want, TYPES[dtype], dh, "prefill")
    again = kv8.cache8_prefill(cache, q, i32(cu, gpu), i32(table, gpu), i32([a for a, _ in seqs], gpu), causal)
    assert torch.equal(again[:T], out[:T])


def test_prefill_of_one_row_each_is_decode(gpu):
    lens = [64, 1, 700, 129]
    cache, table, q = attention_case(gpu, 42, "int8", "bf16", 128, 16, 2, 4, lens, 4)
    a = kv8.cache8_prefill(cache, q, i32(range(5), gpu), i32(table, gpu), i32(lens, gpu), return_lse=True)
    want = clean(oracle_of(cache)).attend(rows_np(q), table, lens)
    check_attention(*a, *want, torch.bfloat16, 128, "one row each")


def test_prefill_rows_do_not_see_later_tokens(gpu):
    """Whatever later tokens hold, e4m3 NaN codes among them, a causal row's output is the same."""
    cache, table, q = attention_case(gpu, 44, "int8", "fp16", 128, 16, 2, 4, [400], 400)
    t, cu, n = i32(table, gpu), i32([0, 400], gpu), i32([400], gpu)
    want = kv8.cache8_prefill(cache, q, cu, t, n)
    cache.k_codes[int(table[0, 20])] = 127
    cache.v_codes[int(table[0, 20])] = 127
    got = kv8.cache8_prefill(cache, q, cu, t, n)
    assert torch.equal(got[:320], want[:320]) and not torch.equal(got[320:], want[320:])


# ---- together ------------------------------------------------------------------------

@pytest.mark.parametrize("fmt, dtype, dh, ps", [("int8", "fp16", 128, 16), ("e4m3", "bf16", 64, 64)])
def test_prompts_then_decode_steps(gpu, fmt, dtype, dh, ps):
    """A batch's prompts in two chunks, then decode steps: each call's output is that of the cache as the
    oracle has it, and near the attention over the keys and values as they came."""
    rng = np.random.default_rng(50)
    n, num_kv, gqa, steps = 3, 2, 4, 20
    chunks = [[37, 64, 1], [50, 3, 0]]
    total = [sum(c[s] for c in chunks) + steps for s in range(n)]
    blocks = [-(-x // ps) for x in total]
    cache = kv8.Cache8.allocate(sum(blocks) + 1, num_kv, dh, ps, fmt, gpu)
    want = oracle_of(cache)
    table = tables(51, cache.num_pages, blocks)
    td = i32(table, gpu)
    held = np.zeros(n, np.int64)
    seen = [[[], []] for _ in range(n)]
    for call in chunks + [[1] * n] * steps:
        cu = np.cumsum([0] + call)
        T = int(cu[-1])
        k, v = (torch.from_numpy(rng.standard_normal((T, num_kv, dh))).to(gpu).to(TYPES[dtype]) for _ in range(2))
        q = torch.from_numpy(rng.standard_normal((T, num_kv * gqa, dh))).to(gpu).to(TYPES[dtype])
        one = call == [1] * n
        start, lens = i32(held, gpu), i32(held + call, gpu)
        kv8.cache8_write(cache, k, v, td, start, None if one else i32(cu, gpu))
        want.write(rows_np(k), rows_np(v), table, held, cu)
        if one:
            out, lse = kv8.cache8_decode(cache, q, td, lens, return_lse=True)
        else:
            out, lse = kv8.cache8_prefill(cache, q, i32(cu, gpu), td, lens, return_lse=True)
        res = want.attend(rows_np(q), table, held + call, cu)
        check_attention(out, lse, *res, TYPES[dtype], dh, f"call {call}")
        for s in range(n):
            for i, x in enumerate((k, v)):
                seen[s][i].append(rows_np(x)[cu[s]:cu[s + 1]])
        held += call
    same_cache(cache, want, "after the steps")
    k, v = kv8.cache8_read(cache, td, i32(np.zeros(n), gpu), i32(np.cumsum([0] + list(held)), gpu), int(held.sum()),
                           torch.float32)
    for i, got in enumerate((k, v)):
        x = np.concatenate([np.concatenate(seen[s][i]) for s in range(n)])
        rel = np.linalg.norm(rows_np(got) - x) / np.linalg.norm(x)
        # int8: half a code of amax / 127 (Gaussian rows: amax about 4) and a rounding per growth; e4m3: 2^-4 of a value
        assert rel < (0.03 if fmt == "int8" else 0.05)


def test_captured_step_follows_its_tensors(gpu):
    """A captured write + decode replayed with other tokens, starts and lengths, eager work in between."""
    rng = np.random.default_rng(52)
    n, num_kv, gqa, dh, ps = 4, 2, 4, 128, 16
    cache = random_cache(gpu, 53, 40, num_kv, dh, ps, "int8")
    table = tables(54, 40, [9] * n)
    td = i32(table, gpu)
    held = np.array([0, 15, 60, 100])
    start, lens = i32(held, gpu), i32(held + 1, gpu)
    k, v = (torch.zeros(n, num_kv, dh, dtype=torch.float16, device=gpu) for _ in range(2))
    q = torch.zeros(n, num_kv * gqa, dh, dtype=torch.float16, device=gpu)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):                                        # warm up off the default stream
        kv8.cache8_write(cache, k, v, td, start)
        kv8.cache8_decode(cache, q, td, lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv8.cache8_write(cache, k, v, td, start)
        out = kv8.cache8_decode(cache, q, td, lens)
        start.add_(1)
        lens.add_(1)
    eager = kv8.Cache8(cache.k_codes.clone(), cache.v_codes.clone(), cache.scales.clone(), "int8")
    for step in range(20):
        for t in (k, v, q):
            t.copy_(torch.from_numpy(rng.standard_normal(tuple(t.shape))))
        s0, l0 = start.clone(), lens.clone()
        kv8.cache8_write(eager, k, v, td, s0)
        want = kv8.cache8_decode(eager, q, td, l0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {step}"
        assert torch.equal(cache.scales, eager.scales) and torch.equal(cache.k_codes, eager.k_codes)
        assert torch.equal(cache.v_codes, eager.v_codes)
    assert start.tolist() == [x + 20 for x in held]


def test_captured_prefill(gpu):
    seqs = [(200, 60), (90, 90), (33, 1)]
    cu = i32(np.cumsum([0] + [m for _, m in seqs]), gpu)
    cache, table, q = attention_case(gpu, 55, "e4m3", "bf16", 128, 16, 2, 4, [a for a, _ in seqs], 151)
    td, lens = i32(table, gpu), i32([a for a, _ in seqs], gpu)
    kv8.cache8_prefill(cache, q, cu, td, lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = kv8.cache8_prefill(cache, q, cu, td, lens)
    for i in range(4):
        q.copy_(torch.randn(q.shape, device=gpu))
        lens.copy_(i32([200 - 16 * i, 90 - i, 33], gpu))
        want = kv8.cache8_prefill(cache, q, cu, td, lens)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {i}"


def test_two_streams(gpu):
    """Two caches used at once on two streams: each call has a workspace of its own."""
    cases = [attention_case(gpu, 60 + i, "int8", "fp16", 128, 16, 8, 4, [3000 + 500 * i, 50], 2) for i in range(2)]
    args = [(c, q, i32(t, gpu), i32([3000 + 500 * i, 50], gpu)) for i, (c, t, q) in enumerate(cases)]
    want = [kv8.cache8_decode(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(kv8.cache8_decode(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_offsets_past_32_bits(gpu):
    """Pages whose codes lie past 2^32 bytes: written, read and attended."""
    num_pages, num_kv, dh, ps = 40000, 8, 128, 128                       # 5.2 GB of keys, as much of values
    cache = kv8.Cache8(torch.empty((num_pages, num_kv, ps, dh), dtype=torch.uint8, device=gpu),
                       torch.empty((num_pages, num_kv, ps // 16, dh, 16), dtype=torch.uint8, device=gpu),
                       torch.empty((num_pages, num_kv, 2), dtype=torch.float32, device=gpu), "int8")
    low = kv8.Cache8.allocate(4, num_kv, dh, ps, "int8", gpu)
    pages = [num_pages - 1, 33000, num_pages - 3]
    t_far, t_low = i32([pages], gpu), i32([[0, 1, 2]], gpu)
    k, v = (torch.randn(300, num_kv, dh, device=gpu).half() for _ in range(2))
    q = torch.randn(300, num_kv * 4, dh, device=gpu).half()
    zero, cu, n = i32([0], gpu), i32([0, 300], gpu), i32([300], gpu)
    for c, t in ((cache, t_far), (low, t_low)):
        kv8.cache8_write(c, k, v, t, zero, cu)
    assert torch.equal(cache.scales[pages], low.scales[:3])
    for a, b in ((kv8.cache8_read(cache, t_far, zero, cu, 300), kv8.cache8_read(low, t_low, zero, cu, 300)),):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(kv8.cache8_decode(cache, q[:1], t_far, n), kv8.cache8_decode(low, q[:1], t_low, n))
    assert torch.equal(kv8.cache8_prefill(cache, q, cu, t_far, n), kv8.cache8_prefill(low, q, cu, t_low, n))


# ---- weights of the second product -------------------------------------------------------

def check_residual(out, want, mass, reach, under, dtype, dh, n, what):
    """check_attention's bound for weights held as two fp16 numbers: a weight is off by 2^-22 of it (the second
    number holds what the first leaves out, to 2^-11 of that) or by half of the smallest fp16 step.  The products
    are summed in fp32: n of them in each of two numbers' sums, of which a partial sum is at most the mass, and 64
    more steps (rescales, joins of waves, splits and workgroups, the division), each by at most 2^-24 of it."""
    out = out.double().cpu().numpy()
    delta = 2.0 ** -24 * (dh + 24) * reach + 2.0 ** -21
    tol = (2.0 ** -22 + 2.2 * delta + 2.0 ** -24 * (2 * n + 64))[..., None] * mass + 2.0 ** -33 * under \
        + torch.finfo(dtype).eps / 2 * np.abs(want) + 2.0 ** -25
    err = np.abs(out - want)
    log(f"  {what}: max err {err.max():.3g}, {(err / tol).max():.3f} of the bound")
    assert (err <= tol).all(), f"{what}: {(err > tol).sum()} of {err.size} outputs off"


def cancelling_cache(gpu, seed, fmt, dh, num_kv, lens):
    """Values of +-1 and 2, in some dims of random signs: outputs far below sum p|v| that show a weight's rounding."""
    ps = 16
    cache, table, _ = attention_case(gpu, seed, fmt, "fp16", dh, ps, num_kv, 1, lens, len(lens), spread=0.5, absent=False)
    codes = {"int8": [1, 2, 255, 254], "e4m3": [0x38, 0x40, 0xB8, 0xC0]}[fmt]
    g = np.random.default_rng(seed)
    cache.v_codes.copy_(torch.from_numpy(np.array(codes, np.uint8)[g.integers(0, 4, tuple(cache.v_codes.shape))]))
    cache.scales[..., 0] = 1 / 128 if fmt == "int8" else 1 / 512          # small scores, whose own errors stay below
    cache.scales[..., 1] = 1 / 64
    return cache, table


@pytest.mark.parametrize("fmt, dtype, dh, num_kv, gqa", [
    ("int8", "fp16", 128, 2, 1), ("e4m3", "fp16", 64, 2, 8), ("int8", "bf16", 128, 1, 4),
    ("int8", "fp16", 128, 2, 9), ("e4m3", "fp16", 128, 1, 16), ("int8", "fp16", 64, 1, 33), ("e4m3", "bf16", 64, 1, 64),
    ("int8", "bf16", 128, 2, 16),
])
def test_decode_weights_hold_22_bits(gpu, fmt, dtype, dh, num_kv, gqa):
    lens = [16, 5, 33, 2, 64, 90]
    cache, table = cancelling_cache(gpu, 80, fmt, dh, num_kv, lens)
    q = (torch.randn(6, num_kv * gqa, dh, device=gpu, generator=torch.Generator(gpu).manual_seed(81)) / 8).to(TYPES[dtype])
    out = kv8.cache8_decode(cache, q, i32(table, gpu), i32(lens, gpu))
    want, _, *bounds = clean(oracle_of(cache)).attend(rows_np(q), table, lens)
    check_residual(out, want, *bounds, TYPES[dtype], dh, np.array(lens)[:, None], f"decode gqa {gqa}")


@pytest.mark.parametrize("fmt, dh, num_kv, gqa, new", [
    ("int8", 128, 2, 4, [16, 5, 33, 1, 64, 90]),          # a row tile of 256, unsplit
    ("e4m3", 128, 1, 8, [1, 2, 3, 1, 4, 5]),              # few rows: two groups of waves take turns
    ("e4m3", 64, 2, 2, [16, 5, 33, 2, 64, 90]),
    ("int8", 64, 1, 33, [2, 5, 1, 2, 3, 1]),
])
def test_prefill_fp16_weights_hold_22_bits(gpu, fmt, dh, num_kv, gqa, new):
    lens = [16, 5, 33, 2, 64, 90]
    cu = np.cumsum([0] + new)
    cache, table = cancelling_cache(gpu, 82, fmt, dh, num_kv, lens)
    q = (torch.randn(int(cu[-1]), num_kv * gqa, dh, device=gpu, generator=torch.Generator(gpu).manual_seed(83)) / 8).half()
    out = kv8.cache8_prefill(cache, q, i32(cu, gpu), i32(table, gpu), i32(lens, gpu))
    want, _, *bounds = clean(oracle_of(cache)).attend(rows_np(q), table, lens, cu)
    check_residual(out, want, *bounds, torch.float16, dh, np.repeat(lens, new)[:, None], f"prefill gqa {gqa}")


# ---- the cache's own tensors -------------------------------------------------------------

def test_calls_follow_the_tensors_storage(gpu):
    """Storage that a caller puts under the cache's tensors is what the next call reads and writes."""
    lens = [40, 17]
    cache, table, q = attention_case(gpu, 84, "int8", "fp16", 64, 16, 2, 2, lens, 2, absent=False)
    other, _, _ = attention_case(gpu, 85, "int8", "fp16", 64, 16, 2, 2, lens, 2, absent=False)
    t, n = i32(table, gpu), i32(lens, gpu)
    first, second = kv8.cache8_decode(cache, q, t, n), kv8.cache8_decode(other, q, t, n)
    assert not torch.equal(first, second)
    held = [x.data for x in (cache.k_codes, cache.v_codes, cache.scales)]
    before = [x.clone() for x in held]
    cache.k_codes.data, cache.v_codes.data, cache.scales.data = (x.clone() for x in (other.k_codes, other.v_codes, other.scales))
    assert torch.equal(kv8.cache8_decode(cache, q, t, n), second)
    k = torch.randn(2, 2, 64, device=gpu).half()
    for c in (cache, other):
        kv8.cache8_write(c, k, k, t, i32([0, 0], gpu))
    pairs = [(cache.k_codes, other.k_codes), (cache.v_codes, other.v_codes), (cache.scales, other.scales), *zip(held, before)]
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in pairs)     # (by bytes: poisoned scales are NaN)


# ---- decode beyond one tile a wave -------------------------------------------------------

LONG_DECODES = [
    # (fmt, dtype, dh, page, num_kv, gqa, lens)
    ("int8", "fp16", 128, 16, 1, 64, [40000, 777, 3]),
    ("e4m3", "bf16", 128, 64, 8, 8, [30000, 5000, 70]),
    ("e4m3", "fp16", 64, 32, 8, 1, [30000, 5000, 0, 130]),
    ("int8", "bf16", 64, 16, 8, 7, [40000, 9000, 1]),
    ("int8", "fp16", 128, 128, 4, 12, [50000, 300, 20000]),
]


def decode_shape(cache, lens, gqa):
    """(workgroups, tiles of each, all tiles): the workspace has two partials a workgroup; its four waves take turns."""
    groups = kv8.decode_workspace_bytes(cache, 0, gqa) // (8 * (32 + min(gqa, 16) * cache.dh))
    tiles = sum(-(-n // 64) for n in lens) * cache.num_kv * (-(-gqa // 16))
    return groups, 4 * -(-tiles // (4 * groups)), tiles


@pytest.mark.parametrize("fmt, dtype, dh, ps, num_kv, gqa, lens", LONG_DECODES)
def test_decode_many_tiles_a_wave(gpu, fmt, dtype, dh, ps, num_kv, gqa, lens):
    """Waves that take several tiles of a pair: the next tile's loads, page ids looked up ahead, a reference that
    moves with sums in hand, lengths and absent pages in later tiles.  Even heads have small queries, whose flat
    softmax shows a single wrong tile; odd ones large queries, whose scores keep rising."""
    cache, table, q = attention_case(gpu, 90, fmt, dtype, dh, ps, num_kv, gqa, lens, len(lens))
    table[0, 5:lens[0] // ps:37] = -1                                    # absent pages all along the longest
    table[0, lens[0] // ps // 2] = cache.num_pages + 3
    table[0, (lens[0] - 1) // ps] = -1                                   # and its last one
    size = torch.tensor([1 / 16, 4.0], device=gpu).repeat(num_kv * gqa)[:num_kv * gqa]
    q = (q.float() * size[None, :, None]).to(q.dtype)
    groups, per, tiles = decode_shape(cache, lens, gqa)
    assert groups in (512, 768) and per >= 8 and tiles > 4 * groups      # two tiles a wave and more
    out, lse = kv8.cache8_decode(cache, q, i32(table, gpu), i32(lens, gpu), return_lse=True)
    o = clean(oracle_of(cache))
    want = o.attend(rows_np(q), table, lens)
    check_attention(out, lse, *want, TYPES[dtype], dh, "decode")
    # sums: the tokens of a wave, then the partials of a pair
    pair = -(-max(lens) // 64)
    check_residual(out, want[0], *want[2:], TYPES[dtype], dh, np.array([[per // 4 * 64 + pair // per + 2]]), "decode")
    assert torch.equal(kv8.cache8_decode(cache, q, i32(table, gpu), i32(lens, gpu)), out)
    # the reference moves by a rise of 2^4 and more: there is one between tiles of the same wave
    head = min(1, gqa - 1) if num_kv == 1 or gqa > 1 else 1              # a head of large queries
    k, _, present = o.tokens(table, 0, 0, lens[0])
    x = k[:, head // gqa] @ rows_np(q)[0, head] / math.sqrt(dh) * math.log2(math.e)
    sv = np.repeat(o.scales[np.maximum(np.where(table[0] < cache.num_pages, table[0], 0), 0), head // gqa, 1], ps)[:lens[0]]
    x = np.where(present, x + np.log2(np.where(present, sv, 1)), -np.inf)
    x = np.pad(x, (0, -lens[0] % 64), constant_values=-np.inf).reshape(-1, 64).max(1)
    first = (head // gqa) * (-(-gqa // 16)) * pair                       # the pair's first tile among all
    t = np.arange(pair - 4)
    same = (first + t) // per == (first + t + 4) // per
    assert ((x[4:] > x[:-4] + 4) & np.isfinite(x[:-4]) & same).sum() > 3


@pytest.mark.parametrize("fmt, dtype, dh", [("int8", "fp16", 128), ("e4m3", "bf16", 64)])
def test_decode_one_long_among_many_short(gpu, fmt, dtype, dh):
    """One wave joins all partials of a long pair where there are 128 pairs and more."""
    lens = [30000] + [(i * 7) % 50 for i in range(69)]
    num_kv, gqa = 2, 4
    cache, table, q = attention_case(gpu, 92, fmt, dtype, dh, 16, num_kv, gqa, lens, len(lens))
    _, per, _ = decode_shape(cache, lens, gqa)
    assert len(lens) * num_kv >= 128 and 30000 // 64 // per > 100        # partials of the long pair
    q[:, ::2] /= 16
    out, lse = kv8.cache8_decode(cache, q, i32(table, gpu), i32(lens, gpu), return_lse=True)
    want = clean(oracle_of(cache)).attend(rows_np(q), table, lens)
    check_attention(out, lse, *want, TYPES[dtype], dh, "one long")
    check_residual(out, want[0], *want[2:], TYPES[dtype], dh, np.array([[64 + 469 // per + 2]]), "one long")


# ---- masks inside a tile, row starts that are none ---------------------------------------

@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dh", [64, 128])
def test_prefill_mask_inside_a_tile(gpu, fmt, dh):
    """A page from the middle of a tile of 64 tokens takes the largest finite codes: rows before it keep their bits,
    those of the same tile among them (a NaN code there would make them NaN, by the product with a weight of 0)."""
    cache, table, q = attention_case(gpu, 94, fmt, "fp16", dh, 16, 2, 4, [400], 400)
    t, cu, n = i32(table, gpu), i32([0, 400], gpu), i32([400], gpu)
    want = kv8.cache8_prefill(cache, q, cu, t, n)
    largest = 127 if fmt == "int8" else 0x7E
    cache.k_codes[int(table[0, 21])] = largest                           # tokens 336 .. 351 of the tile 320 .. 383
    cache.v_codes[int(table[0, 21])] = largest
    got = kv8.cache8_prefill(cache, q, cu, t, n)
    assert torch.isfinite(got).all()
    assert torch.equal(got[:336], want[:336]) and not torch.equal(got[336:], want[336:])


@pytest.mark.parametrize("ps", [16, 64])
@pytest.mark.parametrize("cu", [[0, 40, 10, 60], [50, 0, 60, 20], [-5, 1000, 3, 60], [60, 40, 20, 0], [2 ** 31 - 1, -2 ** 31, 30, 31]])
def test_row_starts_out_of_order(gpu, cu, ps):
    """Which rows such row starts stand for is not defined; every call ends, and no row outside 0 .. num_rows - 1 and
    no page outside the tables is touched."""
    rows, num_kv, gqa, dh = 60, 2, 4, 64
    cache = random_cache(gpu, 96, 20, num_kv, dh, ps, "int8")
    table = tables(97, 16, [4, 4, 4])
    spare = np.setdiff1d(np.arange(20), table)
    before = [x[spare].clone() for x in (cache.k_codes, cache.v_codes, cache.scales)]
    td, start, lens, c = i32(table, gpu), i32([0, 3, 20], gpu), i32([64, 30, 50], gpu), i32(cu, gpu)
    k = torch.full((rows + 8, num_kv, dh), float("inf"), device=gpu)     # rows around the given ones: would fill pages
    k[4:-4] = torch.rand(rows, num_kv, dh, device=gpu)
    kv8.cache8_write(cache, k[4:-4], k[4:-4], td, start, c)
    assert all(torch.equal(x[spare], y) for x, y in zip((cache.k_codes, cache.v_codes, cache.scales), before))
    assert torch.isfinite(cache.scales).all()
    ko, vo = (torch.full((rows + 8, num_kv, dh), 7.0, dtype=torch.float16, device=gpu) for _ in range(2))
    kv8.cache8_read(cache, td, start, c, rows, torch.float16, ko[4:-4], vo[4:-4])
    q = torch.randn(rows, num_kv * gqa, dh, device=gpu).half()
    out = torch.full((rows + 8, num_kv * gqa, dh), 7.0, dtype=torch.float16, device=gpu)
    lse = torch.full((rows + 8, num_kv * gqa), 7.0, device=gpu)
    kv8.cache8_prefill(cache, q, c, td, lens, out=out[4:-4], lse=lse[4:-4])
    for x in (ko, vo, out, lse):
        assert (x[:4] == 7).all() and (x[-4:] == 7).all()


def test_head_counts_that_no_call_takes_are_refused(gpu):
    for num_kv in (0, 1025):
        with pytest.raises(ValueError, match="num_kv must be"):
            kv8.Cache8.allocate(1, num_kv, 64, 16, "int8", gpu)
