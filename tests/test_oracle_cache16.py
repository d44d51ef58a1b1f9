"""CPU tests of the 16-bit KV cache: its oracle, the C entries' refusals (no
launch) and the Python layer's checks."""
import ctypes

import numpy as np
import pytest
import torch

import sphkv_kv16 as kv16
import sphkv_kv8 as kv8
import sphkv_lib
from oracle import cache16 as o16

LIB = sphkv_lib.load()
P = 1 << 20                      # an address that nothing reads


# ---- the oracle ------------------------------------------------------------------

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("parts", [1, 2])
def test_rotation_is_that_of_complex_numbers(interleaved, parts):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((5, 3, 64))
    pos, f = np.array([0, 1, 7, 1000, -4]), 10000.0 ** (-np.arange(8) / 8)
    y = o16.rotated(x, pos, f, interleaved, parts)
    w = 64 // parts
    for p in range(parts):
        a, b = x[..., p * w:(p + 1) * w], y[..., p * w:(p + 1) * w]
        pair = (lambda t: t[..., 0:16:2] + 1j * t[..., 1:16:2]) if interleaved else (lambda t: t[..., :8] + 1j * t[..., 8:16])
        assert np.allclose(pair(b), pair(a) * np.exp(1j * pos[:, None, None] * f), atol=1e-12)
        assert np.array_equal(b[..., 16:], a[..., 16:])
    assert np.array_equal(y[0], x[0])


def test_attention_of_the_oracle_is_softmax():
    rng = np.random.default_rng(2)
    H, gqa, dh, ps, L, m = 2, 3, 64, 16, 37, 9
    c = o16.Cache(np.full((4, H, ps, dh), np.nan), np.full((4, H, ps, dh), np.nan))
    k, v = rng.standard_normal((2, L, H, dh))
    table = np.array([[3, 0, 2]])
    c.append(k, v, table, [0], [0, L])
    q = rng.standard_normal((m, H * gqa, dh))
    for causal, window in ((True, 0), (True, 5), (False, 0)):
        out, lse = c.attend(q, table, [L], [0, m], causal, window)[:2]
        j, at = torch.arange(L)[None, :], L - m + torch.arange(m)[:, None]
        see = (j <= at) & ((j > at - window) if window else (j >= 0)) if causal else torch.ones(m, L, dtype=torch.bool)
        for h in range(H * gqa):
            x = torch.from_numpy(q[:, h] @ k[:, h // gqa].T) / 8.0
            x = x.masked_fill(~see, -np.inf)
            assert np.allclose(out[:, h], torch.softmax(x, 1).numpy() @ v[:, h // gqa])
            assert np.allclose(lse[:, h], torch.logsumexp(x, 1).numpy())


def test_difference_of_maps():
    rng = np.random.default_rng(3)
    H, dh, ps, L = 1, 64, 16, 20
    c = o16.Cache(*rng.standard_normal((2, 2, H, ps, dh)))
    q = rng.standard_normal((1, 2, dh))
    table = np.array([[1, 0]])
    maps = c.maps(q, table, [L])
    k, v = (np.concatenate([x[1, 0], x[0, 0]])[:L] for x in (c.k, c.v))
    lam, w = [0.3, 0.7], rng.standard_normal(dh)
    out, x, _ = o16.difference(maps[0][0], maps[1][0], lam, w, 1e-5)
    for h in range(2):
        a = [np.exp(q[0, h, d] @ k[:, d].T / np.sqrt(32)) for d in (slice(0, 32), slice(32, 64))]
        y = (a[0] / a[0].sum() - lam[h] * a[1] / a[1].sum()) @ v
        assert np.allclose(x[0, h], y)
        assert np.allclose(out[0, h], y / np.sqrt((y ** 2).mean() + 1e-5) * w)


# ---- refusals of the C entries -----------------------------------------------------

def struct(**kw):
    d = dict(k=P, v=P, k_page=16 * 64, k_head=0, k_token=64, v_page=16 * 64, v_head=0, v_token=64, num_pages=4, num_kv=1, dh=64,
             page_size=16, type=0)
    d.update(kw)
    return sphkv_lib.Cache16Struct(*(d[n] for n, _ in sphkv_lib.Cache16Struct._fields_))


# the struct's fields by the names that the cases use: its k and v are "ck" and "cv"
FIELDS = {{"k": "ck", "v": "cv"}.get(n, n): n for n, _ in sphkv_lib.Cache16Struct._fields_}


def call(name, order, defaults, kw):
    s = struct(**{FIELDS[k]: v for k, v in kw.items() if k in FIELDS})
    rest = {k: v for k, v in kw.items() if k not in FIELDS}
    d = dict(defaults)
    d.update(rest)
    cache = d.pop("cache", ctypes.addressof(s))
    assert set(d) == set(order), set(d) ^ set(order)
    rc = getattr(LIB, name)(cache, *(d[n] for n in order), None)
    return rc, LIB.sphkv_last_error().decode()


APPEND = ["k", "v", "q", "in_type", "k_row", "k_head_", "v_row", "v_head_", "q_row", "q_head", "gqa", "q_out", "o_row", "o_head",
          "num_rows", "cu_rows", "start", "table", "table_stride", "max_blocks", "num_seqs", "inv_freq", "freq_type", "num_freqs",
          "parts", "interleaved"]
APPEND_DEFAULTS = dict(k=P, v=P, q=P, in_type=0, k_row=64, k_head_=64, v_row=64, v_head_=64, q_row=64, q_head=64, gqa=1, q_out=P,
                       o_row=64, o_head=64, num_rows=0, cu_rows=None, start=P, table=P, table_stride=2, max_blocks=2, num_seqs=0,
                       inv_freq=P, freq_type=3, num_freqs=32, parts=1, interleaved=0)
DECODE = ["q", "q_row", "q_head", "gqa", "lens", "window", "table", "table_stride", "max_blocks", "num_seqs", "sm_scale", "out",
          "lse", "ws", "ws_bytes"]
DECODE_DEFAULTS = dict(q=P, q_row=64, q_head=64, gqa=1, lens=P, window=0, table=P, table_stride=2, max_blocks=2, num_seqs=0,
                       sm_scale=0.125, out=P, lse=None, ws=P, ws_bytes=1 << 40)
DIFF = ["lambda_", "norm_weight", "norm_eps"]
PREFILL = DECODE[:4] + ["num_rows", "cu_rows", "lens", "causal"] + DECODE[5:]
PREFILL_DEFAULTS = dict(DECODE_DEFAULTS, num_rows=0, cu_rows=P, causal=1)
ENTRIES = {
    "append": ("sphkv_cache16_append", APPEND, APPEND_DEFAULTS),
    "decode": ("sphkv_cache16_decode", DECODE, DECODE_DEFAULTS),
    "diff_decode": ("sphkv_cache16_diff_decode", DECODE[:4] + DIFF + DECODE[4:], dict(DECODE_DEFAULTS, lambda_=P, norm_weight=P, norm_eps=1e-5)),
    "prefill": ("sphkv_cache16_prefill", PREFILL, PREFILL_DEFAULTS),
    "diff_prefill": ("sphkv_cache16_diff_prefill", PREFILL[:4] + DIFF + PREFILL[4:], dict(PREFILL_DEFAULTS, lambda_=P, norm_weight=P, norm_eps=1e-5)),
}
ATTENTION = ["decode", "diff_decode", "prefill", "diff_prefill"]
SHARED = [
    (dict(cache=None), "null pointer"),
    (dict(dh=96), "dh must be"),
    (dict(page_size=48), "page_size must be"),
    (dict(page_size=256), "page_size must be"),
    (dict(type=2), "fp16 or bf16"),
    (dict(type=-1), "fp16 or bf16"),
    (dict(num_kv=0), "negative size"),
    (dict(num_kv=1025), "num_kv must be"),
    (dict(num_pages=-1), "negative size"),
    (dict(num_pages=1 << 31), "num_pages exceeds"),
    (dict(num_seqs=-1), "negative size"),
    (dict(max_blocks=-1), "negative size"),
    (dict(k_page=-8), "strides must be"),
    (dict(k_token=65), "strides must be"),
    (dict(v_head=4), "strides must be"),
    (dict(k_token=(1 << 24) + 8), "token stride"),
    (dict(v_token=(1 << 24) + 8), "token stride"),
    (dict(num_seqs=(1 << 16) + 1), "2^16 sequences"),
    (dict(num_seqs=1 << 16, num_kv=1024), "num_kv exceeds"),
    (dict(max_blocks=(1 << 26) + 1, table_stride=1 << 27), "exceeds 2^30"),
    (dict(num_seqs=2, max_blocks=5, table_stride=4), "table_stride"),
    (dict(ck=P + 8), "16-byte aligned"),
    (dict(cv=P + 2), "16-byte aligned"),
    (dict(num_seqs=1, ck=None), "null pointer"),
    (dict(num_seqs=1, table=None), "null pointer"),
]


@pytest.mark.parametrize("kw, msg", SHARED)
@pytest.mark.parametrize("entry", ENTRIES)
def test_refusals_of_a_cache(entry, kw, msg):
    rc, text = call(*ENTRIES[entry], kw)
    assert rc == -1 and msg in text and ENTRIES[entry][0] in text


@pytest.mark.parametrize("kw, msg", [
    (dict(in_type=3), "unknown type"),
    (dict(in_type=-1), "unknown type"),
    (dict(gqa=-1), "gqa must be"),
    (dict(gqa=65), "gqa must be"),
    (dict(num_seqs=1, num_rows=1, gqa=0), "gqa must be 0 without q"),
    (dict(num_seqs=1, num_rows=1, q=None), "gqa must be 0 without q"),
    (dict(parts=0), "parts must be"),
    (dict(parts=3), "parts must be"),
    (dict(interleaved=2), "interleaved must be"),
    (dict(num_freqs=-8), "num_freqs must be"),
    (dict(num_freqs=12), "num_freqs must be"),
    (dict(num_freqs=40), "num_freqs must be"),
    (dict(num_freqs=24, parts=2), "num_freqs must be"),
    (dict(num_freqs=2 ** 31 - 8), "num_freqs must be"),
    (dict(freq_type=0), "inv_freq must be"),
    (dict(num_rows=1), "one row per sequence"),
    (dict(num_rows=-1), "negative size"),
    (dict(num_rows=(1 << 26) + 1, cu_rows=P), "2^26 rows"),
    (dict(num_rows=1 << 26, cu_rows=P), "below 2^26"),
    (dict(num_seqs=1, num_rows=1, k=None), "null pointer"),
    (dict(num_seqs=1, num_rows=1, v=None), "null pointer"),
    (dict(num_seqs=1, num_rows=1, start=None), "null pointer"),
    (dict(num_seqs=1, num_rows=1, q_out=None), "null pointer"),
    (dict(num_seqs=1, num_rows=1, inv_freq=None), "null pointer"),
])
def test_append_refusals(kw, msg):
    rc, text = call(*ENTRIES["append"], kw)
    assert rc == -1 and msg in text, text


# what an append writes is written once and not read as something else.  Caches that are in order, and the other way
# round queries' outputs that are, are shown by the refusal of what is looked at next
A, B, Q, O, K, V = (i << 32 for i in range(1, 7))
ONE = dict(num_seqs=1, num_rows=1, ck=A, cv=B, q=Q, q_out=O, k=K, v=V)
GOOD_CACHES = [
    dict(),
    dict(num_kv=3, k_head=16 * 64, v_head=16 * 64, k_page=3 * 16 * 64, v_page=3 * 16 * 64),
    dict(num_kv=3, k_head=64, v_head=64, k_token=3 * 64, v_token=3 * 64, k_page=3 * 16 * 64, v_page=3 * 16 * 64),
    dict(cv=A + 2 * 16 * 64, k_page=2 * 16 * 64, v_page=2 * 16 * 64),                             # a page's keys, then its values
    dict(cv=A + 2 * 64, k_token=128, v_token=128, k_page=16 * 128, v_page=16 * 128),              # a token's
    dict(cv=A + 2 * 64, num_kv=3, k_head=128, v_head=128, k_token=3 * 128, v_token=3 * 128, k_page=3 * 16 * 128, v_page=3 * 16 * 128),
    dict(num_pages=1, k_page=0, v_page=0),
    dict(cv=A + 2 * 4 * 16 * 64),                                                                  # behind each other
]
BAD_CACHES = [
    dict(cv=A),
    dict(cv=A + 2 * 64),
    dict(cv=A + 2 * 4 * 16 * 64 - 16),
    dict(k_page=0),
    dict(v_page=0),
    dict(v_token=0),
    dict(k_token=56),
    dict(num_kv=2),                                                                                # (head strides 0)
    dict(num_kv=2, k_head=16 * 64, v_head=16 * 64),                                                # (page strides for one head)
    dict(k_page=16 * 64 - 8),
]


@pytest.mark.parametrize("kw", GOOD_CACHES)
def test_append_takes_caches_in_order(kw):
    rc, text = call(*ENTRIES["append"], {**ONE, "q_out": Q + 2, **kw})
    assert rc == -1 and "q_out must be q itself" in text, text


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_append_refuses_caches_that_share_memory(kw):
    rc, text = call(*ENTRIES["append"], {**ONE, **kw})
    assert rc == -1 and "the cache, or its k and v, share memory" in text, text
    rc, text = call(*ENTRIES["append"], {**ONE, "q": None, "gqa": 0, **kw})
    assert rc == -1 and "the cache, or its k and v, share memory" in text, text


ROWS = dict(num_seqs=3, num_rows=3, gqa=2, q_row=128, q_head=64, o_row=128, o_head=64)


@pytest.mark.parametrize("kw", [
    dict(),
    dict(q_out=Q),
    dict(q_out=Q + 2 * 128, q_row=256, o_row=256),                                                 # halves of a row
    dict(q_out=Q + 2 * 64, q_row=256, q_head=128, o_row=256, o_head=128),                          # every other head
    dict(q_out=Q, q_row=-200, o_row=-200),
    dict(q=K - 2 * 128, q_out=K - 2 * 128, q_row=320, o_row=320, k_row=320, v=K + 128, v_row=320),  # q, k, v of one row
], ids=range(6))
def test_append_takes_outputs_in_order(kw):
    """(The keys or values are laid over the outputs then.)"""
    good = {**ONE, **ROWS, **kw}
    if "v" not in kw:
        rc, text = call(*ENTRIES["append"], {**good, "v": good["q_out"] + 2})
    else:
        rc, text = call(*ENTRIES["append"], {**good, "v": good["q_out"] + 4})
    assert rc == -1 and "shares memory with k or v" in text, text


@pytest.mark.parametrize("kw, msg", [
    (dict(o_row=64), "rows and heads of q_out overlap"),
    (dict(o_row=0), "rows and heads of q_out overlap"),
    (dict(o_head=63), "rows and heads of q_out overlap"),
    (dict(o_row=-127), "rows and heads of q_out overlap"),
    (dict(q_out=Q + 2), "q_out must be q itself"),
    (dict(q_out=Q + 2 * 64), "q_out must be q itself"),
    (dict(q_out=Q, o_row=192), "q_out must be q itself"),
    (dict(q_out=Q, o_row=64, o_head=192), "q_out must be q itself"),
    (dict(q_out=Q, in_type=2), "q_out must be q itself"),
    (dict(q_out=Q, in_type=1), "q_out must be q itself"),
    (dict(q_out=Q - 2 * 383), "q_out must be q itself"),
    (dict(q_out=K), "shares memory with k or v"),
    (dict(q_out=V + 2 * 191), "shares memory with k or v"),
])
def test_append_refuses_outputs_that_share_memory(kw, msg):
    rc, text = call(*ENTRIES["append"], {**ONE, **ROWS, **kw})
    assert rc == -1 and msg in text, text


@pytest.mark.parametrize("kw, msg", [
    (dict(gqa=0), "gqa must be"),
    (dict(gqa=65), "gqa must be"),
    (dict(window=-1), "window must be"),
    (dict(sm_scale=0.0), "sm_scale"),
    (dict(sm_scale=-1.0), "sm_scale"),
    (dict(sm_scale=float("nan")), "sm_scale"),
    (dict(sm_scale=float("inf")), "sm_scale"),
])
@pytest.mark.parametrize("entry", ATTENTION)
def test_attention_refusals(entry, kw, msg):
    rc, text = call(*ENTRIES[entry], kw)
    assert rc == -1 and msg in text


@pytest.mark.parametrize("kw, msg", [
    (dict(q=None), "null pointer"),
    (dict(lens=None), "null pointer"),
    (dict(out=None), "null pointer"),
    (dict(ws=None), "workspace needs"),
    (dict(ws_bytes=100), "workspace needs"),
    (dict(ws=P + 4), "workspace must be"),
])
@pytest.mark.parametrize("entry", ATTENTION)
def test_attention_refusals_of_work(entry, kw, msg):
    more = dict(num_seqs=1, num_rows=1, cu_rows=P) if "prefill" in entry else dict(num_seqs=1)
    rc, text = call(*ENTRIES[entry], dict(more, **kw))
    assert rc == -1 and msg in text


@pytest.mark.parametrize("kw", [
    dict(out=Q + 2),
    dict(out=Q, q_row=192),
    dict(out=Q, q_row=64, q_head=192),
    dict(out=Q, q_head=0),
    dict(out=Q + 2 * 128, q_row=200),
    dict(out=Q - 2 * 127),
])
@pytest.mark.parametrize("entry", ATTENTION)
def test_attention_refuses_outputs_over_other_queries(entry, kw):
    more = dict(num_rows=3, cu_rows=P) if "prefill" in entry else {}
    rc, text = call(*ENTRIES[entry], dict(dict(num_seqs=3, gqa=2, q=Q, q_row=128, q_head=64, **more), **kw))
    assert rc == -1 and "out must be q itself" in text, text


@pytest.mark.parametrize("kw, msg", [
    (dict(gqa=33), "gqa must be"),
    (dict(norm_eps=-1e-9), "norm_eps"),
    (dict(norm_eps=float("nan")), "norm_eps"),
    (dict(norm_eps=float("inf")), "norm_eps"),
    (dict(num_seqs=1, num_rows=1, lambda_=None), "null pointer"),
])
@pytest.mark.parametrize("entry", ["diff_decode", "diff_prefill"])
def test_differential_refusals(entry, kw, msg):
    if entry == "diff_decode":
        kw = {k: v for k, v in kw.items() if k != "num_rows"}
    rc, text = call(*ENTRIES[entry], kw)
    assert rc == -1 and msg in text


@pytest.mark.parametrize("entry", ["prefill", "diff_prefill"])
def test_prefill_refusals(entry):
    for kw, msg in ((dict(causal=2), "causal must be"), (dict(causal=0, window=4), "window must be"),
                    (dict(num_seqs=1, num_rows=1, cu_rows=None), "null pointer"),
                    (dict(num_rows=1 << 26, num_seqs=1, gqa=16), "too many")):
        rc, text = call(*ENTRIES[entry], kw)
        assert rc == -1 and msg in text


def test_decode_grid_past_32_bits_is_refused():
    rc, text = call(*ENTRIES["decode"], dict(num_seqs=1 << 16, gqa=64, num_kv=4))
    assert rc == -1 and "too many" in text


@pytest.mark.parametrize("entry", ENTRIES)
def test_nothing_to_do_is_no_error(entry):
    rc, text = call(*ENTRIES[entry], {})
    assert rc == 0 and text == ""
    if "prefill" in entry or entry == "append":
        more = dict(num_seqs=3, num_rows=0, cu_rows=P)
        assert call(*ENTRIES[entry], more)[0] == 0


def test_workspace_sizes():
    d, p = LIB.sphkv_cache16_decode_workspace_bytes, LIB.sphkv_cache16_prefill_workspace_bytes
    for bad in ((-1, 1, 1, 64, 0), (1, 0, 1, 64, 0), (1, 1, 0, 64, 0), (1, 1, 65, 64, 0), (1, 1, 33, 64, 1), (1, 1, 1, 96, 0)):
        assert d(*bad) == -1 and p(1, *bad) == -1
    assert p(-1, 1, 1, 1, 64, 0) == -1
    assert d(1, 8, 4, 128, 0) > 0 and d(1, 8, 4, 128, 1) > d(1, 8, 4, 128, 0)
    assert p(0, 1, 1, 1, 64, 0) == 0 and p(100000, 1, 8, 4, 128, 0) == 0
    assert p(1, 1, 1, 1, 64, 0) > 0


# ---- the Python layer -----------------------------------------------------------------

def test_python_refuses_cpu_tensors_and_other_types():
    x = torch.zeros((2, 1, 16, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        kv16.Cache16(x, x)
    with pytest.raises(TypeError, match="fp16 or bf16"):
        kv16.Cache16(x.float(), x.float())
    with pytest.raises(TypeError, match="fp16 or bf16"):
        kv16.Cache16(None, x)


def test_struct_matches_the_header():
    """Eight 8-byte words of pointers and strides, num_pages, then four ints."""
    S = sphkv_lib.Cache16Struct
    assert ctypes.sizeof(S) == 9 * 8 + 4 * 4
    assert S.num_pages.offset == 64 and S.num_kv.offset == 72 and S.type.offset == 84


def test_default_frequencies():
    f = kv16.rope_inv_freq(128, 500000.0, "cpu")
    assert f.dtype is torch.float64 and f.shape == (64,) and f[0] == 1.0
    assert abs(f[1].item() - 500000.0 ** (-2 / 128)) < 1e-15


@pytest.fixture
def on_cpu(monkeypatch):
    """CPU tensors pass for the GPU's; a call that would be launched says so."""
    def need(t, dtype, name, device=None):
        if not isinstance(t, torch.Tensor) or t.dtype != dtype:
            raise TypeError(name)

    def launched(self, fn, *args):
        raise AssertionError("launched")

    for module in (kv8, kv16):
        monkeypatch.setattr(module, "_need", need)
    monkeypatch.setattr(kv16.Cache16, "_call", launched)


def half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("k, v, msg", [
    (half(2, 1, 16, 64), half(2, 1, 16, 128), "v must be"),
    (half(1, 16, 64), half(1, 16, 64), "k must be"),
    (half(2, 1, 24, 64), half(2, 1, 24, 64), "page_size must be"),
    (half(2, 1, 16, 96), half(2, 1, 16, 96), "dh must be"),
    (half(1, 1025, 16, 64), half(1, 1025, 16, 64), "num_kv must be"),
    (half(2, 1, 16, 68)[..., :64], half(2, 1, 16, 64), "multiples of 8"),
    (half(2, 1, 64, 16).transpose(2, 3)[:, :, :16], half(2, 1, 16, 64), "k must be|page_size|dh must be|contiguous"),
    (half(4, 1, 16, 64).view(-1)[1:2049].view(2, 1, 16, 64), half(2, 1, 16, 64), "16-byte aligned"),
])
def test_python_refuses_caches(on_cpu, k, v, msg):
    with pytest.raises(ValueError, match=msg):
        kv16.Cache16(k, v)


APPEND_ARGS = dict(k=half(2, 1, 64), v=half(2, 1, 64), table=torch.zeros((2, 1), dtype=torch.int32), start=ints(0, 0))


@pytest.mark.parametrize("kw, error, msg", [
    (dict(), AssertionError, "launched"),
    (dict(q=half(2, 3, 64), q_out=half(3, 2, 64).transpose(0, 1)), AssertionError, "launched"),
    (dict(q=half(2, 3, 64), q_out=half(2, 1, 64).expand(2, 3, 64)), ValueError, "overlap"),
    (dict(q=half(2, 3, 64), q_out=half(1, 3, 64).expand(2, 3, 64)), ValueError, "overlap"),
    (dict(q=half(2, 1, 64), q_out=half(100).as_strided((2, 1, 64), (32, 64, 1))), ValueError, "overlap"),
    (dict(q=half(2, 2, 64), q_out=half(300).as_strided((2, 2, 64), (100, 64, 1))), ValueError, "overlap"),
    (dict(q=half(2, 2, 64), q_out=half(300).as_strided((2, 2, 64), (64, 100, 1))), ValueError, "overlap"),
    (dict(q=half(2, 2, 64), q_out=half(2, 1, 64)), ValueError, "q_out must be"),
    (dict(q_out=half(2, 1, 64)), ValueError, "goes with q"),
    (dict(q=half(3, 1, 64)), ValueError, "q must be"),
    (dict(q=half(2, 0, 64)), ValueError, "q must be"),
    (dict(q=half(2, 1, 64).float()), TypeError, "q"),
    (dict(k=half(2, 1, 64).double()), TypeError, "k must be"),
    (dict(v=half(3, 1, 64)), ValueError, "as many rows"),
    (dict(v=half(2, 64, 2).transpose(1, 2)[:, :1]), ValueError, "contiguous"),
    (dict(start=ints(0, 0, 0)), ValueError, "table must be"),
    (dict(start=ints(0, 0).long()), TypeError, "start"),
    (dict(table=torch.zeros((2, 2), dtype=torch.int32).t()), ValueError, "contiguous"),
    (dict(table=torch.zeros((1, 2), dtype=torch.int32).expand(2, 2)), ValueError, "overlap"),
    (dict(cu_rows=ints(0, 2)), ValueError, "cu_rows must be"),
    (dict(k=half(3, 1, 64), v=half(3, 1, 64)), ValueError, "one row per sequence"),
    (dict(parts=3), ValueError, "parts must be"),
    (dict(parts=2 ** 32 + 1), ValueError, "parts must be"),
    (dict(inv_freq=half(32)), TypeError, "inv_freq must be"),
    (dict(inv_freq=torch.zeros(64)[::2]), ValueError, "inv_freq must be"),
])
def test_python_refuses_appends(on_cpu, kw, error, msg):
    cache = kv16.Cache16(half(2, 1, 16, 64), half(2, 1, 16, 64))
    with pytest.raises(error, match=msg):
        kv16.cache16_append(cache, **{**APPEND_ARGS, **kw})


@pytest.mark.parametrize("name", ["decode", "prefill", "diff_decode", "diff_prefill"])
@pytest.mark.parametrize("kw, error, msg", [
    (dict(), AssertionError, "launched"),
    (dict(window=2 ** 31 - 1), AssertionError, "launched"),
    (dict(window=2 ** 31), ValueError, "window must be"),
    (dict(window=2 ** 32 + 5), ValueError, "window must be"),
    (dict(window=-1), ValueError, "window must be"),
    (dict(window=2.5), ValueError, "window must be"),
    (dict(window=0.4), ValueError, "window must be"),
    (dict(q=torch.nn.Parameter(half(2, 2, 64))), AssertionError, "launched"),
    (dict(lens=ints(1, 7, 1, 7)[::2]), ValueError, "contiguous"),
    (dict(table=torch.zeros((2, 4), dtype=torch.int32)[:, ::2]), ValueError, "contiguous"),
    (dict(lens=None), TypeError, "lens"),
    (dict(q=half(2, 0, 64)), ValueError, "q must be"),
    (dict(q=half(2, 2, 32)), ValueError, "q must be"),
    (dict(q=half(2, 65, 64)), ValueError, "bad num"),
    (dict(q=half(2, 2, 64).bfloat16()), TypeError, "q"),
    (dict(out=half(2, 4, 64)[:, ::2]), ValueError, "out must be"),
    (dict(lse=torch.zeros(1)), ValueError, "lse must be"),
    (dict(lens=ints(1)), ValueError, "table must be"),
    (dict(workspace=torch.zeros(4, dtype=torch.uint8)), ValueError, "workspace"),
])
def test_python_refuses_attention(on_cpu, name, kw, error, msg):
    cache = kv16.Cache16(half(2, 1, 16, 64), half(2, 1, 16, 64))
    args = dict(q=half(2, 2, 64), table=torch.zeros((2, 1), dtype=torch.int32), lens=ints(1, 1))
    if "prefill" in name:
        args["cu_rows"] = ints(0, 1, 2)
    if "diff" in name:
        args["lam"] = torch.zeros(kw["q"].shape[1] if "q" in kw else 2)
    with pytest.raises(error, match=msg):
        getattr(kv16, "cache16_" + name)(cache, **{**args, **kw})


@pytest.mark.parametrize("kw, error, msg", [
    (dict(lam=torch.zeros(3)), ValueError, "lam must be"),
    (dict(lam=torch.zeros(4)[::2]), ValueError, "lam must be"),
    (dict(lam=torch.zeros(1).expand(2)), ValueError, "lam must be"),
    (dict(lam=half(2)), TypeError, "lam"),
    (dict(norm_weight=torch.zeros(128)[::2]), ValueError, "norm_weight must be"),
    (dict(norm_weight=half(64)), TypeError, "norm_weight"),
])
def test_python_refuses_differential_weights(on_cpu, kw, error, msg):
    cache = kv16.Cache16(half(2, 1, 16, 64), half(2, 1, 16, 64))
    args = dict(q=half(2, 2, 64), lam=torch.zeros(2), table=torch.zeros((2, 1), dtype=torch.int32), lens=ints(1, 1))
    with pytest.raises(error, match=msg):
        kv16.cache16_diff_decode(cache, **{**args, **kw})
    with pytest.raises(error, match=msg):
        kv16.cache16_diff_prefill(cache, cu_rows=ints(0, 1, 2), **{**args, **kw})
    with pytest.raises(TypeError, match="cu_rows"):
        kv16.cache16_diff_prefill(cache, cu_rows=None, **args)
