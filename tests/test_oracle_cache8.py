"""The 8-bit cache's oracle (oracle/cache8.py) against direct formulas, and the
library's host-side checks: every refusal of the C ABI and of the Python
entries, without a GPU."""
import numpy as np
import pytest
import torch

import sphkv_kv8 as kv8
import sphkv_lib
from oracle import cache8 as o8

_FAKE = 1 << 20       # an aligned non-null address that no refused call follows


# ---- the oracle -------------------------------------------------------------

def test_code_tables_are_those_of_torch():
    b = torch.arange(256, dtype=torch.uint8)
    assert np.array_equal(o8.VALUES["int8"], b.view(torch.int8).double().numpy())
    want = b.view(torch.float8_e4m3fn).float().double().numpy()
    assert np.array_equal(o8.VALUES["e4m3"], want, equal_nan=True)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_codes_are_the_nearest(fmt):
    rng = np.random.default_rng(0)
    y = np.concatenate([rng.uniform(-140, 140, 4000), rng.uniform(-1, 1, 4000) * 2.0 ** rng.integers(-12, 9, 4000),
                        np.arange(-128, 128) + 0.5, [0.0, 500.0, -500.0, np.nan, np.inf, -np.inf]])
    got = o8.code_values(y, fmt)
    table = np.unique(o8.VALUES[fmt][np.isfinite(o8.VALUES[fmt])])
    if fmt == "int8":
        table = table[table >= -127]
    z = np.where(np.isnan(y), 0, np.clip(y, table[0], table[-1]))
    best = np.abs(z[:, None] - table[None, :]).min(1)
    assert (np.abs(z - got) == best).all()                       # ties: either neighbour is the nearest
    assert np.array_equal(o8.VALUES[fmt][o8.codes_of(got, fmt)], got)
    if fmt == "e4m3":                                            # torch rounds half to even
        t = torch.from_numpy(z).float()
        keep = (t.double().numpy() == z)
        assert np.array_equal(t.to(torch.float8_e4m3fn).float().double().numpy()[keep], got[keep])


@pytest.mark.parametrize("fmt, top", [("int8", 127.0), ("e4m3", 448.0)])
def test_scales_hold_the_largest_value(fmt, top):
    for a in (1.0, 3.7, 448.0, 449.0, 224.0, 1e-3, 6.1e4, 2.0 ** -24):
        s = o8.scale_of(a, fmt)
        assert a / s <= top * (1 + 2.0 ** -23)
        assert a / s > (top / 2 if fmt == "e4m3" else top * (1 - 2.0 ** -23))
    assert o8.scale_of(0.0, fmt) == 2.0 ** -60 and o8.scale_of(1e30, fmt) == 2.0 ** 60


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_appending_grows_a_scale_and_keeps_the_values(fmt):
    rng = np.random.default_rng(1)
    c = o8.Cache(4, 2, 64, 16, fmt)
    table = np.array([[2, -1, 3]])
    x = rng.standard_normal((40, 2, 64)) * np.exp(rng.normal(0, 1, (40, 1, 1)))
    for t in range(40):
        c.write(x[t:t + 1], -x[t:t + 1], table, [t])
    k, v, present = c.tokens(table, 0, 0, 40)
    assert present.tolist() == [True] * 16 + [False] * 16 + [True] * 8
    # each growth rounds once more, each at most half a code of its scale (int8) or 2^-4 of the value (e4m3)
    for a, b in ((0, 16), (32, 40)):
        top = np.abs(x[a:b]).max((0, 2), keepdims=True)
        worst = np.abs(k[a:b] - x[a:b])
        assert (worst <= (16 * top / 254 if fmt == "int8" else np.abs(x[a:b]) * 2.0 ** -3 + top * 2.0 ** -15)).all()
    assert np.array_equal(v, -k)


def test_attention_of_the_oracle_is_softmax():
    rng = np.random.default_rng(2)
    c = o8.Cache(6, 2, 64, 16, "int8")
    table = np.array([[1, 0, 5], [3, 2, -1]])
    x = rng.standard_normal((60, 2, 64))
    c.write(x, x[::-1], table, [0, 0], [0, 40, 60])
    q = rng.standard_normal((5, 4, 64))
    out, lse, *_ = c.attend(q, table, [40, 20], [0, 3, 5])
    k, v, _ = c.tokens(table, 0, 0, 39)                          # row 1 of sequence 0: positions 0..38
    s = k[:, 1] @ q[1, 3] / 8.0
    p = np.exp(s - s.max())
    assert np.allclose(out[1, 3], p @ v[:, 1] / p.sum(), rtol=1e-12) and np.isclose(lse[1, 3], np.log(np.exp(s).sum()))
    out, lse, *_ = c.attend(q[:2], table, [0, 7])
    assert (out[0] == 0).all() and (lse[0] == -np.inf).all() and np.isfinite(lse[1]).all()


# ---- refusals of the C ABI ----------------------------------------------------

def _write_args(**kw):
    a = dict(k=_FAKE, v=_FAKE, in_type=0, ks=1024, kh=128, vs=1024, vh=128, num_rows=4, cu=_FAKE, start=_FAKE, table=_FAKE,
             ts=8, mb=8, num_seqs=2, kc=_FAKE, vc=_FAKE, sc=_FAKE, pages=16, num_kv=8, dh=128, ps=16, fmt=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


def _read_args(**kw):
    a = dict(kc=_FAKE, vc=_FAKE, sc=_FAKE, pages=16, num_kv=8, dh=128, ps=16, fmt=0, cu=_FAKE, start=_FAKE, table=_FAKE,
             ts=8, mb=8, num_seqs=2, num_rows=4, k=_FAKE, v=_FAKE, out_type=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


def _attend_args(decode, **kw):
    a = dict(q=_FAKE, q_type=0, qs=4096, qh=128, num_rows=4, cu=_FAKE, lens=_FAKE, causal=1, table=_FAKE, ts=8, mb=8,
             num_seqs=2, kc=_FAKE, vc=_FAKE, sc=_FAKE, pages=16, num_kv=8, gqa=4, dh=128, ps=16, fmt=0, sm=0.1, out=_FAKE,
             lse=None, ws=_FAKE, wsb=1 << 40, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    if decode:
        for name in ("num_rows", "cu", "causal"):
            del a[name]
    return list(a.values())


_SHARED = [
    (dict(dh=96), "dh must be 64 or 128"), (dict(ps=8), "page_size must be"), (dict(ps=48), "page_size must be"),
    (dict(ps=256), "page_size must be"), (dict(fmt=2), "unknown fmt"), (dict(num_seqs=-1), "negative size"),
    (dict(pages=-1), "negative size"), (dict(num_kv=0), "negative size"), (dict(num_kv=1025), "num_kv must be"),
    (dict(pages=1 << 31), "exceeds int32"), (dict(mb=1 << 27, ts=1 << 27), "exceeds 2^30"),
    (dict(ts=7), "table_stride"), (dict(kc=_FAKE + 8), "16-byte aligned"), (dict(sc=_FAKE + 4), "16-byte aligned"),
    (dict(vc=None), "null pointer"), (dict(table=None), "null pointer"), (dict(num_seqs=(1 << 16) + 1), "at most 2^16"),
    (dict(num_seqs=1 << 16, num_kv=1024), "exceeds 2^25"),
]


@pytest.mark.parametrize("kw, msg", _SHARED + [
    (dict(in_type=3), "unknown type"), (dict(cu=None), "one row per sequence"), (dict(k=None), "null pointer"),
    (dict(v=None), "null pointer"), (dict(start=None), "null pointer"), (dict(num_rows=-1), "negative size"),
    (dict(num_rows=(1 << 26) + 1), "2^26 rows"),
])
def test_write_refusals(kw, msg):
    lib = sphkv_lib.load()
    assert lib.sphkv_cache8_write(*_write_args(**kw)) == -1
    assert msg in lib.sphkv_last_error().decode()


@pytest.mark.parametrize("kw, msg", _SHARED + [
    (dict(out_type=-1), "unknown type"), (dict(cu=None), "one row per sequence"), (dict(start=None), "null pointer"),
    (dict(k=_FAKE + 2), "16-byte aligned"), (dict(num_rows=-1), "negative size"),
])
def test_read_refusals(kw, msg):
    lib = sphkv_lib.load()
    assert lib.sphkv_cache8_read(*_read_args(**kw)) == -1
    assert msg in lib.sphkv_last_error().decode()


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("kw, msg", _SHARED + [
    (dict(gqa=0), "gqa must be"), (dict(gqa=65), "gqa must be"), (dict(q_type=2), "q must be fp16 or bf16"),
    (dict(sm=0.0), "sm_scale"), (dict(sm=float("inf")), "sm_scale"), (dict(sm=float("nan")), "sm_scale"),
    (dict(q=None), "null pointer"), (dict(lens=None), "null pointer"), (dict(out=None), "null pointer"),
    (dict(ws=_FAKE + 4), "16-byte aligned"),
])
def test_attention_refusals(decode, kw, msg):
    lib = sphkv_lib.load()
    fn = lib.sphkv_cache8_decode if decode else lib.sphkv_cache8_prefill
    assert fn(*_attend_args(decode, **kw)) == -1
    assert msg in lib.sphkv_last_error().decode()


def test_prefill_refusals():
    lib = sphkv_lib.load()
    for kw, msg in ((dict(cu=None), "null pointer"), (dict(causal=2), "causal must be"), (dict(num_rows=-1), "negative"),
                    (dict(num_rows=1 << 22, num_kv=16, gqa=64), "too many")):
        assert lib.sphkv_cache8_prefill(*_attend_args(False, **kw)) == -1
        assert msg in lib.sphkv_last_error().decode()


def test_nothing_to_do_is_no_error():
    lib = sphkv_lib.load()
    assert lib.sphkv_cache8_write(*_write_args(num_seqs=0, num_rows=0, k=None, v=None, start=None, table=None)) == 0
    assert lib.sphkv_cache8_write(*_write_args(num_rows=0)) == 0
    assert lib.sphkv_cache8_read(*_read_args(k=None, v=None)) == 0
    assert lib.sphkv_cache8_decode(*_attend_args(True, num_seqs=0, q=None, lens=None, table=None)) == 0
    assert lib.sphkv_cache8_prefill(*_attend_args(False, num_rows=0)) == 0


def test_workspace_sizes():
    lib = sphkv_lib.load()
    for args in ((-1, 8, 4, 128), (4, 0, 4, 128), (4, 8, 0, 128), (4, 8, 65, 128), (4, 8, 4, 96)):
        assert lib.sphkv_cache8_decode_workspace_bytes(*args) == -1
        assert lib.sphkv_cache8_prefill_workspace_bytes(16, *args) == -1
    assert lib.sphkv_cache8_prefill_workspace_bytes(-1, 4, 8, 4, 128) == -1
    assert lib.sphkv_cache8_decode_workspace_bytes(4, 8, 4, 128) >= 0


# ---- refusals of the Python entries: no CPU path ------------------------------

def test_python_refuses_cpu_tensors_and_bad_formats():
    k = torch.zeros((2, 1, 16, 64), dtype=torch.uint8)
    v = torch.zeros((2, 1, 1, 64, 16), dtype=torch.uint8)
    s = torch.zeros((2, 1, 2))
    with pytest.raises(ValueError, match="GPU device"):
        kv8.Cache8(k, v, s)
    with pytest.raises(ValueError, match="fmt must be"):
        kv8.Cache8(k, v, s, "fp4")
    with pytest.raises(TypeError, match="k_codes must be torch.uint8"):
        kv8.Cache8(k.to(torch.int8), v, s)
    with pytest.raises(TypeError, match="torch.Tensor"):
        kv8.Cache8(None, v, s)


def test_what_a_cache_consists_of_is_read_only():
    """Another tensor or format in an existing cache would be checked against nothing."""
    c = object.__new__(kv8.Cache8)
    for name in ("k_codes", "v_codes", "scales", "fmt", "num_pages", "num_kv", "page_size", "dh", "device"):
        with pytest.raises(AttributeError):
            setattr(c, name, None)
    with pytest.raises(AttributeError):
        c.other = None


def test_grids_past_32_bits_are_refused():
    """Calls whose workgroups would hold 2^32 threads or more, which no launch takes: each fills its grid to 2^32."""
    lib = sphkv_lib.load()
    n = 1 << 16
    for ps, kw in ((32, dict(num_kv=256)), (64, dict(num_kv=128)), (128, dict(num_kv=64)),
                   (128, dict(num_kv=128, cu=None, num_rows=n))):
        assert lib.sphkv_cache8_write(*_write_args(**{**dict(ps=ps, num_seqs=n), **kw})) == -1
        assert "below 2^30 / page_size" in lib.sphkv_last_error().decode()
    assert lib.sphkv_cache8_prefill(*_attend_args(False, num_rows=16, num_seqs=n, num_kv=128, gqa=1)) == -1
    assert "too many (row, head) pairs" in lib.sphkv_last_error().decode()
