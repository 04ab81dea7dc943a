"""CPU tests of the 4-bit cache's and the norm's C entries: refusals before any device work, plans, and the
reference used by the GPU tests against closed forms."""
import ctypes

import numpy as np
import pytest

import kv4ref as R
import mxfa

FAKE = 1 << 20                                   # aligned, never dereferenced


def _err():
    return mxfa.lib().mxfa_last_error().decode()


def _append(shape=(2, 2, 128, 256), fmt=mxfa.C_BF16, k=FAKE, v=FAKE, ks=None, vs=None, pos=None, pos0=0, counts=None, n=1,
            cache=FAKE):
    c = mxfa.Kv4Shape(*shape) if shape else None
    return mxfa.lib().mxfa_kv4_append(c, fmt, k, ks, v, vs, pos, pos0, counts, n, cache, cache, cache, cache, None)


def _read(shape=(2, 2, 128, 256), fmt=mxfa.C_BF16, out=FAKE, st=None, pos=None, pos0=0, n=1, cache=FAKE):
    c = mxfa.Kv4Shape(*shape) if shape else None
    return mxfa.lib().mxfa_kv4_read(c, fmt, cache, cache, cache, cache, pos, pos0, n, out, st, out, st, None)


@pytest.mark.parametrize("call", [_append, _read])
def test_copy_refusals(call):
    assert call(shape=None) == 1
    for bad in ((0, 2, 128, 256), (2, 0, 128, 256), (2, 2, 48, 256), (2, 2, 0, 256), (2, 2, 128, 250), (2, 2, 128, 0)):
        assert call(shape=bad) == 1, bad
    assert call(fmt=2) == 1
    assert call(n=-1) == 1
    assert call(pos0=-1) == 1
    assert call(pos0=250, n=7) == 1 and "max_len" in _err()
    assert call(pos0=256, n=0) == 0                             # nothing to do
    assert call(pos=FAKE + 2, n=7) == 1                         # misaligned index
    assert call(cache=None) == 1 and call(cache=FAKE + 8) == 1
    assert call(n=1 << 20, pos=FAKE, shape=(1 << 12, 64, 128, 1 << 20)) == 2 and "2^32 work-items" in _err()
    assert call(n=(1 << 31) - 1, pos=FAKE, shape=((1 << 31) - 1, (1 << 31) - 1, 1024, 256)) == 2


def test_copy_strides_and_pointers():
    S = mxfa.Strides
    assert _append(ks=S(8, 8, 12)) == 1 and "K strides" in _err()
    assert _append(vs=S(4, 0, 0)) == 1 and "V strides" in _err()
    assert _append(fmt=mxfa.C_F32, vs=S(4, 2, 0)) == 1
    assert _read(st=S(0, 0, 4)) == 1
    assert _append(k=None) == 1 and _append(v=FAKE + 8) == 1
    assert _append(counts=FAKE + 1) == 1


def _params(**kw):
    a = dict(B=2, Hq=8, Hkv=2, Sq=1, Sk=200, D=128, max_len=256, causal=True, q_pos0=0, window=0, softcap=0.0, o_fmt=1)
    a.update(kw)
    return mxfa.make_kv4_params(a["B"], a["Hq"], a["Hkv"], a["Sq"], a["Sk"], a["D"], a["max_len"], causal=a["causal"],
                                q_pos0=a["q_pos0"], window=a["window"], softcap=a["softcap"], o_fmt=a["o_fmt"],
                                scale=kw.get("scale"))


def _attend(p, q=FAKE, qs=None, cache=FAKE, lens=None, o=FAKE, os_=None, ws=FAKE, ws_bytes=1 << 40):
    return mxfa.lib().mxfa_kv4_attention(p, q, qs, cache, cache, cache, cache, lens, o, os_, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", [
    (dict(B=0), 1), (dict(Hkv=0), 1), (dict(Hq=3), 1), (dict(Sq=0), 1), (dict(Sk=0), 1), (dict(D=48), 1), (dict(D=96), 2),
    (dict(max_len=128), 1), (dict(max_len=200), 1), (dict(q_pos0=-1), 1), (dict(window=-1), 1), (dict(softcap=-1.0), 1),
    (dict(softcap=float("nan")), 1), (dict(scale=0.0), 1), (dict(scale=float("inf")), 1), (dict(o_fmt=2), 1),
    (dict(max_len=1 << 25), 2),                                   # 2^31 bytes of codes in a head
    (dict(q_pos0=1 << 30), 2), (dict(Hq=1 << 21, Hkv=1, Sq=1 << 10), 2),
    (dict(B=1 << 26, Sq=1 << 14), 2),
])
def test_attention_refusals(kw, status):
    p = _params(**kw)
    assert mxfa.lib().mxfa_kv4_attention_plan(p, None, None) == status, _err()
    assert _attend(p) == status
    with pytest.raises(mxfa.MxfaError):
        mxfa.kv4_attention_plan(p)


def test_attention_pointers_strides_and_workspace():
    S, p = mxfa.Strides, _params()
    assert _attend(None) == 1
    for kw in (dict(q=None), dict(q=FAKE + 8), dict(cache=None), dict(o=None), dict(o=FAKE + 4), dict(lens=FAKE + 2)):
        assert _attend(p, **kw) == 1, kw
    assert _attend(p, qs=S(8, 8, 4)) == 1 and "q strides" in _err()
    assert _attend(p, os_=S(8, 4, 8)) == 1 and "o strides" in _err()
    assert _attend(_params(o_fmt=0), os_=S(8, 2, 8)) == 1
    long = _params(B=1, Sk=100000, max_len=100000)
    shares, need = mxfa.kv4_attention_plan(long)
    assert shares > 1 and need >= 2 * 4 * shares * (128 + 2) * 4
    assert _attend(long, ws=None) == 5 and _attend(long, ws_bytes=need - 1) == 5 and "workspace needs" in _err()
    assert _attend(long, ws=FAKE + 8) == 1


def test_plan_of_short_caches_and_large_batches_needs_no_workspace():
    for kw in (dict(), dict(B=600), dict(Sq=900, Sk=900, max_len=1024), dict(B=2048, Sk=8192, max_len=8192)):
        assert mxfa.kv4_attention_plan(_params(**kw)) == (0, 0), kw


def _norm(rows=4, cols=256, fmt=mxfa.C_BF16, eps=1e-6, off=0.0, ld=0, x=FAKE, res=None, w=FAKE, h=None, codes=FAKE, sc=FAKE):
    p = mxfa.NormParams(rows, cols, fmt, eps, off, ld)
    return mxfa.lib().mxfa_rmsnorm_quantize(p, x, res, w, h, codes, sc, None)


def test_norm_refusals():
    assert mxfa.lib().mxfa_rmsnorm_quantize(None, FAKE, None, FAKE, None, FAKE, FAKE, None) == 1
    assert _norm(rows=0) == 0
    for kw in (dict(rows=-1), dict(cols=0), dict(cols=48), dict(fmt=3), dict(eps=-1.0), dict(eps=float("nan")),
               dict(off=float("inf")), dict(ld=3), dict(ld=-1), dict(x=None), dict(x=FAKE + 8), dict(w=None), dict(codes=None),
               dict(sc=None), dict(res=FAKE), dict(h=FAKE + 4), dict(res=FAKE + 4, h=FAKE)):
        assert _norm(**kw) == 1, kw
    assert _norm(rows=1 << 33) == 2 and "2^32 work-items" in _err()


def test_reference_rule_on_the_values_themselves():
    """Every level times a power of two is its own code; halfway points go to the even one."""
    x = np.zeros((1, 32), np.float32)
    x[0, :8], x[0, 8:16] = R.LEVELS * 2.0 ** -5, -R.LEVELS * 2.0 ** -5
    codes, sc = R.quantize(x)
    assert sc[0, 0] == 127 - 5 and list(codes[0, :8]) == list(range(8)) and list(codes[0, 9:16]) == list(range(9, 16))
    assert np.array_equal(R.values(codes, sc), x.astype(np.float64))
    x[0, :7], x[0, 7] = R.STEPS, 6.0
    assert list(R.quantize(x)[0][0, :7]) == [0, 2, 2, 4, 4, 6, 6]
    t, b = np.meshgrid(np.arange(64), np.arange(4), indexing="ij")
    assert sorted(R.scale_place(t, b, 4).ravel()) == list(range(256))
    by = np.random.default_rng(0).integers(0, 256, (1, 2, 64, 4)).astype(np.uint8)
    assert np.array_equal(R.scales_by_token(R.scales_in_cache(by)), by)


def test_values_past_32_bits_are_refused_not_cut():
    for kw in (dict(window=1 << 32), dict(q_pos0=1 << 32), dict(Sk=1 << 32), dict(max_len=(1 << 32) + 256), dict(B=(1 << 32) + 1)):
        with pytest.raises(mxfa.MxfaError, match="32 bits"):
            _params(**kw)
    for args in ((0, 1, 64, 32), (1, 1, 48, 32), (1, 1, 64, 33), (1, 1, 64, 0), (1, 1, 64, (1 << 32) + 32)):
        with pytest.raises(mxfa.MxfaError):
            mxfa.Kv4Cache(*args, device="cpu")


def test_scales_that_leave_the_float_range_are_refused():
    for kw in (dict(scale=3e38), dict(softcap=3e38), dict(softcap=1e-42)):
        assert _attend(_params(**kw)) == 1 and "log2 units" in _err(), kw
