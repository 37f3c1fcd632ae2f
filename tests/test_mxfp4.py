"""Microscaled 4-bit matrices without a GPU: sizes, the oracle against hand-made values, and every refusal of the C ABI
(arguments are checked before the context)."""
import ctypes as C

import numpy as np
import pytest

from aiehlc_b200 import _capi
from oracle import mxfp4 as X

BUF = C.create_string_buffer(4096)
P = (C.addressof(BUF) + 15) // 16 * 16     # an aligned address; nothing is read through it: the context is null


def _refused(rc, code, text):
    assert rc == code, _capi.load().aiehlc_last_error()
    assert text in _capi.load().aiehlc_last_error().decode()


@pytest.mark.parametrize("rows,cols,pitch,scales", [(1, 1, 16, 512), (1, 32, 16, 512), (1, 33, 32, 512), (128, 128, 64, 512),
                                                    (129, 128, 64, 1024), (128, 129, 80, 1024), (1000, 2999, 1504, 98304)])
def test_sizes(rows, cols, pitch, scales):
    lib = _capi.load()
    assert lib.aiehlc_mxfp4_pitch(cols) == pitch and lib.aiehlc_mxfp4_scale_bytes(rows, cols) == scales
    assert lib.aiehlc_mxfp4_pitch(0) == 0 and lib.aiehlc_mxfp4_scale_bytes(0, cols) == 0
    assert lib.aiehlc_mxfp4_scale_bytes(1 << 33, 1 << 20) == (1 << 26) * (1 << 13) * 512   # past 32 bits


def test_oracle_known_answers():
    row = np.array([[0, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 5.1, 7.9, -0.3, -1.0] + [0.0] * 19])
    want = [0, 0, 0.5, 1, 1, 2, 2, 4, 4, 6, 6, -0.5, -1] + [0.0] * 19       # max 7.9: e = 0; ties go to the even code
    codes, scales = X.quantize(row)
    assert scales.tolist() == [[127]] and X.values(codes, scales, 32)[0].tolist() == want
    assert X.rounded([[8.0, 3.0, 0.5]])[0].tolist() == [8.0, 3.0, 0.0]       # e = 1: 0.25 is a tie and goes to 0
    assert X.quantize([[0.0]])[1].tolist() == [[0]] and X.quantize([[2.0 ** -149]])[1].tolist() == [[0]]
    assert np.isnan(X.rounded([[1.0, np.inf]])).all() and np.isnan(X.rounded([[np.nan, 2.0]])).all()
    s = np.arange(129 * 5).reshape(129, 5).astype(np.uint8)
    t = X.tile_scales(s)
    assert t.size == 2 * 2 * 512 and (X.untile_scales(t, 129, 160) == s).all() and t[33 % 32 * 16 + 4 + 2] == s[33, 2]


def test_quantize_refusals():
    f = _capi.load().aiehlc_quantize_mxfp4_dev
    ok = dict(x=P, type=1, rows=4, cols=64, ld=64, q=P, qs=P, t=P, ts=P)

    def call(**kw):
        a = {**ok, **kw}
        return f(None, a["x"], a["type"], a["rows"], a["cols"], a["ld"], a["q"], a["qs"], a["t"], a["ts"], None)
    inv, uns = _capi.ERR_INVALID, _capi.ERR_UNSUPPORTED
    _refused(call(), inv, "null context")
    _refused(call(type=3), inv, "unknown type")
    _refused(call(type=-1), inv, "unknown type")
    _refused(call(rows=-1), inv, "negative")
    _refused(call(cols=-1, ld=0), inv, "negative")
    _refused(call(ld=63), inv, "pitch")
    _refused(call(x=None), inv, "null matrix")
    _refused(call(x=P + 1), inv, "misaligned")
    _refused(call(x=P + 2, type=0), inv, "misaligned")
    _refused(call(q=None, qs=None, t=None, ts=None), inv, "no output")
    _refused(call(q=None), inv, "null codes")
    _refused(call(qs=None), inv, "null codes")
    _refused(call(ts=None), inv, "null codes")
    _refused(call(q=P + 8), inv, "16-byte")
    _refused(call(ts=P + 4), inv, "16-byte")
    _refused(call(rows=1 << 40, cols=1 << 20, ld=1 << 20), uns, "2^31 tiles")
    _refused(call(rows=(1 << 62), cols=(1 << 62), ld=(1 << 62)), uns, "2^31 tiles")
    _refused(call(rows=0, q=None, qs=None, t=None, ts=None), inv, "null context")   # empty: nothing else is looked at


def test_dequantize_refusals():
    f = _capi.load().aiehlc_dequantize_mxfp4_dev
    ok = dict(q=P, qs=P, rows=4, cols=64, y=P, type=1, ld=64)

    def call(**kw):
        a = {**ok, **kw}
        return f(None, a["q"], a["qs"], a["rows"], a["cols"], a["y"], a["type"], a["ld"], None)
    inv = _capi.ERR_INVALID
    _refused(call(), inv, "null context")
    _refused(call(type=7), inv, "unknown type")
    _refused(call(cols=-5, ld=0), inv, "negative")
    _refused(call(ld=10), inv, "pitch")
    _refused(call(y=None), inv, "null matrix")
    _refused(call(y=P + 1), inv, "misaligned")
    _refused(call(q=None), inv, "null codes")
    _refused(call(qs=P + 1), inv, "16-byte")


def test_gemm_refusals():
    f = _capi.load().aiehlc_gemm_mxfp4_dev
    ok = dict(A=P, As=P, B=P, Bs=P, C=P, type=1, M=4, N=8, K=64, ldc=8, acc=0)

    def call(**kw):
        a = {**ok, **kw}
        return f(None, a["A"], a["As"], a["B"], a["Bs"], a["C"], a["type"], a["M"], a["N"], a["K"], a["ldc"], a["acc"], None)
    inv, uns = _capi.ERR_INVALID, _capi.ERR_UNSUPPORTED
    _refused(call(), inv, "null context")
    _refused(call(type=5), inv, "unknown type")
    _refused(call(M=-1), inv, "negative")
    _refused(call(N=-1, ldc=0), inv, "negative")
    _refused(call(K=-1), inv, "negative")
    _refused(call(K=(1 << 26) + 1), uns, "2^26")
    _refused(call(M=(1 << 30) + 1), uns, "2^30")
    _refused(call(M=1 << 30, N=1 << 30, ldc=1 << 30), uns, "too many output tiles")
    _refused(call(acc=1), uns, "only f32")
    _refused(call(acc=1, type=2), uns, "only f32")
    _refused(call(ldc=7), inv, "pitch")
    _refused(call(C=None), inv, "null or misaligned C")
    _refused(call(C=P + 1), inv, "null or misaligned C")
    _refused(call(A=None), inv, "null codes")
    _refused(call(Bs=None), inv, "null codes")
    _refused(call(B=P + 4), inv, "16-byte")
    _refused(call(As=P + 8), inv, "16-byte")
    _refused(call(K=0, A=None, As=None, B=None, Bs=None), inv, "null context")


def test_gemm_to_mxfp4_refusals():
    f = _capi.load().aiehlc_gemm_mxfp4_mxfp4_dev
    ok = dict(A=P, As=P, B=P, Bs=P, C=P, Cs=P, M=4, N=8, K=64)

    def call(**kw):
        a = {**ok, **kw}
        return f(None, a["A"], a["As"], a["B"], a["Bs"], a["C"], a["Cs"], a["M"], a["N"], a["K"], None)
    inv, uns = _capi.ERR_INVALID, _capi.ERR_UNSUPPORTED
    _refused(call(), inv, "null context")
    _refused(call(M=-1), inv, "negative")
    _refused(call(N=(1 << 30) + 1), uns, "2^30")
    _refused(call(C=None), inv, "null codes")
    _refused(call(Cs=None), inv, "null codes")
    _refused(call(Cs=P + 2), inv, "16-byte")
    _refused(call(A=P + 2), inv, "16-byte")
