"""Refusals of the 8-bit token operators on the host: every check of sizes, codes, alignment and overlap comes
before the first device call, so no GPU is needed and the made-up addresses are never read."""
import ctypes

import pytest

from sdcb.gcdrnet_b200 import ArgumentError, ArgumentOutOfRangeError, BlockNormDesc, I8GemmDesc, check, lib

OK, ARG, RANGE = 0, 1, 2
A = 1 << 30                # made-up addresses, 256 MB apart
AT = [A + (k << 28) for k in range(12)]
NAN = float("nan")


def _quant(x=AT[0], dtype=0, rows=4, C=64, ldx=64, q=AT[1], ldq=64, scale=AT[2]):
    return lib().gcdr_k_quant_rows(x, dtype, rows, C, ldx, q, ldq, scale, None)


@pytest.mark.parametrize("want,bad", [
    (ARG, {"dtype": 3}), (ARG, {"dtype": -1}), (RANGE, {"rows": -1}), (RANGE, {"C": 0}), (RANGE, {"C": 32769, "ldx": 40000, "ldq": 40000}),
    (ARG, {"x": None}), (ARG, {"q": None}), (ARG, {"scale": None}), (RANGE, {"ldx": 63}), (RANGE, {"ldq": 63}), (RANGE, {"ldx": -64}),
    (ARG, {"x": A + 1}), (ARG, {"x": A + 2, "dtype": 2}), (ARG, {"scale": AT[2] + 2}), (RANGE, {"rows": 1 << 62}),
    (RANGE, {"ldx": 1 << 60}), (RANGE, {"rows": 1 << 40, "ldx": 1 << 30}), (ARG, {"q": A}), (ARG, {"q": A + 500}), (ARG, {"scale": AT[1] + 8}),
    (OK, {"rows": 0, "x": None, "q": None, "scale": None}),
], ids=str)
def test_quant_rows_refuses(want, bad):
    assert _quant(**bad) == want


def _gemm(**kw):
    d = dict(M=8, N=32, K=64, x=AT[0], ldx=64, xs=AT[1], w=AT[2], ldw=64, ws=AT[3], bias=AT[4], relu=0, dtype=0, out=AT[5],
             ldo=32)
    d.update(kw)
    return lib().gcdr_k_i8_gemm(ctypes.byref(I8GemmDesc(**d)), None)


@pytest.mark.parametrize("want,bad", [
    (ARG, {"dtype": 3}), (RANGE, {"M": -1}), (RANGE, {"M": 1 << 31}), (RANGE, {"N": 0}), (RANGE, {"K": 0}),
    (RANGE, {"K": 131072, "ldx": 131072, "ldw": 131072}), (RANGE, {"wait_cycles": -1}),
    (ARG, {"x": None}), (ARG, {"xs": None}), (ARG, {"w": None}), (ARG, {"ws": None}), (ARG, {"out": None}),
    (ARG, {"x": A + 8}), (ARG, {"w": AT[2] + 4}), (ARG, {"ldx": 72}), (ARG, {"ldw": 65}), (RANGE, {"ldx": 48}), (RANGE, {"ldw": 0}),
    (RANGE, {"ldo": 31}), (ARG, {"out": AT[5] + 1}), (ARG, {"bias": AT[4] + 1}), (ARG, {"xs": AT[1] + 2}),
    (ARG, {"out": AT[0]}), (ARG, {"out": AT[2] + 64}), (ARG, {"out": AT[4]}), (RANGE, {"ldo": 1 << 60}),
    (OK, {"M": 0, "x": None, "out": None}),
], ids=str)
def test_i8_gemm_refuses(want, bad):
    assert _gemm(**bad) == want


def test_null_descriptors():
    assert lib().gcdr_k_i8_gemm(None, None) == ARG
    assert lib().gcdr_k_block_norm(None, None) == ARG


def _norm(**kw):
    d = dict(rows=4, C=64, dtype=0, x=AT[0], ldx=64, f=AT[1], ldf=64, post=1, g1=AT[2], b1=AT[3], eps1=1e-5, gate=AT[4],
             ldg=64, gate_rows=2, res_scale=1.0, r=AT[5], ldr=64, pre=2, g2=AT[6], b2=None, eps2=1e-5, y=AT[7], ldy=64,
             q=AT[8], ldq=64, qs=AT[9])
    d.update(kw)
    return lib().gcdr_k_block_norm(ctypes.byref(BlockNormDesc(**d)), None)


@pytest.mark.parametrize("want,bad", [
    (ARG, {"dtype": 7}), (RANGE, {"rows": -3}), (RANGE, {"C": 0}), (RANGE, {"C": 32769}), (ARG, {"post": 3}), (ARG, {"pre": -1}),
    (ARG, {"eps1": -1.0}), (ARG, {"eps2": NAN}), (RANGE, {"gate_rows": 0}), (ARG, {"x": None, "f": None, "post": 0, "gate": None}),
    (ARG, {"f": None}), (ARG, {"f": None, "post": 0}), (ARG, {"r": None, "y": None, "q": None, "qs": None}), (ARG, {"qs": None}),
    (ARG, {"q": None}), (RANGE, {"ldx": 63}), (RANGE, {"ldf": 1}), (RANGE, {"ldg": 60}), (RANGE, {"ldr": 63}), (RANGE, {"ldy": 0}),
    (RANGE, {"ldq": 63}), (ARG, {"x": A + 1}), (ARG, {"g1": AT[2] + 2}), (ARG, {"b1": AT[3] + 1}), (ARG, {"qs": AT[9] + 1}),
    (ARG, {"r": AT[0], "ldr": 72}), (ARG, {"r": AT[0] + 2}), (ARG, {"y": AT[5]}), (ARG, {"q": AT[0]}), (ARG, {"r": AT[4]}),
    (ARG, {"y": AT[2], "rows": 1, "dtype": 2}), (ARG, {"qs": AT[6]}), (OK, {"rows": 0, "x": None, "f": None, "r": None}),
], ids=str)
def test_block_norm_refuses(want, bad):
    assert _norm(**bad) == want


def test_status_raises():
    check(0)
    with pytest.raises(ArgumentError):
        check(ARG)
    with pytest.raises(ArgumentOutOfRangeError):
        check(RANGE)
