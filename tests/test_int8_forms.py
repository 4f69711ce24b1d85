"""The kernels that gcdr_k_i8_gemm chooses from: which one a call takes (gcdr_k_i8_gemm_form, on the host), and the
results of each of them against the 64-bit form (on the GPU), so that a change of the choice cannot leave a kernel
without a test."""
import ctypes
import random

import pytest

from sdcb.gcdrnet_b200 import I8GemmDesc, I8GemmForm, lib

OK, ARG, RANGE = 0, 1, 2
DOT, NARROW, WIDE, PAIR = 1, 2, 3, 4
SMS = 148
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
CODE = {"f16": 0, "bf16": 1, "f32": 2}


def _desc(M, N, K, dtype, pad=0, off=0):
    ld = -(-K // 16) * 16
    return I8GemmDesc(M=M, N=N, K=K, ldx=ld, ldw=ld, dtype=CODE[dtype], out=(1 << 30) + off, ldo=N + pad)


def form_of(d, sms=SMS):
    """((form, tile, split, epilogue warps, accumulators, tensor store), the whole answer)"""
    f = I8GemmForm()
    assert lib().gcdr_k_i8_gemm_form(ctypes.byref(d), sms, ctypes.byref(f)) == OK
    return (f.form, f.tile, f.split, f.epilogue_warps, f.accumulators, f.tensor_store), f


# Every kernel the choice reaches: (form, tile, split, epilogue warps, accumulators, tensor store) -> for 16-bit and for
# fp32 results M, N, K and what the result's pitch is longer than N.  K is long enough to go round the operand ring
# where the form is chosen for such a K at all; M and N end inside a tile.
FORMS = {
    (DOT, 1, 0, 0, 0, 0): [(3, 301, 1030, 1), (2, 301, 1030, 3)],
    (DOT, 2, 0, 0, 0, 0): [(4, 4099, 1030, 1), (1, 4101, 2070, 3)],
    (NARROW, 16, 1, 8, 2, 0): [(8, 281, 1652, 4), (5, 27, 1656, 8)],
    (NARROW, 16, 2, 8, 2, 0): [(5, 5507, 3506, 8), (5, 4860, 3218, 2)],
    (NARROW, 16, 4, 8, 2, 0): [(5, 1584, 6438, 0), (5, 1625, 6070, 2)],
    (NARROW, 16, 8, 8, 2, 0): [(5, 6, 12186, 4), (5, 4, 12161, 2)],
    (NARROW, 32, 1, 8, 2, 0): [(34, 6720, 1605, 4), (38, 6400, 1441, 2)],
    (NARROW, 32, 2, 8, 2, 0): [(17, 4896, 2779, 2), (17, 5772, 2763, 4)],
    (NARROW, 32, 4, 8, 2, 0): [(17, 2448, 5971, 2), (17, 2358, 5911, 8)],
    (NARROW, 32, 8, 8, 2, 0): [(17, 784, 11199, 1), (17, 908, 11812, 4)],
    (NARROW, 64, 1, 8, 2, 0): [(129, 4802, 1453, 0), (134, 5285, 1160, 0)],
    (NARROW, 64, 2, 8, 2, 0): [(34, 5185, 6639, 1), (35, 4928, 6677, 1)],
    (NARROW, 64, 4, 8, 2, 0): [(33, 3592, 5950, 4), (36, 3248, 6557, 2)],
    (NARROW, 64, 8, 8, 2, 0): [(39, 793, 19791, 4), (33, 816, 17997, 1)],
    (NARROW, 128, 1, 8, 2, 0): [(161, 6735, 4960, 4), (163, 6880, 915, 1)],
    (NARROW, 128, 2, 8, 2, 0): [(97, 4787, 10653, 0), (70, 6464, 10206, 0)],
    (NARROW, 128, 4, 8, 2, 0): [(65, 3280, 12227, 2), (66, 3721, 10602, 8)],
    (NARROW, 128, 8, 8, 2, 0): [(99, 1381, 28081, 8), (99, 1381, 28081, 8)],
    (WIDE, 64, 1, 8, 1, 0): [(5, 2, 1137, 2), (5, 16, 1142, 4)],
    (WIDE, 64, 1, 8, 2, 0): [(641, 3089, 1059, 4), (513, 3808, 1191, 1)],
    (WIDE, 64, 1, 8, 2, 1): [(685, 3104, 1116, 0), (809, 2800, 1073, 0)],
    (WIDE, 64, 1, 16, 4, 0): [(38095, 30, 2, 1), (701, 3391, 886, 4)],
    (WIDE, 64, 1, 16, 4, 1): [(19733, 88, 3, 0), (468, 5152, 882, 0)],
    (WIDE, 128, 1, 8, 1, 0): [(129, 6544, 1057, 0), (169, 6523, 868, 1)],
    (WIDE, 128, 1, 8, 2, 0): [(680, 6519, 826, 0), (564, 7826, 842, 4)],
    (WIDE, 128, 1, 8, 2, 1): [(661, 6160, 951, 0), (523, 8000, 989, 8)],
    (WIDE, 128, 1, 16, 4, 0): [(543, 8495, 754, 8), (529, 7778, 539, 0)],
    (WIDE, 128, 1, 16, 4, 1): [(687, 6928, 633, 0), (532, 7984, 518, 0)],
    (WIDE, 256, 1, 8, 1, 0): [(356, 6480, 525, 0), (655, 4844, 518, 4)],
    (WIDE, 256, 1, 8, 2, 0): [(902, 7424, 916, 4), (3392, 2782, 1030, 4)],
    (WIDE, 256, 1, 8, 2, 1): [(925, 7856, 689, 8), (1697, 5392, 954, 8)],
    (WIDE, 256, 1, 16, 2, 0): [(1403, 7245, 387, 8), (4204, 2210, 557, 2)],
    (WIDE, 256, 1, 16, 2, 1): [(2006, 6728, 507, 0), (1484, 6464, 519, 4)],
    (PAIR, 256, 1, 8, 1, 0): [(276, 6448, 2104, 0), (284, 8192, 1697, 4)],
    (PAIR, 256, 1, 8, 2, 0): [(574, 8284, 1824, 4), (779, 6894, 2949, 2)],
    (PAIR, 256, 1, 8, 2, 1): [(527, 7632, 1688, 0), (1047, 6960, 1318, 0)],
}
CASES = [(form, dtype) + sizes[dtype == "f32"] for form, sizes in FORMS.items() for dtype in ("f16", "bf16", "f32")]


def _id(c):
    return "%s%d_split%d_%dwarps_%dacc%s_%s" % (("", "dot", "narrow", "wide", "pair")[c[0][0]], c[0][1], c[0][2], c[0][3], c[0][4],
                                               "_store" if c[0][5] else "", c[1])


@pytest.mark.parametrize("case", CASES, ids=_id)
def test_the_case_takes_its_form(case):
    form, dtype, M, N, K, pad = case
    assert form_of(_desc(M, N, K, dtype, pad))[0] == form


def test_no_size_takes_a_form_without_a_case():
    rng = random.Random(11)

    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    for _ in range(60000):
        M, N, K = log(1, 200000), log(1, 30000), log(1, 131071)
        if rng.random() < 0.5:
            N = -(-N // 16) * 16
        if rng.random() < 0.5:
            K = min(-(-K // 128) * 128, 131071)
        dtype, pad, off = rng.choice(list(CODE)), rng.choice([0, 0, 1, 2, 4, 8]), rng.choice([0, 0, 8, 4])
        d = _desc(M, N, K, dtype, pad, off)
        form, f = form_of(d)
        assert form in FORMS, (M, N, K, dtype, pad, off)
        if form[0] == DOT:
            assert M <= 4 and f.units * f.tile >= N
            continue
        # what the kernel needs of its launch: tiles that cover the result, TMEM columns, shared memory
        rows, cols = {NARROW: (N, M), WIDE: (M, N), PAIR: (M, N)}[form[0]]
        high = 256 if form[0] == PAIR else 128
        assert f.units == -(-rows // high) * -(-cols // f.tile)
        assert 32 <= f.accumulators * f.tile <= 512 and f.accumulators * f.tile in (32, 64, 128, 256, 512)
        assert 1 <= f.split <= -(-K // 128)
        stage = 128 * (128 + f.tile // (2 if form[0] == PAIR else 1))
        extra = f.epilogue_warps * 32 * (128 if f.epilogue_warps == 16 else 64) + 8192
        if form[0] == NARROW:
            extra = (f.tile + f.split) * 129 * 4 if f.split > 1 else 0
        assert 2 <= f.stages <= 12 and 1024 + f.stages * stage + -(-extra // 16) * 16 + 288 <= 227 * 1024
        if f.tensor_store:
            assert (off | (N + pad) * SIZE[dtype] | N * SIZE[dtype]) % 16 == 0


def test_form_on_other_devices():
    """The choice holds together on other numbers of SMs too."""
    for sms in (2, 3, 100, 132, 147, 160):
        for M, N, K in ((1, 64, 64), (16, 1000, 4096), (2000, 512, 512), (60000, 256, 256), (9000, 4096, 4096)):
            form, f = form_of(_desc(M, N, K, "f16"), sms)
            assert f.units >= 1 and form[0] in (DOT, NARROW, WIDE, PAIR)


def test_form_of_nothing():
    form, f = form_of(_desc(0, 64, 64, "f16"))
    assert form == (0, 0, 0, 0, 0, 0) and f.units == 0


@pytest.mark.parametrize("want,bad", [(ARG, {"dtype": 5}), (RANGE, {"M": -1}), (RANGE, {"N": 0}), (RANGE, {"K": 0}), (RANGE, {"K": 131072}),
                                      (RANGE, {"wait_cycles": -1}), (RANGE, {"sms": 1}), (RANGE, {"sms": -5}), (RANGE, {"sms": 5000}),
                                      (ARG, {"form": None}), (ARG, {"desc": None})], ids=str)
def test_form_refuses(want, bad):
    d, f = _desc(64, 64, 64, "f16"), I8GemmForm()
    for k in ("dtype", "M", "N", "K", "wait_cycles"):
        if k in bad:
            setattr(d, k, bad[k])
    assert lib().gcdr_k_i8_gemm_form(None if "desc" in bad else ctypes.byref(d), bad.get("sms", SMS),
                                     None if "form" in bad else ctypes.byref(f)) == want


def _taken(x, w, out, **more):
    from sdcb.gcdrnet_b200 import lib
    from int8_util import code
    d = I8GemmDesc(M=x.shape[0], N=w.shape[0], K=x.shape[1], ldx=x.stride(0), ldw=w.stride(0), dtype=code(out.dtype),
                   out=out.data_ptr(), ldo=out.stride(0), **more)
    return form_of(d, lib().gcdr_device_sms())[0]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=_id)
def test_results_of_every_form(case):
    from int8_util import i8_gemm, ref_product, strided, torch_dtype, untouched, worst
    from test_gpu_int8 import _operands
    form, dtype, M, N, K, pad = case
    dt = torch_dtype(dtype)
    x, xs, w, ws, b = _operands(M, N, K, M + N + K)
    for relu, bias in ((False, b), (True, None)):
        out, buf = strided(M, N, N + pad, dt, 123.0)
        assert _taken(x, w, out) == form
        assert i8_gemm(x, xs, w, ws, bias, out, relu) == 0
        want, bound = ref_product(x, xs, w, ws, bias, relu, dt)
        assert worst(out, want, bound) <= 1.0
        assert untouched(out, buf, 123.0)


# a case of each kernel's way out when a wait ends (the largest tiles and clusters, one and several units a CTA)
GIVE_UP = [(NARROW, 128, 1, 8, 2, 0), (NARROW, 16, 2, 8, 2, 0), (NARROW, 64, 4, 8, 2, 0), (NARROW, 16, 8, 8, 2, 0),
           (WIDE, 64, 1, 8, 1, 0), (WIDE, 128, 1, 8, 2, 0), (WIDE, 128, 1, 8, 2, 1), (WIDE, 64, 1, 16, 4, 0), (WIDE, 128, 1, 16, 4, 1),
           (WIDE, 256, 1, 16, 2, 1), (PAIR, 256, 1, 8, 1, 0), (PAIR, 256, 1, 8, 2, 0), (PAIR, 256, 1, 8, 2, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("form", GIVE_UP, ids=lambda f: _id((f, "")))
def test_every_kernel_gives_up_and_reports_timeout(form, dtype):
    """The test hook issues no copies and no MMAs, so every role's first wait runs out (0.2 ms): nothing is written, the
    status says so once, the kernel's TMEM is free again and the next call of the same kernel is right."""
    import time

    import torch
    from int8_util import i8_gemm, ref_product, strided, torch_dtype, worst
    from test_gpu_int8 import _operands
    L = lib()
    M, N, K, pad = FORMS[form][dtype == "f32"]
    dt = torch_dtype(dtype)
    x, xs, w, ws, b = _operands(M, N, K, M + N + K)
    out, buf = strided(M, N, N + pad, dt, float("nan"))
    want, bound = ref_product(x, xs, w, ws, b, False, dt)
    torch.cuda.synchronize()
    assert L.gcdr_k_status(None) == OK
    assert _taken(x, w, out, timeout_probe=1) == form
    for _ in range(3):
        t0 = time.perf_counter()
        assert i8_gemm(x, xs, w, ws, b, out, wait_cycles=400_000, timeout_probe=1) == 0
        assert L.gcdr_k_status(None) == 5
        assert time.perf_counter() - t0 < 5.0
        assert torch.isnan(buf).all().item(), "the probe wrote outputs"
        assert L.gcdr_k_status(None) == OK
    assert i8_gemm(x, xs, w, ws, b, out) == 0
    assert L.gcdr_k_status(None) == OK
    assert worst(out, want, bound) <= 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("form", GIVE_UP, ids=lambda f: _id((f, "")))
def test_a_wait_that_ends_in_the_middle(form):
    """A limit so short that real work runs into it: copies and MMAs are on their way when the kernel gives up.  It drains
    them and returns; what it has stored is right, what it has not stands as it was, and the status tells the two apart."""
    import time

    import torch
    from int8_util import i8_gemm, ref_product, strided, torch_dtype, worst
    from test_gpu_int8 import _operands
    L = lib()
    M, N, K, pad = FORMS[form][0]
    dt = torch_dtype("f16")
    x, xs, w, ws, b = _operands(M, N, K, M + N + K)
    want, bound = ref_product(x, xs, w, ws, b, False, dt)
    torch.cuda.synchronize()
    assert L.gcdr_k_status(None) == OK
    for limit in (1, 3000, 30000, 1):
        out, buf = strided(M, N, N + pad, dt, float("nan"))
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        assert i8_gemm(x, xs, w, ws, b, out, wait_cycles=limit) == 0
        status = L.gcdr_k_status(None)
        assert time.perf_counter() - t0 < 0.5, "waited for copies that nothing had issued"
        assert status in (OK, 5)
        done = ~torch.isnan(out)
        assert status == 5 or done.all()
        assert worst(torch.where(done, out.double(), want), want, bound) <= 1.0
        assert torch.isnan(buf).sum() >= buf.numel() - M * N
        assert L.gcdr_k_status(None) == OK
    assert i8_gemm(x, xs, w, ws, b, out) == 0
    assert worst(out, want, bound) <= 1.0
