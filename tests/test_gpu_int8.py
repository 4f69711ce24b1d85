"""The 8-bit token operators (gcdr_k_quant_rows, gcdr_k_i8_gemm, gcdr_k_block_norm) against plain 64-bit forms
(int8_util.py), at sizes, pitches and values where they can go wrong.  Bounds count the roundings of each
formula; integer results have to be equal."""
import numpy as np
import pytest

import golden_data as G
from int8_util import (DTYPES, LAYER, RMS, U, block_norm, i8_gemm, quant_rows, ref_block, ref_product, ref_quant, stored,
                       strided, torch_dtype, untouched, worst)

pytestmark = pytest.mark.gpu


def _gen(seed):
    import torch
    return torch.Generator(device="cuda:0").manual_seed(seed)


def _rand(g, *shape, scale=1.0, dtype=None):
    import torch
    t = torch.randn(*shape, generator=g, device="cuda:0") * scale
    return t if dtype is None else t.to(dtype)


# ------------------------------------------------------------------ rows to int8

QUANT_SIZES = [(1, 1), (3, 7), (5, 8), (33, 64), (17, 65), (9, 128), (31, 160), (7, 255), (40, 256), (11, 512), (13, 513),
               (6, 1000), (5, 1024), (4, 1037), (3, 2048), (3, 4096), (2, 4100), (3, 8192), (2, 16384), (2, 16385),
               (2, 32768), (1, 32767), (1201, 96)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", QUANT_SIZES, ids=lambda s: "%dx%d" % s)
def test_quant_rows(size, dtype):
    import torch
    rows, C = size
    dt = torch_dtype(dtype)
    x = _rand(_gen(rows * C), rows, C).to(dt)
    q = torch.full((rows, C), 99, dtype=torch.int8, device="cuda:0")
    s = torch.full((rows,), -1.0, device="cuda:0")
    assert quant_rows(x, q, s) == 0
    wq, ws = ref_quant(x)
    assert torch.equal(q, wq)
    assert torch.equal(s, ws)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C,ldx,ldq", [(40, 48, 64), (41, 43, 47), (256, 260, 257), (520, 1040, 528), (2049, 2051, 2064)])
def test_quant_rows_pitches(C, ldx, ldq, dtype):
    """Rows apart, at pitches that are multiples of no vector: the space between them stays as it was."""
    import torch
    dt = torch_dtype(dtype)
    x, xb = strided(9, C, ldx, dt, float("inf"))     # reading past a row's end would show
    x.copy_(_rand(_gen(C), 9, C))
    q, qb = strided(9, C, ldq, torch.int8, 99)
    s = torch.full((9,), -1.0, device="cuda:0")
    assert quant_rows(x, q, s) == 0
    wq, ws = ref_quant(x)
    assert torch.equal(q, wq) and torch.equal(s, ws)
    assert untouched(q, qb, 99)


def test_quant_rows_borders():
    """Quotients on the border between two steps, and next to it: ties go to the even one."""
    import torch
    # max 127: q = x, so x = k + 1/2 lies on a border; max 254: q = x / 2
    k = torch.arange(-126, 127, device="cuda:0").float() + 0.5
    near = torch.cat([k, torch.nextafter(k, torch.full_like(k, 999.0)), torch.nextafter(k, torch.full_like(k, -999.0))])
    rows = [torch.cat([near * m, torch.tensor([127.0 * m], device="cuda:0")]) for m in
            (1.0, 2.0, 2.0 ** -100, 2.0 ** 100, 2.0 ** -126, 2.0 ** 120, 3.0)]
    x = torch.stack(rows)
    q = torch.zeros(x.shape, dtype=torch.int8, device="cuda:0")
    s = torch.zeros(len(rows), device="cuda:0")
    assert quant_rows(x, q, s) == 0
    wq, ws = ref_quant(x)
    assert torch.equal(q, wq) and torch.equal(s, ws)
    h = torch.cat([k, torch.tensor([127.0], device="cuda:0")]).half()[None]
    q = torch.zeros(h.shape, dtype=torch.int8, device="cuda:0")
    assert quant_rows(h, q, s[:1]) == 0
    assert torch.equal(q, ref_quant(h)[0])


@pytest.mark.parametrize("C", [5, 64, 256, 700, 5000])
def test_quant_rows_extremes(C):
    """Zero rows, the smallest and largest numbers, and rows that hold an infinity or NaN at any place."""
    import torch
    fmax, tiny = torch.finfo(torch.float32).max, 2.0 ** -149
    x = _rand(_gen(C), 12, C)
    x[0] = 0
    x[1] = -0.0
    x[2] *= 1e-42
    x[3] = tiny
    x[4, C // 2] = fmax
    x[5] = x[5].sign() * fmax
    x[6, 0] = float("inf")
    x[7, C - 1] = float("-inf")
    x[8, C // 2] = float("nan")
    x[9, 0], x[9, C - 1] = float("nan"), float("inf")
    x[10] *= 1e30
    q = torch.full(x.shape, 99, dtype=torch.int8, device="cuda:0")
    s = torch.full((12,), -1.0, device="cuda:0")
    assert quant_rows(x, q, s) == 0
    wq, ws = ref_quant(x)
    assert torch.equal(q, wq)
    assert torch.equal(torch.isnan(s), torch.isnan(ws)) and torch.equal(s.nan_to_num(), ws.nan_to_num())
    assert torch.isnan(s).tolist() == [False] * 6 + [True] * 4 + [False] * 2


# ------------------------------------------------------------------ the product

def _operands(M, N, K, seed, ldx=None, ldw=None):
    import torch
    g = _gen(seed)
    up = lambda k: -(-k // 16) * 16  # noqa: E731
    x, _ = strided(M, K, ldx or up(K), torch.int8, 77)
    w, _ = strided(N, K, ldw or up(K), torch.int8, -77)
    x.copy_(torch.randint(-127, 128, (M, K), generator=g, device="cuda:0"))
    w.copy_(torch.randint(-127, 128, (N, K), generator=g, device="cuda:0"))
    xs = torch.rand(M, generator=g, device="cuda:0") * 0.02 + 1e-4
    ws = torch.rand(N, generator=g, device="cuda:0") * 0.002 + 1e-5
    return x, xs, w, ws, _rand(g, N, scale=0.3)


def _check_product(M, N, K, dtype, relu, bias=True, seed=None, ldo=None, **more):
    import torch
    dt = torch_dtype(dtype)
    x, xs, w, ws, b = _operands(M, N, K, seed if seed is not None else M * 31 + N * 7 + K, **more)
    b = b if bias else None
    out, buf = strided(M, N, ldo or N, dt, 123.0)
    assert i8_gemm(x, xs, w, ws, b, out, relu) == 0
    want, bound = ref_product(x, xs, w, ws, b, relu, dt)
    assert worst(out, want, bound) <= 1.0
    assert untouched(out, buf, 123.0)


# the smallest, single tokens, the borders of 16, 32, 64, 128, 256 rows, columns and depths, the blocks' sizes
PRODUCTS = [(1, 1, 1), (1, 16, 16), (1, 512, 512), (1, 1000, 4096), (2, 33, 31), (3, 160, 160), (4, 256, 100), (5, 7, 1024),
            (8, 128, 512), (9, 512, 256), (15, 257, 129), (16, 128, 128), (17, 129, 127), (31, 64, 2048), (32, 255, 96),
            (33, 512, 48), (50, 96, 65), (64, 256, 256), (65, 40, 513), (100, 1037, 1000), (127, 128, 128),
            (128, 128, 32), (128, 256, 256), (129, 257, 257), (200, 512, 512), (256, 256, 128), (257, 100, 1),
            (300, 16, 4096), (511, 160, 160), (1000, 300, 77), (1800, 512, 512), (2049, 513, 640), (7200, 160, 160),
            (1, 20000, 64), (20000, 1, 64), (2, 5000, 700), (4, 4100, 2000), (1, 4097, 2049),
            # few tokens against long rows: K split over two, four and eight CTAs
            (20, 1000, 2000), (12, 100, 4000), (70, 1000, 16000), (33, 300, 9001), (500, 130, 16384), (40, 4096, 1024),
            (61, 1001, 65000), (99, 4096, 16384), (250, 2047, 8190), (500, 639, 32760),
            # units of 256 tokens over two CTAs, the last ones ragged
            (4000, 2500, 3000), (3001, 2051, 3001), (2600, 4104, 4096),
            # several units a CTA: two and four accumulators, groups of 4 and 8 epilogue warps
            (20001, 300, 200), (30011, 100, 64), (40000, 160, 128), (9001, 513, 1024), (5003, 2000, 300)]


@pytest.mark.parametrize("size", PRODUCTS, ids=lambda s: "%dx%dx%d" % s)
def test_i8_gemm(size):
    M, N, K = size
    i = PRODUCTS.index(size)
    _check_product(M, N, K, DTYPES[i % 3], relu=i % 2 == 1)
    _check_product(M, N, K, DTYPES[(i + 1) % 3], relu=i % 2 == 0, bias=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 7, 40, 130, 700])
def test_i8_gemm_pitches(M, dtype):
    """Operand rows apart and results at odd pitches; what lies between the rows is not read and not written."""
    _check_product(M, 131, 200, dtype, True, ldo=131 + 6, ldx=224, ldw=416)
    _check_product(M, 96, 96, dtype, False, ldo=96 + 8, ldx=112, ldw=96)
    _check_product(M, 40, 33, dtype, False, ldo=41, ldx=48, ldw=64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N", [(1, 64), (20, 64), (150, 136), (700, 300), (20001, 72)])
def test_i8_gemm_result_alignments(M, N, dtype):
    """The result's rows start 16, 8, 4 or 2 bytes off a vector's border, at pitches of every such multiple."""
    import torch
    dt = torch_dtype(dtype)
    x, xs, w, ws, b = _operands(M, N, 64, 3)
    want, bound = ref_product(x, xs, w, ws, b, False, dt)
    for off, more in ((1, 0), (2, 0), (4, 8), (0, 2), (0, 4), (0, 1), (3, 5)):
        ldo = N + more
        buf = torch.full(((M - 1) * ldo + N + off + 1,), 9.0, dtype=dt, device="cuda:0")
        out = buf[off:].as_strided((M, N), (ldo, 1))
        assert i8_gemm(x, xs, w, ws, b, out) == 0
        assert worst(out, want, bound) <= 1.0, (off, more)
        assert untouched(out, buf, 9.0), (off, more)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,pad", [(2904, 183, 3), (2904, 183, 1), (300, 183, 5), (2904, 189, 3), (20000, 503, 1), (20000, 502, 2),
                                     (9000, 1001, 3), (9000, 2047, 1)])
def test_i8_gemm_rows_that_end_inside_a_piece(M, N, pad, dtype):
    """Rows at multiples of 4 or 8 bytes whose last elements fill no such piece, after many that do (in several runs: the
    pieces are stored side by side)."""
    import torch
    dt = torch_dtype(dtype)
    x, xs, w, ws, b = _operands(M, N, 40, N)
    want, bound = ref_product(x, xs, w, ws, b, False, dt)
    for _ in range(3):
        out, buf = strided(M, N, N + pad, dt, 9.0)
        assert i8_gemm(x, xs, w, ws, b, out) == 0
        assert worst(out, want, bound) <= 1.0
        assert untouched(out, buf, 9.0)


@pytest.mark.parametrize("M,N", [(1, 40), (24, 70), (200, 130)])
def test_i8_gemm_largest_sums(M, N):
    """-128 x -128 over the longest rows the sum allows: 2^31 - 2^14, and its mirror."""
    import torch
    K = 131071
    x, _ = strided(M, K, 131072, torch.int8, 5)
    w, _ = strided(N, K, 131072, torch.int8, 5)
    x.fill_(-128)
    w.fill_(-128)
    w[1::2] = 127
    one_m, one_n = torch.ones(M, device="cuda:0"), torch.ones(N, device="cuda:0")
    out = torch.empty(M, N, device="cuda:0")
    assert i8_gemm(x, one_m, w, one_n, None, out) == 0
    assert (out[:, 0::2].double() == 2.0 ** 14 * K).all()       # 24 bits hold it
    want = float(np.float32(-128 * 127 * K))
    assert (out[:, 1::2].double() == want).all()


def test_i8_gemm_special_scales():
    """A NaN scale (a row that held an infinity) makes that token's results NaN, relu or not, and no others; zero
    scales leave the bias; very small scales do not lose the product."""
    import torch
    for M in (4, 24, 140):
        x, xs, w, ws, b = _operands(M, 90, 300, M)
        xs[1], xs[2], ws[5] = float("nan"), 0.0, 0.0
        xs[3], ws[7] = 1e-32, 1e-9
        out = torch.empty(M, 90, device="cuda:0")
        for relu in (False, True):
            assert i8_gemm(x, xs, w, ws, b, out, relu) == 0
            assert torch.isnan(out[1]).all() and torch.isnan(out).sum().item() == 90
            want, bound = ref_product(x, xs, w, ws, b, relu, torch.float32)
            assert worst(out, want, bound) <= 1.0
        assert i8_gemm(x, xs, w, ws, None, out) == 0
        want, bound = ref_product(x, xs, w, ws, None, False, torch.float32)
        assert worst(out, want, bound) <= 1.0


def test_i8_gemm_offsets_past_32_bits():
    """Results and tokens beyond 4 GB of their buffers."""
    import torch
    M, ld = 3000, 1 << 21                                        # rows 2 MB apart: 6.3 GB of tokens
    x, _ = strided(M, 48, ld, torch.int8, 0)
    g = _gen(1)
    x.copy_(torch.randint(-127, 128, (M, 48), generator=g, device="cuda:0"))
    _, xs, w, ws, b = _operands(M, 24, 48, 2)
    out, buf = strided(M, 24, 1 << 20, torch.float16, 0.0)
    assert i8_gemm(x, xs, w, ws, b, out) == 0
    want, bound = ref_product(x, xs, w, ws, b, False, torch.float16)
    assert worst(out, want, bound) <= 1.0
    few, _ = strided(4, 48, 1 << 30, torch.int8, 0)              # and with few tokens
    few.copy_(x[:4])
    assert i8_gemm(few, xs[:4], w, ws, b, out[:4]) == 0
    assert worst(out[:4], want[:4], bound[:4]) <= 1.0


# ------------------------------------------------------------------ the norms of a block

# C, rows, dtype, post, gate rows ("all", n or None), pre
NORMS = [(1, 3, "f32", LAYER, None, LAYER), (7, 5, "f16", RMS, 1, LAYER), (8, 9, "bf16", LAYER, "all", RMS),
         (64, 33, "f16", LAYER, 4, LAYER), (65, 17, "f32", RMS, 4, RMS), (96, 50, "f16", 0, None, LAYER),
         (128, 21, "bf16", LAYER, 5, 0), (160, 77, "f16", LAYER, "all", LAYER), (200, 10, "f32", 0, 3, 0),
         (256, 131, "f16", LAYER, "all", LAYER), (256, 12, "f32", RMS, 1, RMS), (257, 6, "bf16", LAYER, None, LAYER),
         (512, 41, "f16", LAYER, 8, LAYER), (512, 5, "f32", LAYER, "all", RMS), (1000, 7, "f16", RMS, 2, LAYER),
         (1024, 9, "bf16", RMS, 1, RMS), (1037, 4, "f32", LAYER, 1, LAYER), (2048, 5, "f16", LAYER, "all", LAYER),
         (2050, 3, "bf16", 0, None, RMS), (4096, 9, "bf16", RMS, 4, RMS), (4096, 3, "f32", LAYER, 1, LAYER),
         (8192, 3, "f16", LAYER, None, LAYER), (8191, 2, "f32", RMS, "all", LAYER), (16384, 2, "bf16", LAYER, 1, RMS),
         (16000, 2, "f32", LAYER, 1, LAYER), (32768, 2, "f32", LAYER, "all", LAYER), (32761, 1, "f16", RMS, None, RMS)]


def _block(C, rows, dtype, post, gate, pre, seed=0, pad=0, affine=True):
    import torch
    dt, g = torch_dtype(dtype), _gen(seed + C + rows)
    t = {}
    for name in ("x", "f"):
        t[name], _ = strided(rows, C, C + pad, dt, float("nan"))
        t[name].copy_(_rand(g, rows, C) * 2 + 0.25)
    per = rows if gate == "all" else gate
    if gate is not None:
        n = -(-rows // per)
        t["gate"], _ = strided(n, C, C + pad, dt, float("nan"))
        t["gate"].copy_(_rand(g, n, C, scale=0.5))
        t["gate_rows"] = per
    for k, kind in (("1", post), ("2", pre)):
        if kind and affine:
            t["g" + k] = 1 + _rand(g, C, scale=0.2)
            t["b" + k] = _rand(g, C, scale=0.2) if kind == LAYER else None
    t.update(post=post, pre=pre, scale=0.7)
    return t


def _norm_outputs(t, pad=0, quant=True):
    import torch
    x = t.get("x") if t.get("x") is not None else t["f"]
    rows, C = x.shape
    o = {}
    for name in ("r", "y"):
        o[name], o[name + "_buf"] = strided(rows, C, C + pad, x.dtype, 55.0)
    if quant:
        o["q"], o["q_buf"] = strided(rows, C, C + 2 * pad, torch.int8, 99)
        o["qs"] = torch.full((rows,), -1.0, device="cuda:0")
    return o


def _check_norm(t, o):
    import torch
    out = {k: o[k] for k in ("r", "y", "q", "qs") if k in o}
    assert block_norm(**t, **out) == 0
    (v, ev), (h, eh) = ref_block(**t)
    for name, val, err in (("r", v, ev), ("y", h, eh)):
        if name in o:
            assert worst(o[name], val, stored(val, err, o[name].dtype) + 1e-300) <= 1.0, name
            assert untouched(o[name], o[name + "_buf"], 55.0)
    if "q" in o:
        top, et = h.abs().amax(1), eh.amax(1)
        assert ((o["qs"].double() - top / 127).abs() <= et / 127 + top / 127 * U * 1.01 + 2.0 ** -149).all()
        some = top > 0
        steps = 127 * h[some] / top[some, None]
        far = 0.5 + 127 * (eh[some] + et[some, None]) / top[some, None] * 1.01
        assert ((o["q"][some].double() - steps).abs() <= far).all()
        assert untouched(o["q"], o["q_buf"], 99)


@pytest.mark.parametrize("case", NORMS, ids=lambda c: "C%d_%d_%s_%s_%s_%s" % c)
def test_block_norm(case):
    C, rows, dtype, post, gate, pre = case
    t = _block(C, rows, dtype, post, gate, pre)
    _check_norm(t, _norm_outputs(t))


@pytest.mark.parametrize("case", NORMS[1::3], ids=lambda c: "C%d_%d_%s_%s_%s_%s" % c)
@pytest.mark.parametrize("pad", [3, 16])
def test_block_norm_pitches(case, pad):
    C, rows, dtype, post, gate, pre = case
    t = _block(C, rows, dtype, post, gate, pre, seed=5, pad=pad)
    _check_norm(t, _norm_outputs(t, pad))


# rows of whole pairs of elements that are no whole vectors: by their length, by their pitch, at every size of a group
PAIRS = [(2, 9, 0), (10, 70, 0), (64, 33, 2), (130, 40, 4), (166, 21, 2), (250, 131, 0), (322, 9, 6), (510, 17, 0), (766, 5, 2),
         (1026, 6, 0), (1534, 4, 10), (2046, 5, 0), (4092, 3, 0), (4622, 3, 2), (8190, 2, 0), (12286, 2, 0), (32766, 2, 2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C,rows,pad", PAIRS)
def test_rows_of_whole_pairs(C, rows, pad, dtype):
    import torch
    t = _block(C, rows, dtype, LAYER, 2, LAYER, seed=9, pad=pad)
    _check_norm(t, _norm_outputs(t, pad))
    q, qb = strided(rows, C, C + 2 * pad, torch.int8, 99)
    s = torch.full((rows,), -1.0, device="cuda:0")
    assert quant_rows(t["x"], q, s) == 0
    wq, ws = ref_quant(t["x"])
    assert torch.equal(q, wq) and torch.equal(s, ws) and untouched(q, qb, 99)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_at_every_start(dtype):
    """Operands that start at each place of a 16-byte piece in turn, gains and shifts at each float of 32 bytes."""
    import torch
    C = 130
    for start in range(1, 9):
        t = _block(C, 6, dtype, LAYER, 1, LAYER, seed=start)
        for name in ("x", "f", "gate", "g1", "b1", "g2", "b2"):
            for only in (name, None) if start < 3 else (None,):
                u = dict(t)
                for k in ("x", "f", "gate", "g1", "b1", "g2", "b2"):
                    if only in (None, k):
                        b = torch.empty(t[k].numel() + start, device="cuda:0", dtype=t[k].dtype)[start:]
                        u[k] = b.view(t[k].shape).copy_(t[k])
                _check_norm(u, _norm_outputs(u))


@pytest.mark.parametrize("C", [64, 100, 512, 3000])
def test_block_norm_parts(C):
    """Each operand and each output left out in turn; norms without gain or shift."""
    for miss_in in ((), ("x",), ("f", "post", "gate", "gate_rows", "g1", "b1"), ("gate", "gate_rows")):
        for outs in (("r",), ("y",), ("q", "qs"), ("r", "q", "qs"), ("y", "q", "qs")):
            t = _block(C, 11, "f16", LAYER, 3, RMS, affine="gate" not in miss_in)
            t = {k: v for k, v in t.items() if k not in miss_in}
            o = _norm_outputs(t)
            _check_norm(t, {k: v for k, v in o.items() if k.split("_")[0] in outs})


@pytest.mark.parametrize("dtype", DTYPES)
def test_block_norm_in_place(dtype):
    """r on x and y on f: the same bytes as apart."""
    import torch
    for C in (64, 250, 2048):
        t = _block(C, 37, dtype, LAYER, 1, LAYER)
        o = _norm_outputs(t, quant=False)
        assert block_norm(**t, r=o["r"], y=o["y"]) == 0
        x, f = t["x"].clone(), t["f"].clone()
        t.update(x=x, f=f)
        assert block_norm(**t, r=x, y=f) == 0
        assert torch.equal(x, o["r"]) and torch.equal(f, o["y"])


def test_block_norm_rows_are_those_of_quant_rows():
    """The int8 rows are the rounding of the unrounded norm: of y itself where y is fp32."""
    import torch
    for C in (48, 77, 512, 4000):
        t = _block(C, 19, "f32", RMS, 4, LAYER)
        o = _norm_outputs(t)
        assert block_norm(**t, y=o["y"], q=o["q"], qs=o["qs"]) == 0
        q, s = torch.empty_like(o["q"]), torch.empty_like(o["qs"])
        assert quant_rows(o["y"], q, s) == 0
        assert torch.equal(q, o["q"]) and torch.equal(s, o["qs"])


def test_block_norm_extremes():
    """Constant rows, a large mean, zero rows, infinities and NaN in one row only, the type's largest values."""
    import torch
    for C in (40, 250, 4096):
        x = _rand(_gen(C), 9, C)
        x[0] = 0.0
        x[1] = 3.5
        x[2] += 1000.0
        x[3, C // 2] = float("inf")
        x[4, 0] = float("nan")
        x[5] *= 1e15
        x[6] *= 1e-15
        t = {"x": x, "pre": LAYER, "g2": 1 + _rand(_gen(1), C, scale=0.1), "b2": _rand(_gen(2), C, scale=0.1)}
        o = _norm_outputs(t)
        assert block_norm(**t, y=o["y"], q=o["q"], qs=o["qs"]) == 0
        assert torch.isnan(o["y"][3]).all() and torch.isnan(o["y"][4]).all()
        assert torch.isnan(o["qs"]).tolist() == [False] * 3 + [True] * 2 + [False] * 4
        assert (o["q"][3:5] == 0).all()
        keep = [0, 1, 2, 5, 6, 7, 8]
        _, (h, eh) = ref_block(**t)
        assert worst(o["y"][keep], h[keep], eh[keep]) <= 1.0
        top = torch.full((3, C), torch.finfo(torch.float16).max, dtype=torch.float16, device="cuda:0")
        top[1, ::2] *= -1
        t = {"x": top, "pre": RMS}
        o = _norm_outputs(t, quant=False)
        _check_norm(t, o)


# ------------------------------------------------------------------ together, and how they are called

@pytest.mark.parametrize("gate", ["all", 1, 50, None])
@pytest.mark.parametrize("C", [96, 256, 1000, 4096])
def test_the_norm_does_not_depend_on_other_rows(C, gate):
    """A token's bytes are the same alone and in any batch, whatever the gate's rows are shared by."""
    import torch
    t = _block(C, 300, "f16", LAYER, gate, LAYER)
    o = _norm_outputs(t)
    assert block_norm(**t, r=o["r"], y=o["y"], q=o["q"], qs=o["qs"]) == 0
    for row in (17, 299):
        one = {k: (v[row:row + 1] if k in ("x", "f") else v) for k, v in t.items()}
        if gate is not None:
            g = row // t["gate_rows"]
            one.update(gate=t["gate"][g:g + 1], gate_rows=1)
        p = _norm_outputs(one)
        assert block_norm(**one, r=p["r"], y=p["y"], q=p["q"], qs=p["qs"]) == 0
        for k in ("r", "y", "q", "qs"):
            assert torch.equal(p[k], o[k][row:row + 1]), (k, row)


def test_product_same_bytes_at_any_batch():
    """A token's results are the same bytes alone and in a batch of any size (every form of the kernel)."""
    import torch
    x, xs, w, ws, b = _operands(3000, 200, 330, 4)
    full = torch.empty(3000, 200, device="cuda:0")
    assert i8_gemm(x, xs, w, ws, b, full) == 0
    for m in (1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 256, 300, 600, 1500):
        out = torch.empty(m, 200, device="cuda:0")
        assert i8_gemm(x[:m], xs[:m], w, ws, b, out) == 0
        assert torch.equal(out, full[:m]), m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("relu", [False, True])
def test_product_same_bytes_of_zeros_and_nan_at_any_batch(dtype, relu):
    """Results that round to a negative zero, and NaN, have the same bytes in every form too; after relu a zero has no
    sign."""
    import torch
    n = 200
    x, xs, w, ws, _ = _operands(40000, n, 96, 8)
    xs[0::3] = 1e-30
    ws[0::2] = 1e-30                        # (their products underflow, half of them from below)
    xs[1] = float("nan")
    whole = torch.int32 if dtype == "f32" else torch.int16
    full = torch.empty(40000, n, device="cuda:0", dtype=torch_dtype(dtype))
    assert i8_gemm(x, xs, w, ws, None, full, relu) == 0
    negative = (full == 0) & torch.signbit(full)
    assert negative.any().item() != relu
    assert torch.isnan(full[1]).all()
    for m in (2, 4, 8, 40, 300, 2000):
        out = torch.empty(m, n, device="cuda:0", dtype=full.dtype)
        assert i8_gemm(x[:m], xs[:m], w, ws, None, out, relu) == 0
        differ = (out.view(whole) != full[:m].view(whole)).sum().item()
        assert differ == 0, (m, differ)


@pytest.mark.parametrize("net,name", [("gc", "block1"), ("dr", "block2")])
def test_shifted_mlp_block_in_8_bits(net, name):
    """One shifted-MLP block on int8 products, as a deployment chains the entries: norm with int8 rows -> fc1 ->
    depthwise + GELU + W shift -> int8 rows -> fc2 -> norm of the sum with the residual.  Each stage is checked
    against its 64-bit form on the stage's own inputs."""
    import ctypes

    import torch
    from gpu_util import Shift
    from oracle import gcdr_oracle as O
    from sdcb.gcdrnet_b200 import lib
    blk = getattr(O.GcdrNet.load(getattr(G, "GC_PATH" if net == "gc" else "DR_PATH")), name)
    H, W = 18, 25
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).to("cuda:0")  # noqa: E731
    wd, bd = blk.dw
    C = wd.shape[0]
    ln_g, ln_b = (dev(v) for v in blk.norm2)
    (w1, c1), (w2, c2) = _fc(blk, "fc1", C), _fc(blk, "fc2", C)
    w1, w2, c1, c2 = dev(w1), dev(w2), dev(c1), dev(c2)
    x = _rand(_gen(5), H * W, C).half()
    q1, s1 = torch.empty(H * W, C, dtype=torch.int8, device="cuda:0"), torch.empty(H * W, device="cuda:0")

    def weights(w):
        q, s = torch.empty(w.shape, dtype=torch.int8, device="cuda:0"), torch.empty(w.shape[0], device="cuda:0")
        assert quant_rows(w, q, s) == 0
        return q, s

    def depthwise(h):
        axis, ends, offs = blk.shift_w
        sh, out = Shift.of(ends, offs), torch.empty(H * W, C, dtype=torch.float16, device="cuda:0")
        wt, b = dev(np.ascontiguousarray(wd.reshape(C, 9).T)), dev(bd)
        assert lib().gcdr_k_dw_gelu_shift(h.data_ptr(), H, W, C, wt.data_ptr(), b.data_ptr(), ctypes.byref(sh),
                                          out.data_ptr(), None) == 0
        return out

    norm = {"x": x, "pre": LAYER, "g2": ln_g, "b2": ln_b}
    y = torch.empty_like(x)
    assert block_norm(**norm, y=y, q=q1, qs=s1) == 0
    # the rows stand for the tokens to half a step (and the fp16 rounding of y)
    off = (q1.double() * s1.double()[:, None] - y.double()).abs()
    assert (off <= s1.double()[:, None] * (0.5 + 1e-4) + y.double().abs() * 2.0 ** -11 + 2.0 ** -25).all()
    wq1, ws1 = weights(w1)
    h1 = torch.empty(H * W, C, dtype=torch.float16, device="cuda:0")
    assert i8_gemm(q1, s1, wq1, ws1, c1, h1) == 0
    want, bound = ref_product(q1, s1, wq1, ws1, c1, False, torch.float16)
    assert worst(h1, want, bound) <= 1.0
    h2 = depthwise(h1)
    q2, s2 = torch.empty_like(q1), torch.empty_like(s1)
    assert quant_rows(h2, q2, s2) == 0
    assert torch.equal(q2, ref_quant(h2)[0])
    wq2, ws2 = weights(w2)
    h3 = torch.empty_like(h1)
    assert i8_gemm(q2, s2, wq2, ws2, c2, h3) == 0
    want, bound = ref_product(q2, s2, wq2, ws2, c2, False, torch.float16)
    assert worst(h3, want, bound) <= 1.0
    last = {"x": x, "f": h3, "pre": LAYER, "g2": ln_g, "b2": ln_b}
    _check_norm(last, _norm_outputs(last))


def _fc(blk, name, C):
    w, b = getattr(blk, name)
    return (w if w.shape[0] == C else w.T), b


def test_calls_are_captured_and_replayed():
    """A chain captured into a graph (nothing is allocated, on the first call either) and replayed on new inputs, beside
    a second graph of the same operators on another stream."""
    import torch
    states = []
    for k in range(2):
        g = _gen(40 + k)
        s = {"x": _rand(g, 70, 256).half(), "w": torch.randint(-127, 128, (192, 256), generator=g, device="cuda:0").to(torch.int8),
             "ws": torch.rand(192, generator=g, device="cuda:0") * 0.01, "q": torch.empty(70, 256, dtype=torch.int8, device="cuda:0"),
             "qs": torch.empty(70, device="cuda:0"), "out": torch.empty(70, 192, dtype=torch.float16, device="cuda:0"),
             "q2": torch.empty(70, 192, dtype=torch.int8, device="cuda:0"), "qs2": torch.empty(70, device="cuda:0")}
        states.append(s)

    def chain(s, stream):
        assert block_norm(x=s["x"], pre=RMS, q=s["q"], qs=s["qs"], stream=stream) == 0
        assert i8_gemm(s["q"], s["qs"], s["w"], s["ws"], None, s["out"], stream=stream) == 0
        assert quant_rows(s["out"], s["q2"], s["qs2"], stream=stream) == 0

    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for s, st in zip(states, streams):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            chain(s, st.cuda_stream)
        graphs.append(gr)
    for rep in range(3):
        for s in states:
            s["x"].copy_(_rand(_gen(90 + rep), 70, 256))
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for s in states:
            got = {k: s[k].clone() for k in ("q", "qs", "out", "q2", "qs2")}
            chain(s, None)
            torch.cuda.synchronize()
            for k, v in got.items():
                assert torch.equal(v, s[k]), k


def test_calls_back_to_back_on_reused_buffers():
    """Calls that follow one another on one stream, each on buffers that the one before read or wrote (in place and
    apart), give what the same calls give with a wait between them."""
    import torch
    g = _gen(77)
    C = 256
    w = torch.randint(-127, 128, (C, C), generator=g, device="cuda:0").to(torch.int8)
    ws, bias = torch.rand(C, generator=g, device="cuda:0") * 2e-3, _rand(g, C, scale=0.1)
    gain, shift = 1 + _rand(g, C, scale=0.1), _rand(g, C, scale=0.1)
    for rows in (1, 700, 9001):
        start = _rand(g, rows, C).half()

        def chain(wait):
            x, q, s = start.clone(), torch.zeros(rows, C, dtype=torch.int8, device="cuda:0"), torch.zeros(rows, device="cuda:0")
            h = torch.zeros(rows, C, dtype=torch.float16, device="cuda:0")
            torch.cuda.synchronize()
            for _ in range(12):
                assert block_norm(x=x, pre=LAYER, g2=gain, b2=shift, q=q, qs=s) == 0
                if wait:
                    torch.cuda.synchronize()
                assert i8_gemm(q, s, w, ws, bias, h, relu=True) == 0
                if wait:
                    torch.cuda.synchronize()
                assert block_norm(x=x, f=h, post=RMS, g1=gain, scale=0.5, r=x, pre=RMS, g2=gain, y=h) == 0
                if wait:
                    torch.cuda.synchronize()
                assert quant_rows(h, q, s) == 0
                assert i8_gemm(q, s, w, ws, None, h) == 0
                assert block_norm(x=x, f=h, scale=0.1, r=x) == 0
                if wait:
                    torch.cuda.synchronize()
            torch.cuda.synchronize()
            return x, h, q, s

        for got, want in zip(chain(False), chain(True)):
            assert torch.equal(got, want)


def test_calls_on_two_streams_at_once():
    """Products of every form and norms on two streams side by side, many times over: the bytes of a call alone."""
    import torch
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    jobs = []
    for k, sizes in enumerate(([(4000, 2500, 3000), (16, 1000, 4000), (9001, 513, 1024)],
                               [(2600, 4104, 4096), (3, 5000, 700), (1800, 512, 512), (12, 100, 4000)])):
        for M, N, K in sizes:
            x, xs, w, ws, b = _operands(M, N, K, M + N + k)
            want = torch.empty(M, N, dtype=torch.float16, device="cuda:0")
            assert i8_gemm(x, xs, w, ws, b, want) == 0
            out = torch.zeros_like(want)
            y, q, s = torch.zeros_like(want), torch.zeros(M, N, dtype=torch.int8, device="cuda:0"), torch.zeros(M, device="cuda:0")
            ref = [torch.zeros_like(t) for t in (y, q, s)]
            assert block_norm(x=want, pre=LAYER, y=ref[0], q=ref[1], qs=ref[2]) == 0
            jobs.append((k, (x, xs, w, ws, b), want, out, (y, q, s), ref))
    torch.cuda.synchronize()
    for _ in range(10):
        for k, ops, _, out, (y, q, s), _ in jobs:
            st = streams[k].cuda_stream
            assert i8_gemm(*ops, out, stream=st) == 0
            assert block_norm(x=out, pre=LAYER, y=y, q=q, qs=s, stream=st) == 0
    torch.cuda.synchronize()
    for _, _, want, out, got, ref in jobs:
        assert torch.equal(out, want)
        for a, b in zip(got, ref):
            assert torch.equal(a, b)


def test_refusals_with_device_operands():
    """Host memory, overlapping operands: refused before anything is launched."""
    import torch
    x = torch.zeros(8, 64, dtype=torch.float16, device="cuda:0")
    q, s = torch.zeros(8, 64, dtype=torch.int8, device="cuda:0"), torch.zeros(8, device="cuda:0")
    assert quant_rows(x.cpu(), q, s) == 1
    assert quant_rows(x, q.cpu(), s) == 1
    assert quant_rows(x, x.view(torch.int8)[:, :64], s) == 1
    assert quant_rows(x, q, q.view(-1)[:32].view(torch.float32)) == 1
    assert block_norm(x=x, pre=RMS, y=x.view(-1)[8:].as_strided((8, 56), (64, 1)), r=None) == 1
    out = torch.zeros(8, 8, device="cuda:0")
    w, ws = torch.zeros(8, 64, dtype=torch.int8, device="cuda:0"), torch.zeros(8, device="cuda:0")
    assert i8_gemm(q, s, w, ws, ws.cpu(), out) == 1
    assert i8_gemm(q, s, w, ws, out[0], out) == 1
    assert i8_gemm(q, s, w, ws, None, out) == 0
    # two column slices of one buffer are apart
    both = torch.zeros(8, 128, dtype=torch.float16, device="cuda:0")
    assert block_norm(x=x, pre=RMS, r=both[:, :64], y=both[:, 64:]) == 0
    assert block_norm(x=x, pre=RMS, r=both[:, :64], y=both[:, 56:120]) == 1
    assert block_norm(x=x, pre=RMS, r=both[:, :64], y=both[:, :64]) == 1
    torch.cuda.synchronize()


# (M, N, K): a split narrow product (clusters), a narrow one, wide ones of one and of several tiles a CTA
I8_CASES = [(20, 128, 2048), (40, 20000, 96), (200, 130, 300), (6000, 600, 256)]


@pytest.mark.parametrize("case", I8_CASES, ids=lambda c: "%dx%dx%d" % c)
def test_i8_gemm_wait_runs_out_and_reports_timeout(case):
    """The test hook issues no copies and no MMAs: every role's first wait runs out, nothing is written, the
    status says so once, and the next call is right."""
    import time

    import torch
    from sdcb.gcdrnet_b200 import lib
    L = lib()
    M, N, K = case
    g = torch.Generator(device="cuda:0").manual_seed(M)
    x = torch.zeros(M, -(-K // 16) * 16, dtype=torch.int8, device="cuda:0")[:, :K]
    w = torch.zeros(N, x.stride(0), dtype=torch.int8, device="cuda:0")[:, :K]
    x.copy_(torch.randint(-127, 128, (M, K), generator=g, device="cuda:0"))
    w.copy_(torch.randint(-127, 128, (N, K), generator=g, device="cuda:0"))
    xs, ws = torch.ones(M, device="cuda:0"), torch.ones(N, device="cuda:0")
    out = torch.full((M, N), float("nan"), dtype=torch.float32, device="cuda:0")
    torch.cuda.synchronize()
    assert L.gcdr_k_status(None) == 0
    t0 = time.perf_counter()
    assert i8_gemm(x, xs, w, ws, None, out, wait_cycles=400_000, timeout_probe=1) == 0
    assert L.gcdr_k_status(None) == 5
    assert time.perf_counter() - t0 < 5.0
    assert torch.isnan(out).all().item(), "the probe wrote outputs"
    assert L.gcdr_k_status(None) == 0
    assert i8_gemm(x, xs, w, ws, None, out) == 0
    assert L.gcdr_k_status(None) == 0
    want, bound = ref_product(x, xs, w, ws, None, False, torch.float32)
    assert worst(out, want, bound) <= 1.0


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_quant_rows_every_quotient_of_16_bits(dtype):
    """Every value of the type from the largest down to 2^-9 of it, against every mantissa of the largest: all borders
    that 16-bit rows can meet, and their neighbours."""
    import torch
    dt = torch_dtype(dtype)
    bits = 11 if dtype == "f16" else 8
    mant = torch.arange(1 << (bits - 1), 1 << bits, device="cuda:0").double()      # every mantissa
    for top_exp in (0, 4):
        vals = torch.cat([mant * 2.0 ** (top_exp - e) for e in range(10)])
        for part in mant.split(128):
            top = part * 2.0 ** top_exp
            x = torch.where(vals[None, :] <= top[:, None], vals[None, :], torch.zeros_like(vals)[None, :])
            sign = torch.where(torch.arange(vals.numel(), device="cuda:0") % 2 == 0, 1.0, -1.0).double()
            x = torch.cat([x * sign, top[:, None]], 1).to(dt)
            x = (x.double() * 2.0 ** -6).to(dt)
            q = torch.empty(x.shape, dtype=torch.int8, device="cuda:0")
            s = torch.empty(x.shape[0], device="cuda:0")
            assert quant_rows(x, q, s) == 0
            wq, ws = ref_quant(x)
            assert torch.equal(q, wq) and torch.equal(s, ws)
