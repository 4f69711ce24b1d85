"""How the 8-bit token operators are called: parameters that the call before computes, a first call inside a capture,
sizes beyond 2^31 rows and 2^30 tokens or channels."""
import os
import subprocess
import sys

import pytest

from int8_util import LAYER, RMS, block_norm, i8_gemm, quant_rows, ref_product, ref_quant, worst
from test_gpu_int8 import _gen, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(2, 500, 384), (16, 1000, 4096), (300, 512, 512), (9000, 384, 256), (2600, 4104, 2048)])
def test_parameters_computed_by_the_call_before(M, N, K):
    """Weights, scales, biases, gains and gates written by one call and read by the next, in the same buffers time and
    again: what the calls give with a wait between them."""
    import torch
    g = _gen(M + N)
    ws_in = [_rand(g, N, K, scale=0.1 * (1 + i)) for i in range(4)]
    xs_in = [_rand(g, M, K) for _ in range(4)]
    rows = [_rand(g, 2, N) for _ in range(4)]

    def chain(wait):
        def call(rc):
            assert rc == 0
            if wait:
                torch.cuda.synchronize()
        w, ws = torch.zeros(N, K, dtype=torch.int8, device="cuda:0"), torch.zeros(N, device="cuda:0")
        x, xs = torch.zeros(M, K, dtype=torch.int8, device="cuda:0"), torch.zeros(M, device="cuda:0")
        p = torch.zeros(2, N, device="cuda:0")
        out, y = torch.zeros(M, N, device="cuda:0"), torch.zeros(M, N, device="cuda:0")
        keep = []
        torch.cuda.synchronize()
        for i in range(12):
            call(quant_rows(xs_in[i % 4], x, xs))
            call(block_norm(x=rows[i % 4], pre=LAYER, y=p))              # a bias and a gain
            call(quant_rows(ws_in[(i + i // 4) % 4], w, ws))             # the weights last
            call(i8_gemm(x, xs, w, ws, p[0], out, relu=i % 2 == 0))
            call(block_norm(x=rows[(i + 1) % 4], pre=RMS, y=p))
            call(block_norm(f=out, post=LAYER, g1=p[0], b1=p[1], gate=p[1:], gate_rows=M, r=y))
            keep.append(y.clone() if i % 3 else out.clone())
        torch.cuda.synchronize()
        return keep

    for got, want in zip(chain(False), chain(True)):
        assert torch.equal(got, want)


def test_first_calls_inside_a_capture():
    """In a process of its own, each operator's first call is captured (rows that spill to local memory among them) and
    replayed: nothing has to be loaded or allocated by an earlier call."""
    code = """
import sys
import torch
from int8_util import LAYER, block_norm, i8_gemm, quant_rows
from sdcb.gcdrnet_b200 import lib
lib()
for C, rows, dt in ((32768, 300, torch.float32), (256, 5000, torch.float16), (4096, 4, torch.bfloat16), (2048, 3000, torch.float16)):
    g = torch.Generator(device="cuda:0").manual_seed(C)
    x, f, gate = (torch.randn(rows, C, generator=g, device="cuda:0").to(dt) for _ in range(3))
    y, r = torch.zeros_like(x), torch.zeros_like(x)
    q, q2 = (torch.zeros(rows, C, dtype=torch.int8, device="cuda:0") for _ in range(2))
    s, s2 = (torch.zeros(rows, device="cuda:0") for _ in range(2))
    w = torch.randint(-127, 128, (257, C), generator=g, device="cuda:0").to(torch.int8)
    ws, out = torch.rand(257, generator=g, device="cuda:0"), torch.zeros(rows, 257, device="cuda:0")

    def run(st):
        assert block_norm(x=x, f=f, post=LAYER, gate=gate, gate_rows=1, pre=LAYER, r=r, y=y, q=q, qs=s, stream=st) == 0
        assert quant_rows(y, q2, s2, st) == 0
        assert i8_gemm(q, s, w, ws, None, out, stream=st) == 0
    torch.cuda.synchronize()
    gr, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(gr, stream=st):
        run(st.cuda_stream)
    gr.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in (r, y, q, s, q2, s2, out)]
    for t in (r, y, q, s, q2, s2, out):
        t.zero_()
    run(None)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, (r, y, q, s, q2, s2, out))), C
    assert out.abs().sum().item() > 0
print("captured")
"""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(here), os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.strip().endswith("captured")


def _some_rows(rows, n=4000):
    """Row numbers over the whole range: the first and last ones and some between."""
    import torch
    g = torch.Generator().manual_seed(rows & 0xFFFF)
    mid = torch.randint(0, rows, (n,), generator=g)
    around = torch.arange(-64, 64) + (1 << 31)
    picks = torch.cat([torch.arange(64), mid, around[around < rows], torch.arange(rows - 200, rows)])
    return picks.unique().to("cuda:0")


def test_more_rows_than_31_bits():
    """2^31 rows and some: the row number itself passes 32 bits (a gate's row is then found by a division)."""
    import torch
    rows = (1 << 31) + 1003
    g = _gen(5)
    x = torch.empty(rows, 1, dtype=torch.float16, device="cuda:0").normal_(generator=g)
    gate = torch.empty(-(-rows // 7), 1, dtype=torch.float16, device="cuda:0").normal_(generator=g)
    y = torch.full((rows, 1), 9.0, dtype=torch.float16, device="cuda:0")
    assert block_norm(f=x, gate=gate, gate_rows=7, scale=0.5, r=y) == 0
    at = _some_rows(rows)
    want = 0.5 * x[at].double() * gate[at // 7].double()
    assert ((y[at].double() - want).abs() <= want.abs() * (2.0 ** -11 + 2.0 ** -22) + 2.0 ** -25).all()
    del gate, y
    q, s = torch.full((rows, 1), 99, dtype=torch.int8, device="cuda:0"), torch.full((rows,), -1.0, device="cuda:0")
    assert quant_rows(x, q, s) == 0
    wq, ws = ref_quant(x[at])
    assert torch.equal(q[at], wq) and torch.equal(s[at], ws)


@pytest.mark.parametrize("M,N", [((1 << 30) + 77, 3), (2, (1 << 30) + 77), (5, (1 << 29) + 77)])
def test_a_product_of_2_to_the_30(M, N):
    """2^30 tokens, and as many channels."""
    import torch
    g = _gen(9)
    big, small = max(M, N), min(M, N)
    rows = torch.empty(big, 16, dtype=torch.int8, device="cuda:0").random_(-127, 128, generator=g)
    few = torch.randint(-127, 128, (small, 16), generator=g, device="cuda:0").to(torch.int8)
    scales = torch.empty(big, device="cuda:0").uniform_(0.001, 0.02, generator=g)
    one = torch.rand(small, generator=g, device="cuda:0") * 0.01
    x, xs, w, ws = (rows, scales, few, one) if M == big else (few, one, rows, scales)
    out = torch.full((M, N), 9.0, dtype=torch.float16, device="cuda:0")
    assert i8_gemm(x, xs, w, ws, None, out) == 0
    at = _some_rows(big)
    xa, xsa, wa, wsa = (x[at], xs[at], w, ws) if M == big else (x, xs, w[at], ws[at])
    want, bound = ref_product(xa, xsa, wa, wsa, None, False, torch.float16)
    assert worst(out[at] if M == big else out[:, at], want, bound) <= 1.0
