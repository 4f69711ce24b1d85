"""gcdr_k_status: one error word for the layer entries of a device, read by one copy and cleared."""
import ctypes

import pytest

from gpu_util import ConvDesc

pytestmark = pytest.mark.gpu

OK, TIMEOUT = 0, 5


def _conv(L, **more):
    """A 1x1 token product by gcdr_k_conv on zeros (128 tokens of 128 channels)."""
    import torch
    t = [torch.zeros(128, 128, dtype=torch.float16, device="cuda:0") for _ in range(3)]
    b = torch.zeros(128, device="cuda:0")
    d = ConvDesc(kind=2, H=8, W=16, C=128, N=128, inp=t[0].data_ptr(), weight=t[1].data_ptr(), bias=b.data_ptr(),
                 out=t[2].data_ptr(), nsplit=1, ksplit=1, **more)
    assert L.gcdr_k_conv(ctypes.byref(d), 0, None) == OK
    return t, b


def _product(**more):
    import torch
    from int8_util import i8_gemm
    x, w = (torch.zeros(64, 64, dtype=torch.int8, device="cuda:0") for _ in range(2))
    s = torch.ones(64, device="cuda:0")
    out = torch.empty(64, 64, dtype=torch.float16, device="cuda:0")
    assert i8_gemm(x, s, w, s, None, out, **more) == OK
    return x, w, s, out


def test_either_kernel_sets_the_word_and_one_call_clears_it():
    import torch
    from sdcb.gcdrnet_b200 import lib
    L = lib()
    L.gcdr_k_status(None)
    probe = {"wait_cycles": 400_000, "timeout_probe": 1}
    for calls in ((_conv,), (_product,), (_conv, _product), (_product, _conv)):
        keep = [c(L, **probe) if c is _conv else c(**probe) for c in calls]
        assert L.gcdr_k_status(None) == TIMEOUT
        assert L.gcdr_k_status(None) == OK
        keep += [_conv(L), _product()]
        assert L.gcdr_k_status(None) == OK
        torch.cuda.synchronize()
        del keep


def test_status_is_one_copy_and_one_clear():
    import torch
    from torch.profiler import ProfilerActivity, profile
    from sdcb.gcdrnet_b200 import lib
    L = lib()
    x = torch.zeros(64, device="cuda:0")
    assert L.gcdr_k_status(None) == OK
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA, ProfilerActivity.CPU]) as p:
        x.add_(1)
        torch.cuda.synchronize()
        assert L.gcdr_k_status(None) == OK
        torch.cuda.synchronize()
    names = [e.name for e in p.events()]
    if not any("elementwise" in n for n in names):
        pytest.skip("the profiler shows no device work here")
    assert sum(n.startswith("Memcpy DtoH") for n in names) == 1, names
    assert sum(n.startswith("Memset") for n in names) == 1, names


def test_first_layer_call_allocates_nothing():
    """In a process of its own: the error word is part of the library, so a first gcdr_k_conv may be captured."""
    import os
    import subprocess
    import sys
    code = """
import ctypes, sys
import torch
from gpu_util import ConvDesc
from sdcb.gcdrnet_b200 import lib
L = lib()
g = torch.Generator(device="cuda:0").manual_seed(1)
a, w = (torch.randn(128, 128, generator=g, device="cuda:0").half() for _ in range(2))
out = torch.zeros(128, 128, dtype=torch.float16, device="cuda:0")
import numpy as np
b = torch.zeros(128, device="cuda:0")
host = np.zeros(128, np.float32)
d = ConvDesc(kind=2, H=8, W=16, C=128, N=128, inp=a.data_ptr(), weight=w.data_ptr(), bias=b.data_ptr(),
             out=out.data_ptr(), nsplit=1, ksplit=1, bias_host=host.ctypes.data)
torch.cuda.synchronize()
gr, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
with torch.cuda.graph(gr, stream=st):
    assert L.gcdr_k_conv(ctypes.byref(d), 0, st.cuda_stream) == 0
gr.replay()
torch.cuda.synchronize()
assert L.gcdr_k_status(None) == 0
want = a.double() @ w.double().t()
# fp32 sums of 128 exact products, then one rounding to fp16
room = (a.double().abs() @ w.double().abs().t()) * 128 * 2.0 ** -24 + want.abs() * 2.0 ** -11 + 2.0 ** -24
assert ((out.double() - want).abs() <= room * 1.01).all()
print("captured")
"""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(here), os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.strip().endswith("captured")
