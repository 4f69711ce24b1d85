"""Plain 64-bit forms of the 8-bit token operators, each with how far fp32 arithmetic may be from it, and
the calls of their entries on torch tensors (strided views included)."""
import ctypes

import numpy as np

U = 2.0 ** -24                      # half a step of fp32, relative
DTYPES = ("f16", "bf16", "f32")
LAYER, RMS = 1, 2


def torch_dtype(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def code(dtype):
    import torch
    return {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}[dtype]


def half_step(t):
    """Half a step of the type: relative, and the absolute one of its subnormal numbers."""
    import torch
    f = torch.finfo(t)
    return f.eps / 2, float(f.smallest_normal) * f.eps / 2


def strided(rows, cols, ld, dtype, fill, device="cuda:0"):
    """(view of rows x cols at pitch ld, its whole buffer filled with `fill`); the buffer ends with the last row."""
    import torch
    buf = torch.full(((rows - 1) * ld + cols,), fill, dtype=dtype, device=device)
    return buf.as_strided((rows, cols), (ld, 1)), buf


def untouched(view, buf, fill):
    """Nothing between the rows of `view` was written."""
    import torch
    mask = torch.ones_like(buf, dtype=torch.bool)
    mask.as_strided(view.shape, view.stride(), view.storage_offset())[:] = False
    rest = buf[mask]
    return bool((rest == fill).all().item()) if rest.numel() else True


def _p(t):
    return None if t is None else t.data_ptr()


def quant_rows(x, q, s, stream=None):
    from sdcb.gcdrnet_b200 import lib
    return lib().gcdr_k_quant_rows(_p(x), code(x.dtype), x.shape[0], x.shape[1], x.stride(0), _p(q), q.stride(0), _p(s),
                                   stream)


def i8_gemm(x, xs, w, ws, bias, out, relu=False, stream=None, **more):
    from sdcb.gcdrnet_b200 import I8GemmDesc, lib
    d = I8GemmDesc(M=x.shape[0], N=w.shape[0], K=x.shape[1], x=_p(x), ldx=x.stride(0), xs=_p(xs), w=_p(w),
                   ldw=w.stride(0), ws=_p(ws), bias=_p(bias), relu=int(relu), dtype=code(out.dtype), out=_p(out),
                   ldo=out.stride(0), **more)
    return lib().gcdr_k_i8_gemm(ctypes.byref(d), stream)


def block_norm(x=None, f=None, post=0, g1=None, b1=None, gate=None, gate_rows=0, scale=1.0, r=None, pre=0, g2=None,
               b2=None, y=None, q=None, qs=None, eps=1e-5, stream=None):
    from sdcb.gcdrnet_b200 import BlockNormDesc, lib
    some = x if x is not None else f
    ld = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    d = BlockNormDesc(rows=some.shape[0], C=some.shape[1], dtype=code(some.dtype), x=_p(x), ldx=ld(x), f=_p(f), ldf=ld(f),
                      post=post, g1=_p(g1), b1=_p(b1), eps1=eps, gate=_p(gate), ldg=ld(gate), gate_rows=gate_rows,
                      res_scale=scale, r=_p(r), ldr=ld(r), pre=pre, g2=_p(g2), b2=_p(b2), eps2=eps, y=_p(y), ldy=ld(y),
                      q=_p(q), ldq=ld(q), qs=_p(qs))
    return lib().gcdr_k_block_norm(ctypes.byref(d), stream)


# ------------------------------------------------------------------ plain forms

def ref_quant(x):
    """(q, scale) of quant_rows, exact: 127 x has 31 bits and its quotient by max|x| no border that 64 bits miss."""
    import torch
    v = x.double()
    top = v.abs().amax(1)
    fine = torch.isfinite(v).all(1)
    safe = torch.where(fine & (top > 0), top, torch.ones_like(top))
    q = torch.where(fine[:, None], torch.round(v * 127.0 / safe[:, None]), torch.zeros_like(v))
    s = (top.float().cpu().numpy() / np.float32(127)).astype(np.float32)   # IEEE division in fp32
    s = torch.from_numpy(s).to(x.device)
    return q.to(torch.int8), torch.where(fine, s, torch.full_like(s, float("nan")))


def ref_product(x, xs, w, ws, bias, relu, dtype):
    """(value, bound) of the product in 64 bits: the sum is exact; its conversion, the two scales and the sum with
    the bias are three roundings of fp32 (the last one with a single multiplication, fused), then the type's."""
    import torch
    acc = x.double() @ w.double().t()
    p = acc * xs.double()[:, None] * ws.double()
    v = p + (bias.double() if bias is not None else 0.0)
    rel, least = half_step(dtype)
    err = p.abs() * 2.01 * U + v.abs() * U + 2.0 ** -148
    err = err * (1 + rel) + v.abs() * (rel if dtype != torch.float32 else 0) + least
    return torch.relu(v) if relu else v, err


# A sum of C <= 32768 values as a group of threads forms it: at most 32 in a row per thread, five levels of shuffles,
# 32 warps' sums in a row, and the division by C.
SUMS = 32 + 5 + 32 + 1


def ref_norm(u, e, kind, g, b, eps):
    """(value, bound) of a norm of u, known to within e: first order in U and e."""
    if kind == 0:
        return u, e
    C = u.shape[1]
    if kind == LAYER:
        mean = u.mean(1, keepdim=True)
        # of the mean: its sum's roundings, and what u's own errors move it by
        dm = SUMS * U * u.abs().mean(1, keepdim=True) + e.mean(1, keepdim=True)
    else:
        mean, dm = 0.0, 0.0
    d = u - mean
    ed = e + dm + U * d.abs()
    var = d.square().mean(1, keepdim=True) + eps
    sd = var.sqrt()
    # of mean(d^2): 2 d ed by Cauchy-Schwarz, ed^2, its roundings (a square each and the sum), and the sum with eps
    rms = ed.square().mean(1, keepdim=True).sqrt()
    evar = 2 * sd * rms + rms.square() + (SUMS + 2) * U * var
    rho = 0.5 * evar / var * (1 + evar / var) + 2 * U        # of 1 / sqrt, with its two roundings
    h = d / sd
    eh = ed / sd + h.abs() * (rho + U)                       # and the product d * rstd
    if g is not None:
        h, eh = h * g.double(), (eh + U * h.abs()) * g.double().abs()
    if b is not None:
        h = h + b.double()
        eh = eh + U * h.abs()
    return h, eh * 1.01 + 2.0 ** -140


def ref_block(x=None, f=None, post=0, g1=None, b1=None, gate=None, gate_rows=0, scale=1.0, pre=0, g2=None, b2=None,
              eps=1e-5):
    """((v, bound), (h, bound)) in 64 bits."""
    import torch
    import struct
    scale = struct.unpack("f", struct.pack("f", scale))[0]
    eps = struct.unpack("f", struct.pack("f", eps))[0]
    if f is not None:
        u = f.double()
        u, e = ref_norm(u, torch.zeros_like(u), post, g1, b1, eps)
        if gate is not None:
            rows = torch.arange(u.shape[0], device=u.device) // gate_rows
            t = gate.double()[rows]
            u, e = u * t, (e + U * u.abs()) * t.abs()
        v, e = scale * u, (e + U * u.abs()) * abs(scale)
        if x is not None:
            v = v + x.double()
            e = e + U * v.abs()
    else:
        v = x.double()
        e = torch.zeros_like(v)
    return (v, e), ref_norm(v, e, pre, g2, b2, eps)


def stored(v, e, dtype):
    """The bound of a value known to within e once it is rounded to the type."""
    import torch
    rel, least = half_step(dtype)
    return e if dtype == torch.float32 else e * (1 + rel) + v.abs() * rel + least


def worst(got, want, bound):
    """Largest |got - want| in units of its bound (infinite where one has a value and the other none)."""
    import torch
    g = got.double()
    if not torch.equal(torch.isnan(g), torch.isnan(want)):
        return float("inf")
    fine = ~torch.isnan(want)
    if not fine.any():
        return 0.0
    return float(((g - want).abs() / bound)[fine].max().item())
