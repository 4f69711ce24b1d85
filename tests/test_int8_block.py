"""The framework's shifted-MLP block with its products in 8 bits, as the layer entries chain it:

    gcdr_k_up_add / gcdr_k_ln_finalize  (norm, shift along H)  ->  gcdr_k_quant_rows  ->  gcdr_k_i8_gemm (fc1)
    ->  gcdr_k_dw_gelu_shift  ->  gcdr_k_quant_rows  ->  gcdr_k_i8_gemm (fc2, fp32)  ->  gcdr_k_ln_finalize (residual, norm)

on the models' parameters, from the block's input to its output, against the oracle's fp32 block (shift along H and the
trailing norm included).  The shift moves channel groups between tokens, so it comes before a token's scale is taken:
gcdr_k_block_norm, which has no shift, cannot hand its int8 rows to fc1 here.
"""
import numpy as np
import pytest

import golden_data as G
from oracle import gcdr_oracle as O

BLOCKS = [(net, name) for net in ("gc", "dr") for name in ("block1", "block2", "dblock1", "dblock2")]
H, W = 18, 26
EPS = 1e-5


@pytest.fixture(scope="module")
def nets():
    return {"gc": O.GcdrNet.load(G.GC_PATH), "dr": O.GcdrNet.load(G.DR_PATH)}


def _t(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).double()


def _f16(t):
    return t.half().double()


def _norm(t, g, b):
    import torch
    d = t - t.mean(-1, keepdim=True)
    return d / torch.sqrt(d.square().mean(-1, keepdim=True) + EPS) * _t(g) + _t(b)


def _shift(t, spec):
    """[H][W][C]: group g of the channels, out[y] = in[y + off] along H (axis 2) or W (axis 3), zeros beyond."""
    import torch
    axis, ends, offs = spec
    dim, out, at = axis - 2, t.clone(), 0
    n = t.shape[dim]
    for end, off in zip(ends, offs):
        part = t[..., at:end]
        moved = torch.zeros_like(part)
        if abs(off) < n:
            moved.narrow(dim, max(-off, 0), n - abs(off)).copy_(part.narrow(dim, max(off, 0), n - abs(off)))
        out[..., at:end] = moved
        at = end
    return out


def _rows8(t):
    """Rows as int8 with a scale each stand for them."""
    import torch
    top = t.abs().amax(-1, keepdim=True)
    safe = torch.where(top > 0, top, torch.ones_like(top))
    return torch.round(t * 127 / safe) * top / 127


def _chain64(blk, x, shift=True):
    """The 8-bit chain in 64 bits: rounded where the entries store fp16 or int8, nowhere else (the first norm takes x as its
    producer holds it, the residual x as stored)."""
    import torch
    import torch.nn.functional as F
    C = x.shape[-1]
    h = _f16(_norm(x, *blk.norm2))
    if shift:
        h = _shift(h, blk.shift_h)
    (w1, b1), (w2, b2), (wd, bd) = blk.fc1, blk.fc2, blk.dw
    h = _f16(_rows8(h) @ _rows8(_rows_of(w1)).t() + _t(b1))
    h = F.conv2d(h.permute(2, 0, 1)[None], _t(wd), _t(bd), padding=1, groups=C)[0].permute(1, 2, 0)
    h = _f16(_shift(0.5 * h * (1 + torch.erf(h / 2 ** 0.5)), blk.shift_w))
    h = _rows8(h) @ _rows8(_rows_of(w2)).t() + _t(b2)
    return _f16(_norm(_f16(x) + h, *blk.norm_out))


def _rows_of(w):
    """A Gemm's B operand [K][N] (out = x @ B) as rows of output channels [N][K]."""
    return _t(np.asarray(w, np.float32).T)


def _rms(t):
    return float(t.square().mean().sqrt())


def _input(nets, net, name, seed):
    """A block's input x as the net makes it, a normed token map (block1, block2) or a join (dblock1, dblock2), and what it is
    made of."""
    import torch
    g = torch.Generator().manual_seed(seed)
    blk = getattr(nets[net], name)
    C = blk.dw[0].shape[0]
    if name in ("block1", "block2"):
        u = torch.randn(H, W, C, generator=g)
        gain, shift = nets[net].pe3_norm if name == "block1" else nets[net].pe4_norm
        return {"u": u, "gain": gain, "shift": shift, "x": _norm(u.double(), gain, shift)}
    d = torch.randn(H // 2, W // 2, C, generator=g).half()
    skip = torch.randn(H, W, C, generator=g).clamp(min=0).half()
    x = O.add(O.relu(O.resize2x(d.float().numpy())), skip.float().numpy())
    return {"d": d, "skip": skip, "x": _t(x)}


@pytest.mark.parametrize("net,name", BLOCKS)
def test_the_chain_in_64_bits(nets, net, name):
    """The chain's error is that of its roundings: less than a hundredth of the block's output (rms).  Without the shift
    along H it is another function, many times further off."""
    blk, i = getattr(nets[net], name), _input(nets, net, name, 7)
    want = _t(O.shifted_block(np.ascontiguousarray(i["x"].float().numpy()), blk))
    err = _rms(_chain64(blk, i["x"]) - want)
    bare = _rms(_chain64(blk, i["x"], shift=False) - want)
    print("%s.%s C %d: rms error %.4f of %.3f; without the shift %.4f" % (net, name, want.shape[-1], err, _rms(want), bare))
    assert err < 0.01 * _rms(want) and bare > 20 * err


def _device_chain(blk, i):
    """The entries on one stream, none waited for; (x, its shifted norm, the block's output) as they are stored."""
    import ctypes

    import torch
    from gpu_util import Act, Shift
    from int8_util import i8_gemm, quant_rows
    from sdcb.gcdrnet_b200 import lib
    L, T, C = lib(), H * W, i["x"].shape[-1]
    eps = ctypes.c_float(EPS)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).to("cuda:0")  # noqa: E731
    half = lambda *s: torch.full(s, float("nan"), dtype=torch.float16, device="cuda:0")  # noqa: E731
    shift_h, shift_w = (Shift.of(*s[1:]) for s in (blk.shift_h, blk.shift_w))
    (g2, b2), (go, bo) = ([dev(v) for v in p] for p in (blk.norm2, blk.norm_out))
    zero = torch.zeros(C, device="cuda:0")

    def weights(fc):
        w, b = dev(np.asarray(fc[0]).T), dev(fc[1])
        q, s = torch.empty(C, C, dtype=torch.int8, device="cuda:0"), torch.empty(C, device="cuda:0")
        assert quant_rows(w, q, s) == 0
        return q, s, b

    (w1, s1, c1), (w2, s2, c2) = weights(blk.fc1), weights(blk.fc2)
    x, h, f, m, out = half(T, C), half(T, C), half(T, C), half(T, C), half(T, C)
    xa, oa = Act(x.data_ptr(), H, W, C, 0), Act(out.data_ptr(), H, W, C, 0)
    q, qs, sums = torch.empty(T, C, dtype=torch.int8, device="cuda:0"), torch.empty(T, device="cuda:0"), torch.empty(T, C, device="cuda:0")
    if "u" in i:
        u, g, b = i["u"].to("cuda:0"), dev(i["gain"]), dev(i["shift"])
        assert L.gcdr_k_ln_finalize(u.data_ptr(), 1, H, W, C, zero.data_ptr(), None, g.data_ptr(), b.data_ptr(), eps, g2.data_ptr(),
                                    b2.data_ptr(), eps, ctypes.byref(shift_h), ctypes.byref(xa), h.data_ptr(), None) == 0
    else:
        d, skip = i["d"].to("cuda:0"), i["skip"].to("cuda:0")
        sa = Act(skip.data_ptr(), H, W, C, 0)
        assert L.gcdr_k_up_add(d.data_ptr(), ctypes.byref(sa), ctypes.byref(xa), g2.data_ptr(), b2.data_ptr(), eps,
                               ctypes.byref(shift_h), h.data_ptr(), None) == 0
    assert quant_rows(h, q, qs) == 0
    assert i8_gemm(q, qs, w1, s1, c1, f) == 0
    wt, bd = dev(np.asarray(blk.dw[0]).reshape(C, 9).T), dev(blk.dw[1])
    assert L.gcdr_k_dw_gelu_shift(f.data_ptr(), H, W, C, wt.data_ptr(), bd.data_ptr(), ctypes.byref(shift_w), m.data_ptr(), None) == 0
    assert quant_rows(m, q, qs) == 0
    assert i8_gemm(q, qs, w2, s2, None, sums) == 0
    assert L.gcdr_k_ln_finalize(sums.data_ptr(), 1, H, W, C, c2.data_ptr(), x.data_ptr(), go.data_ptr(), bo.data_ptr(), eps, None,
                                None, ctypes.c_float(0), None, ctypes.byref(oa), None, None) == 0
    torch.cuda.synchronize()
    return [t.double().cpu().view(H, W, C) for t in (x, h, out)]


@pytest.mark.gpu
@pytest.mark.parametrize("net,name", BLOCKS)
def test_the_chain_on_the_device(nets, net, name):
    """The entries' block against the fp32 block and against the same chain in 64 bits.  The two chains round the same
    values; fp32 and 64 bits part where one of about 2^11 stored fp16 values falls on the other side, which moves
    an int8 value by a step in one of eight such cases at most: some 2^-14 of them, each twelve times the variance of a
    rounding, is under a fiftieth of the chain's own error in each of its two roundings, and a fifth is allowed."""
    blk, i = getattr(nets[net], name), _input(nets, net, name, 7)
    want = _t(O.shifted_block(np.ascontiguousarray(i["x"].float().numpy()), blk))
    plain = _chain64(blk, i["x"])
    err = _rms(plain - want)
    x, h, out = _device_chain(blk, i)
    # stored fp16: half a step, and fp32 arithmetic of some hundred operations before it
    assert ((x - i["x"]).abs() <= (2.0 ** -11 + 2.0 ** -17) * i["x"].abs() + 2.0 ** -17).all()
    wh = _shift(_norm(i["x"], *blk.norm2), blk.shift_h)
    assert ((h - wh).abs() <= (2.0 ** -11 + 2.0 ** -17) * wh.abs() + 2.0 ** -16).all()
    print("%s.%s: rms error %.4f, of the chain in 64 bits %.4f, between them %.5f" % (net, name, _rms(out - want), err, _rms(out - plain)))
    assert _rms(out - plain) <= 0.2 * err
    assert _rms(out - want) <= 1.2 * err
