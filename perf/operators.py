"""The 8-bit token operators, measured: rows rounded to int8 with a scale each (gcdr_k_quant_rows), the
int8 matrix product with scales for each token and channel (gcdr_k_i8_gemm), and the norms around a block
with its gate and residual scale (gcdr_k_block_norm), alone and as one step (norm, rounding and product).

With `own` false, run() computes them from elementary torch operations; with `own` true it calls the
library.  Sizes are those of the shifted-MLP blocks (channels 128 to 512; a 1600x1152 page has 7200 tokens at
/16 and 1800 at /32, a batch of eight pages 57600) and generic wider layers."""
import ctypes

import torch

own = False

_DT = {"f16": (torch.float16, 0), "bf16": (torch.bfloat16, 1), "f32": (torch.float32, 2)}
_NORM = {"none": 0, "layer": 1, "rms": 2}
_EPS = 1e-5


def listed():
    return [
        # the bottleneck of one 32x32 thumbnail: a single token through a 512-channel layer (latency)
        {"name": "product one token", "op": "product", "rows": 1, "k": 512, "n": 512, "type": "f16", "relu": False},
        # one token of a wide layer: the weights' bytes are all there is
        {"name": "product one token wide", "op": "product", "rows": 1, "k": 8192, "n": 8192, "type": "bf16", "relu": False},
        # the DR bottleneck of one 1600x1152 page (36 x 50 tokens)
        {"name": "product page bottleneck", "op": "product", "rows": 1800, "k": 512, "n": 512, "type": "f16", "relu": False},
        # the 256-channel blocks of a batch of eight pages at /16
        {"name": "product eight pages", "op": "product", "rows": 57600, "k": 256, "n": 256, "type": "f16", "relu": True},
        # odd sizes: the last tile is ragged in every direction, fp32 results
        {"name": "product ragged", "op": "product", "rows": 1213, "k": 1000, "n": 1037, "type": "f32", "relu": True},
        # a wide layer over a long batch: arithmetic alone
        {"name": "product wide", "op": "product", "rows": 8192, "k": 8192, "n": 8192, "type": "bf16", "relu": False},
        # activations of a wide layer
        {"name": "rounding wide", "op": "quant", "rows": 16384, "c": 8192, "type": "bf16"},
        # fp32 rows of odd length: no row but the first is aligned
        {"name": "rounding ragged", "op": "quant", "rows": 4099, "c": 1037, "type": "f32"},
        # one page's block at /16: norm of the block's output, layer scale, residual, the next norm
        {"name": "norms page", "op": "norm", "rows": 7200, "c": 256, "type": "f16", "post": "layer", "gate": "all", "pre": "layer"},
        # a wide block over eight sequences of 2048 tokens, a gate for each sequence
        {"name": "norms wide", "op": "norm", "rows": 16384, "c": 4096, "type": "bf16", "post": "rms", "gate": "sequence", "pre": "rms"},
        # odd channels, a gate for every token, fp32
        {"name": "norms ragged", "op": "norm", "rows": 2111, "c": 1037, "type": "f32", "post": "none", "gate": "token", "pre": "layer"},
        # the step in use: the norms of eight pages' tokens, rounded rows out, and the product that takes them
        {"name": "step eight pages", "op": "step", "rows": 57600, "c": 256, "n": 256, "type": "f16", "post": "layer", "gate": "all", "pre": "layer", "relu": False},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["product", "product", "quant", "norm", "norm", "step"])
    kind = rng.choice(["f16", "bf16", "f32"])
    c = {"op": op, "type": kind}
    if op == "product":
        rows, k, n = _log(rng, 1, 57600), _log(rng, 16, 8192), _log(rng, 1, 8192)
        while rows * k * n > 8192 ** 3 // 4 or rows * n > 1 << 27:
            rows = max(1, rows // 2)
        c.update(rows=rows, k=k, n=n, relu=rng.random() < 0.5)
        return c
    c["rows"], c["c"] = _log(rng, 1, 57600), _log(rng, 8, 8192)
    if rng.random() < 0.5:
        c["c"] = -(-c["c"] // 8) * 8
    while c["rows"] * c["c"] > 1 << 25:
        c["rows"] //= 2
    if op != "quant":
        c.update(post=rng.choice(["none", "layer", "rms"]), gate=rng.choice(["none", "all", "sequence", "token"]),
                 pre=rng.choice(["layer", "rms"]))
    if op == "step":
        # 16-bit streams only: a step of the rounding that falls the other way, which 32-bit sums in another order
        # can cause, is within 16 bits' error of the product and beyond that of 32
        c.update(type=rng.choice(["f16", "bf16"]), n=_log(rng, 16, 1024), relu=rng.random() < 0.5)
    return c


def _gate_rows(case):
    """Tokens that share a row of the gate (0: there is no gate)."""
    rows = case["rows"]
    return {"none": 0, "all": rows, "sequence": -(-rows // 8), "token": 1}[case["gate"]]


def _quant(x):
    """Rows to int8: scale = max|x| / 127, q = x * 127 / max|x| to nearest even (in 64 bits: next to a border 32 lose)."""
    top = x.abs().amax(1, keepdim=True).double()
    scale = (top.float() / 127.0)[:, 0]
    q = torch.round(x.double() * 127.0 / torch.where(top > 0, top, torch.ones_like(top)))
    return q.to(torch.int8), scale


def _padded(q):
    """Rows at a pitch of a multiple of 16 bytes, as the product takes them; the padding holds no zeros."""
    ld = -(-q.shape[1] // 16) * 16
    buf = torch.full((q.shape[0], ld), 77, dtype=torch.int8, device=q.device)
    buf[:, : q.shape[1]] = q
    return buf[:, : q.shape[1]]


def _weights(s, n, k, g):
    q, s["ws"] = _quant(torch.randn(n, k, generator=g, device="cuda") / k ** 0.5)
    s["w"] = _padded(q)
    s["bias"] = torch.randn(n, generator=g, device="cuda") * 0.1


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, rows = _DT[case["type"]][0], case["rows"]
    s = {"case": case}

    def act(c):
        # token activations: unit normal with a few channels of larger range
        return torch.randn(rows, c, generator=g, device="cuda") * (1 + 4 * (torch.rand(c, generator=g, device="cuda") > 0.97))

    if case["op"] == "product":
        q, s["xs"] = _quant(act(case["k"]))
        s["x"] = _padded(q)
        _weights(s, case["n"], case["k"], g)
        s["out"] = torch.empty(rows, case["n"], dtype=dt, device="cuda")
        return s
    c = case["c"]
    ld = -(-c // 16) * 16
    s["x"] = act(c).to(dt)
    s["q"] = torch.empty(rows, ld, dtype=torch.int8, device="cuda")[:, :c]
    s["qs"] = torch.empty(rows, dtype=torch.float32, device="cuda")
    if case["op"] == "quant":
        return s
    s["f"] = (act(c) * 0.5 + 0.1).to(dt)
    for name in ("g1", "g2"):
        s[name] = 1 + 0.1 * torch.randn(c, generator=g, device="cuda")
    for name, norm in (("b1", case["post"]), ("b2", case["pre"])):
        s[name] = 0.1 * torch.randn(c, generator=g, device="cuda") if norm == "layer" else None
    per = _gate_rows(case)
    s["gate"] = (0.3 * torch.randn(-(-rows // per), c, generator=g, device="cuda")).to(dt) if per else None
    s["scale"] = 0.7
    s["r"], s["y"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
    if case["op"] == "step":
        _weights(s, case["n"], c, g)
        s["out"] = torch.empty(rows, case["n"], dtype=dt, device="cuda")
    return s


def _norm(v, kind, gain, shift):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v * torch.rsqrt(v.square().mean(1, keepdim=True) + _EPS) * gain
    return v if shift is None else v + shift


def _block(s, case):
    """(residual stream, normed stream), both in 32 bits."""
    u = _norm(s["f"].float(), case["post"], s["g1"], s["b1"])
    per = _gate_rows(case)
    if per:
        u = u * s["gate"].float().repeat_interleave(per, 0)[: case["rows"]]
    v = s["x"].float() + s["scale"] * u
    return v, _norm(v, case["pre"], s["g2"], s["b2"])


def _product(x, xs, w, ws, bias, relu):
    v = (x.float() @ w.float().t()) * xs[:, None] * ws + bias
    return torch.relu(v) if relu else v


def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    dt = _DT[case["type"]][0]
    if case["op"] == "product":
        return _product(s["x"], s["xs"], s["w"], s["ws"], s["bias"], case["relu"]).to(dt)
    if case["op"] == "quant":
        return _quant(s["x"].float())
    v, y = _block(s, case)
    if case["op"] == "norm":
        return v.to(dt), y.to(dt)
    q, scale = _quant(y)
    return v.to(dt), _product(q, scale, s["w"], s["ws"], s["bias"], case["relu"]).to(dt)


def _own_block(gcdr, s, case, stream):
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    rounded = case["op"] == "step"
    x, per, y = s["x"], _gate_rows(case), None if rounded else s["y"]
    c = x.shape[1]
    d = gcdr.BlockNormDesc(
        rows=case["rows"], C=c, dtype=_DT[case["type"]][1], x=ptr(x), ldx=c, f=ptr(s["f"]), ldf=c,
        post=_NORM[case["post"]], g1=ptr(s["g1"]), b1=ptr(s["b1"]), eps1=_EPS, gate=ptr(s["gate"]), ldg=c,
        gate_rows=per, res_scale=s["scale"], r=ptr(s["r"]), ldr=c, pre=_NORM[case["pre"]], g2=ptr(s["g2"]),
        b2=ptr(s["b2"]), eps2=_EPS, y=ptr(y), ldy=c, q=ptr(s["q"]) if rounded else None, ldq=s["q"].stride(0),
        qs=ptr(s["qs"]) if rounded else None)
    gcdr.check(gcdr.lib().gcdr_k_block_norm(ctypes.byref(d), stream))


def _own_product(gcdr, s, case, x, xs, stream):
    w, out = s["w"], s["out"]
    d = gcdr.I8GemmDesc(
        M=x.shape[0], N=w.shape[0], K=x.shape[1], x=x.data_ptr(), ldx=x.stride(0), xs=xs.data_ptr(),
        w=w.data_ptr(), ldw=w.stride(0), ws=s["ws"].data_ptr(), bias=s["bias"].data_ptr(), relu=int(case["relu"]),
        dtype=_DT[case["type"]][1], out=out.data_ptr(), ldo=out.stride(0))
    gcdr.check(gcdr.lib().gcdr_k_i8_gemm(ctypes.byref(d), stream))
    return out


def _run_own(s, case):
    import sdcb.gcdrnet_b200 as gcdr
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "product":
        return _own_product(gcdr, s, case, s["x"], s["xs"], stream)
    if case["op"] == "quant":
        x, q = s["x"], s["q"]
        gcdr.check(gcdr.lib().gcdr_k_quant_rows(x.data_ptr(), _DT[case["type"]][1], case["rows"], case["c"], case["c"],
                                                q.data_ptr(), q.stride(0), s["qs"].data_ptr(), stream))
        return q, s["qs"]
    _own_block(gcdr, s, case, stream)
    if case["op"] == "norm":
        return s["r"], s["y"]
    return s["r"], _own_product(gcdr, s, case, s["q"], s["qs"], stream)


def work(case):
    size = {"f16": 2, "bf16": 2, "f32": 4}[case["type"]]
    rows = case["rows"]
    if case["op"] == "product":
        k, n = case["k"], case["n"]
        return {"bytes": rows * k + n * k + 4 * rows + 8 * n + rows * n * size, "flops": 2 * rows * n * k}
    c = case["c"]
    if case["op"] == "quant":
        return {"bytes": rows * c * (size + 1) + 4 * rows, "flops": 4 * rows * c}
    per = _gate_rows(case)
    gates = -(-rows // per) * c * size if per else 0
    stream = rows * c * size * 3 + gates + 4 * c * ((case["post"] != "none") + (case["post"] == "layer") + 1 + (case["pre"] == "layer"))
    if case["op"] == "norm":
        return {"bytes": stream + rows * c * size, "flops": 16 * rows * c}
    n = case["n"]
    return {"bytes": stream + n * c + 8 * n + rows * n * size, "flops": 20 * rows * c + 2 * rows * n * c}


def exact(case, seed):
    s = prepare(case, seed)
    rows = case["rows"]

    def product(q, scale):
        # int8 values and their sums are exact in 64 bits
        t = torch.matmul(q.to(torch.float64), s["w"].to(torch.float64).transpose(0, 1))
        t = t.mul_(scale.to(torch.float64).view(-1, 1)).mul_(s["ws"].to(torch.float64)).add_(s["bias"].to(torch.float64))
        return t.clamp_(min=0) if case["relu"] else t

    def rounded(x):
        top = torch.linalg.vector_norm(x, float("inf"), dim=1)
        share = x / torch.where(top == 0, 1.0, top)[:, None]
        return torch.round(share.mul_(127)), top / 127

    if case["op"] == "product":
        return product(s["x"], s["xs"])
    if case["op"] == "quant":
        # the whole numbers are compared with the plain form's; the scale has a value in 64 bits
        return None, rounded(s["x"].to(torch.float64))[1]

    def normed(v, kind, gain, shift):
        if kind == "none":
            return v
        if kind == "layer":
            spread, mid = torch.var_mean(v, dim=1, keepdim=True, correction=0)
            v = (v - mid) / torch.sqrt(spread + _EPS)
        else:
            v = v / torch.sqrt(torch.linalg.vecdot(v, v)[:, None] / v.shape[1] + _EPS)
        v = v * gain.to(torch.float64)
        return v if shift is None else v + shift.to(torch.float64)

    u = normed(s["f"].to(torch.float64), case["post"], s["g1"], s["b1"])
    if s["gate"] is not None:
        u = u * s["gate"].to(torch.float64)[torch.arange(rows, device="cuda") // _gate_rows(case)]
    stream = s["x"].to(torch.float64) + s["scale"] * u
    after = normed(stream, case["pre"], s["g2"], s["b2"])
    if case["op"] == "norm":
        return stream, after
    return stream, product(*rounded(after))
