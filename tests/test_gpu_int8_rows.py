"""The row operators (gcdr_k_quant_rows, gcdr_k_block_norm) over more rows than the GPU holds at once, against their
64-bit forms: blocks walk several rows each, with the next row's operands and gate on their way, and the last pass is
ragged.  And rows that lie further apart than 32 bits reach."""
import pytest

from int8_util import DTYPES, LAYER, RMS, block_norm, quant_rows, ref_block, ref_quant, stored, strided, torch_dtype, untouched, worst
from test_gpu_int8 import _block, _check_norm, _gen, _norm_outputs, _rand

pytestmark = pytest.mark.gpu


def _at_once(C):
    """Rows that all SMs hold at once, at most: 2048 threads each, 8 or more to a row and at most 32 elements a thread."""
    from sdcb.gcdrnet_b200 import lib
    return lib().gcdr_device_sms() * 2048 // max(8, -(-C // 32))


# C, rows (of several passes and a rest, none a multiple of the groups of a block)
LONG = [(5, 120011), (40, 80003), (64, 76001), (96, 120001), (250, 80001), (256, 80003), (384, 30011), (700, 20011), (1037, 19003),
        (1536, 9001), (2046, 9501), (2048, 9501), (4096, 5003), (8192, 2501), (12288, 1601), (16384, 1201), (32768, 613)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C,rows", LONG)
def test_quant_rows_of_several_passes(C, rows, dtype):
    import torch
    assert rows > _at_once(C)
    x = _rand(_gen(C), rows, C).to(torch_dtype(dtype))
    x[rows - 1] = 0
    x[rows // 2, C // 2] = float("inf")
    q = torch.full((rows, C), 99, dtype=torch.int8, device="cuda:0")
    s = torch.full((rows,), -1.0, device="cuda:0")
    assert quant_rows(x, q, s) == 0
    wq, ws = ref_quant(x)
    assert torch.equal(q, wq)
    assert torch.equal(torch.isnan(s), torch.isnan(ws)) and torch.equal(s.nan_to_num(-2.0), ws.nan_to_num(-2.0))


# post, gate rows, pre: every norm, every way that a gate is shared (a divisor that is no power of two, all, one each)
KINDS = [(LAYER, "all", LAYER), (RMS, 977, RMS), (0, 1, LAYER), (LAYER, None, 0), (RMS, 3, LAYER)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C,rows", LONG)
def test_block_norm_of_several_passes(C, rows, dtype):
    """Both streams and int8 rows."""
    assert rows > _at_once(C)
    i = LONG.index((C, rows)) + DTYPES.index(dtype)
    post, gate, pre = KINDS[i % len(KINDS)]
    t = _block(C, rows, dtype, post, gate, pre)
    _check_norm(t, _norm_outputs(t))


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("C,rows", [(40, 80003), (256, 40013), (1037, 19003), (2046, 5003), (4096, 2501)])
def test_every_kind_of_several_passes(C, rows, kind):
    """Each norm and gate, without int8 rows, at a pitch."""
    assert rows > _at_once(C)
    dtype = DTYPES[(C + KINDS.index(kind)) % 3]
    t = _block(C, rows, dtype, kind[0], kind[1], kind[2], seed=3, pad=8)
    _check_norm(t, _norm_outputs(t, pad=8, quant=False))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C,rows", [(40, 80003), (256, 40013), (1037, 19003), (2046, 5003), (4096, 2501)])
def test_in_place_of_several_passes(C, rows, dtype):
    """r on x and y on f: a row is loaded ahead, never after it was written."""
    import torch
    assert rows > _at_once(C)
    t = _block(C, rows, dtype, LAYER, 7, RMS)
    (v, ev), (h, eh) = ref_block(**t)
    x, f = t["x"].clone(), t["f"].clone()
    t.update(x=x, f=f)
    qs = torch.full((rows,), -1.0, device="cuda:0")
    q = torch.full((rows, C), 99, dtype=torch.int8, device="cuda:0")
    assert block_norm(**t, r=x, y=f, q=q, qs=qs) == 0
    assert worst(x, v, stored(v, ev, x.dtype) + 1e-300) <= 1.0
    assert worst(f, h, stored(h, eh, f.dtype) + 1e-300) <= 1.0
    steps, room = 127 * h / h.abs().amax(1, keepdim=True), 0.5 + 127 * 2.02 * eh.amax(1, keepdim=True) / h.abs().amax(1, keepdim=True)
    assert ((q.double() - steps).abs() <= room).all()


def test_only_some_rows_hold_an_infinity():
    """A row's infinity or NaN stays its own in every pass: the reductions of the next row start afresh."""
    import torch
    for C, rows in ((64, 80003), (1037, 19003), (4096, 2501)):
        x = _rand(_gen(C), rows, C)
        bad = torch.arange(0, rows, 5, device="cuda:0")
        x[bad, bad % C] = float("nan")
        x[bad[::2], (bad[::2] * 7) % C] = float("inf")
        t = {"x": x, "pre": LAYER}
        o = _norm_outputs(t)
        assert block_norm(**t, y=o["y"], q=o["q"], qs=o["qs"]) == 0
        is_bad = torch.zeros(rows, dtype=torch.bool, device="cuda:0")
        is_bad[bad] = True
        assert torch.equal(torch.isnan(o["qs"]), is_bad)
        assert torch.equal(torch.isnan(o["y"]).all(1), is_bad) and torch.equal(torch.isnan(o["y"]).any(1), is_bad)
        assert (o["q"][bad] == 0).all()
        keep = ~is_bad
        _, (h, eh) = ref_block(x=x[keep], pre=LAYER)
        assert worst(o["y"][keep], h, eh + 1e-300) <= 1.0


def test_offsets_past_32_bits():
    """Rows at places beyond 2^32 elements of their buffers: 16-byte pieces, pairs and single elements."""
    import torch
    rows, ld = 2101, (1 << 21) + 8
    assert (rows - 40) * ld > 1 << 32
    wide, _ = strided(rows, 250, ld, torch.float16, 7.0)
    out, _ = strided(rows, 250, ld, torch.float16, 9.0)
    q, _ = strided(rows, 250, ld, torch.int8, 99)
    s = torch.full((rows,), -1.0, device="cuda:0")
    for C in (248, 250, 249):
        t = {"x": wide[:, :C], "pre": RMS}
        t["x"].copy_(_rand(_gen(C), rows, C))
        assert block_norm(**t, y=out[:, :C], q=q[:, :C], qs=s) == 0
        _, (h, eh) = ref_block(**t)
        assert worst(out[:, :C], h, stored(h, eh, torch.float16)) <= 1.0
        assert (out[:, C:] == 9.0).all() if C == 248 else True
        top = h.abs().amax(1, keepdim=True)
        assert ((q[:, :C].double() - 127 * h / top).abs() <= 0.5 + 127 * 2.02 * eh.amax(1, keepdim=True) / top).all()
        assert quant_rows(t["x"], q[:, :C], s) == 0
        wq, ws = ref_quant(t["x"])
        assert torch.equal(q[:, :C], wq) and torch.equal(s, ws)
    # the block's output and its gate so far away too
    t = {"f": wide[:, :248], "post": LAYER, "gate": wide[:, :248], "gate_rows": 1, "scale": 0.5}
    assert block_norm(**t, r=out[:, :248]) == 0
    (v, ev), _ = ref_block(**t)
    assert worst(out[:, :248], v, stored(v, ev, torch.float16)) <= 1.0
