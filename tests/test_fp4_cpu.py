"""4-bit microscaled operators without a GPU: sizes, refusals, and the float64 restatement against itself."""
import copy
import ctypes as C
import pickle

import pytest
import torch

from block_lut_b200 import _lib
from block_lut_b200 import fp4 as F
from tests import _fp4_ref as R


def desc(kind=1, rows=4, cols=64):
    return _lib.FP4Desc(kind, 0, rows, cols)


@pytest.mark.parametrize("kind,rows,cols,codes,scales,tiled", [
    (1, 1, 1, 64, 8, 9216), (2, 1, 1, 64, 4, 8704), (1, 128, 128, 8192, 1024, 9216), (2, 129, 256, 129 * 128, 129 * 8, 4 * 8704),
    (1, 2816, 2048, 2816 * 1024, 2816 * 128, 22 * 16 * 9216)])
def test_sizes(kind, rows, cols, codes, scales, tiled):
    L, d = _lib.lib(), desc(kind, rows, cols)
    assert L.blut_fp4_codes_bytes(C.byref(d)) == codes
    assert L.blut_fp4_scales_bytes(C.byref(d)) == scales
    assert L.blut_fp4_tiled_bytes(C.byref(d)) == tiled


@pytest.mark.parametrize("d", [desc(0), desc(3), desc(rows=0), desc(cols=0), desc(rows=-1), desc(rows=1 << 31), desc(cols=(1 << 24) + 1)])
def test_bad_descriptions(d):
    L = _lib.lib()
    for f in (L.blut_fp4_codes_bytes, L.blut_fp4_scales_bytes, L.blut_fp4_tiled_bytes):
        assert f(C.byref(d)) == _lib.BLUT_ERR_INVALID
    assert L.blut_fp4_codes_bytes(None) == _lib.BLUT_ERR_INVALID
    P = 256
    assert L.blut_fp4_quantize(C.byref(d), P, 1, 1 << 25, None, d.rows, P, P, P, None) == _lib.BLUT_ERR_INVALID
    assert L.blut_fp4_dequantize(C.byref(d), P, P, P, P, 1, 1 << 25, None) == _lib.BLUT_ERR_INVALID
    assert L.blut_fp4_pack_tiled(C.byref(d), P, P, P, None) == _lib.BLUT_ERR_INVALID


def test_c_refusals():
    """Every refusal comes from the host, before any launch."""
    L, P, bad, uns = _lib.lib(), 256, _lib.BLUT_ERR_INVALID, _lib.BLUT_ERR_UNSUPPORTED
    d = desc()
    q = L.blut_fp4_quantize
    assert q(None, P, 1, 64, None, 4, P, P, P, None) == bad
    for hole in range(3):
        a = [P, P, P]
        a[hole] = None
        assert q(C.byref(d), a[0], 1, 64, None, 4, P, a[1], a[2], None) == bad
    assert q(C.byref(d), P, 1, 63, None, 4, P, P, P, None) == bad  # pitch below the columns
    assert q(C.byref(d), P, 1, 64, None, 5, P, P, P, None) == bad  # rows without an index
    assert q(C.byref(d), P, 1, 64, P, 0, P, P, P, None) == bad  # an index into nothing
    assert q(C.byref(d), P, 1, 64, None, 4, None, P, P, None) == bad  # nvfp4 without g
    assert q(C.byref(d), P, 1, 64, None, 4, P, P + 8, P, None) == bad  # alignment
    assert q(C.byref(d), P + 1, 1, 64, None, 4, P, P, P, None) == bad
    assert q(C.byref(d), P, 7, 64, None, 4, P, P, P, None) == uns
    s = L.blut_fp4_silu_mul_quantize
    assert s(C.byref(d), P, 1, 127, P, P, P, None) == bad
    assert s(None, P, 1, 128, P, P, P, None) == bad
    assert L.blut_fp4_dequantize(C.byref(d), P, P, P, P, 1, 63, None) == bad
    assert L.blut_fp4_dequantize(C.byref(d), P, P, P, P, 9, 64, None) == uns
    assert L.blut_fp4_global_scale(P, 1, 0, 64, 64, 0, P, None) == bad
    assert L.blut_fp4_global_scale(P, 1, 4, 64, 64, 1, P, None) == bad
    assert L.blut_fp4_global_scale(P, 1, 4, 64, 64, 0, P + 4, None) == bad
    assert L.blut_fp4_global_scale(P, 5, 4, 64, 64, 0, P, None) == uns
    assert L.blut_fp4_import(C.byref(d), None, P, P, P, None) == bad
    assert L.blut_fp4_export(C.byref(d), P, P, P, None, None) == bad


def mm_args(**kw):
    a = _lib.FP4MMArgs()
    a.w = desc(1, 256, 128)
    a.w_tiled = a.x_codes = a.x_scales = a.y = a.offsets = 256
    a.w_stride = 2 * 9216
    a.out_dtype, a.x_rows, a.y_ld = _lib.BF16, 8, 256
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [
    (dict(w_tiled=None), -1), (dict(x_codes=None), -1), (dict(x_scales=None), -1), (dict(y=None), -1), (dict(x_rows=0), -1),
    (dict(x_rows=(1 << 22) + 1), -1), (dict(y_ld=255), -1), (dict(num_experts=-1), -1), (dict(num_experts=1025), -1),
    (dict(num_experts=2, offsets=None), -1), (dict(num_experts=2, w_stride=9216), -1), (dict(num_experts=2, w_stride=18440), -1),
    (dict(w_tiled=264), -1), (dict(x_codes=260), -1), (dict(y=257), -1), (dict(out_dtype=3), -2), (dict(w=desc(9)), -1)])
def test_product_refusals(kw, rc):
    a = mm_args(**kw)
    assert _lib.lib().blut_fp4_matmul(C.byref(a), None) == rc
    assert _lib.lib().blut_fp4_matmul(None, None) == -1


def test_python_refusals():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        F.quantize_fp4(x)
    with pytest.raises(ValueError, match="CUDA"):
        F.silu_mul_quantize_fp4(x)
    with pytest.raises(ValueError, match="CUDA"):
        F.fp4_global_scale(x)
    with pytest.raises(ValueError, match="kind"):
        F.FP4Matrix.empty("fp4", 1, 1, "cpu")
    with pytest.raises(ValueError, match="codes"):
        F.FP4Matrix.from_checkpoint("nvfp4", torch.zeros(4, 31, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 64)
    with pytest.raises(ValueError, match="CUDA"):
        F.FP4Matrix.from_checkpoint("nvfp4", torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 64)
    with pytest.raises(ValueError, match="no global scale"):
        F._given_scale("mxfp4", 1.0, x.device)
    for g in (0.0, -1.0, float("inf"), float("nan"), 1e-40, 2e30, torch.ones(2), torch.ones(1, dtype=torch.float64)):
        with pytest.raises(ValueError, match="global_scale"):
            F._given_scale("nvfp4", g, x.device)
    m = F.FP4Matrix.empty("nvfp4", 4, 64, "cpu", torch.ones(1))
    w = F.FP4Weight("nvfp4", 128, 64, None, torch.zeros(9216, dtype=torch.uint8), 9216, torch.ones(1))
    ws = F.FP4Weight("nvfp4", 128, 64, 2, torch.zeros(2 * 9216, dtype=torch.uint8), 9216, torch.ones(2))
    off = torch.zeros(3, dtype=torch.int32)
    for bad, match in (((F.fp4_matmul, m, ws), "grouped"), ((F.fp4_grouped_matmul, m, w, off), "stack"),
                       ((F.fp4_grouped_matmul, m, ws, off[:2]), "offsets"), ((F.fp4_grouped_matmul, m, ws, off.long()), "offsets"),
                       ((F.fp4_matmul, x, w), "FP4Matrix"),
                       ((F.fp4_matmul, F.FP4Matrix.empty("mxfp4", 4, 64, "cpu"), w), "columns"),
                       ((F.fp4_matmul, F.FP4Matrix.empty("nvfp4", 4, 65, "cpu"), w), "columns"),
                       ((F.fp4_matmul, m, w, torch.zeros(4, 127)), "out must"),
                       ((F.fp4_matmul, m, w, torch.zeros(4, 128, dtype=torch.int32)), "output"),
                       ((F.fp4_matmul, m, w, torch.zeros(4, 128), torch.bfloat16), "output"),
                       ((F.fp4_matmul, m, w, torch.zeros(128, 4).t()), "contiguous"),
                       ((F.fp4_matmul, m, w, torch.zeros(1, 128).expand(4, -1)), "separate")):
        with pytest.raises(ValueError, match=match):
            bad[0](*bad[1:])
    with pytest.raises(ValueError, match="single"):
        F.FP4Linear(ws)
    with pytest.raises(ValueError, match="one kind"):
        F.FP4Weight.from_quantized([])
    with pytest.raises(ValueError, match="dtype"):
        F.dequantize_fp4(m, torch.int8)


@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
def test_restatement(kind):
    """Every value of the 4-bit form is its own quantisation, and rounding goes to the nearest one."""
    r = torch.Generator().manual_seed(0)
    b = R.BLOCK[kind]
    codes = torch.randint(0, 256, (5, 2 * b), generator=r, dtype=torch.uint8)
    codes[:, 0::b // 2] = 0x7F  # a 6 in every block fixes its scale (even column -6, odd column 6)
    scales = torch.randint(20, 100, (5, 4), generator=r, dtype=torch.uint8)
    v = R.values(codes, scales, kind, 4 * b, 0.5 if kind == "nvfp4" else 1.0)
    c, s = R.quantize(v, kind, 0.5 if kind == "nvfp4" else 1.0)
    assert torch.equal(s, scales) and torch.equal(c, codes)
    x = torch.randn(7, 3 * b + 5, generator=r)
    g = 0.001 if kind == "nvfp4" else 1.0
    c, s = R.quantize(x, kind, g)
    unit = R.values(torch.full_like(c, 0x22), s, kind, x.shape[1], g)  # code 2 is 1: the blocks' units
    t = (x.double() / unit).abs().clamp(max=6)
    best = (t[..., None] - R.LEVELS).abs().min(-1).values
    got = (R.values(c, s, kind, x.shape[1], g) / unit).abs()
    assert torch.allclose((t - got).abs(), best, rtol=0, atol=1e-12)


def test_linear_refusals():
    L = _lib.lib()
    d = desc(1, 256, 128)
    size = L.blut_fp4_linear_workspace_size
    assert size(C.byref(d), 8, 1) == 0 and size(C.byref(d), 8, 0) == 256 and size(C.byref(d), 9, 1) > 9 * 72
    assert size(C.byref(desc(2, 256, 128)), 3, 0) == 0
    assert size(C.byref(d), 0, 1) < 0 and size(C.byref(d), (1 << 22) + 1, 1) < 0 and size(None, 1, 1) < 0
    f = L.blut_fp4_linear
    a = mm_args()
    assert f(None, 256, 1, 128, 256, 1 << 20, None) == -1
    assert f(C.byref(a), None, 1, 128, 256, 1 << 20, None) == -1
    assert f(C.byref(a), 256, 1, 127, 256, 1 << 20, None) == -1  # pitch
    assert f(C.byref(a), 257, 1, 128, 256, 1 << 20, None) == -1  # alignment
    assert f(C.byref(a), 256, 4, 128, 256, 1 << 20, None) == -2
    assert f(C.byref(a), 256, 1, 128, None, 0, None) == -3  # g has no place
    assert f(C.byref(mm_args(x_rows=9, x_scale=256)), 256, 1, 128, 256, 64, None) == -3
    assert f(C.byref(mm_args(num_experts=2)), 256, 1, 128, 256, 1 << 20, None) == -1
    assert f(C.byref(mm_args(y=None, x_scale=256)), 256, 1, 128, None, 0, None) == -1
    w = F.FP4Weight("nvfp4", 128, 64, None, torch.zeros(9216, dtype=torch.uint8), 9216, torch.ones(1))
    lin = F.FP4Linear(w)
    for x in (torch.zeros(4, 63), torch.zeros(())):
        with pytest.raises(ValueError, match="x must be"):
            lin(x)
    with pytest.raises(ValueError, match="CUDA"):
        lin(torch.zeros(4, 64))


def test_packed_arguments():
    """The products' arguments are packed in the order and size of the C structure's fields."""
    assert F._MM.size == C.sizeof(_lib.FP4MMArgs)
    a = _lib.FP4MMArgs.from_buffer_copy(F._MM.pack(2, 0, 130, 70, 10, 11, 12, 3, 2, 21, 22, 23, 24, 25, 26, 27))
    assert (a.w.kind, a.w.reserved, a.w.rows, a.w.cols) == (2, 0, 130, 70)
    assert (a.w_tiled, a.w_stride, a.w_scale) == (10, 11, 12)
    assert (a.num_experts, a.offsets, a.out_dtype, a.x_codes, a.x_scales, a.x_scale) == (3, 21, 2, 22, 23, 24)
    assert (a.x_rows, a.y, a.y_ld) == (25, 26, 27)


@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
def test_operands_are_checked_where_they_are_read(kind):
    """Matrices and weights can be made and changed by hand: what a kernel would read past, or on the host, is refused."""
    b, unit = (72, 9216) if kind == "nvfp4" else (68, 8704)
    g = torch.ones(1) if kind == "nvfp4" else None

    def mat(n, dtype=torch.uint8, g=g):
        return F.FP4Matrix(kind, 4, 130, torch.zeros(n, dtype=dtype), g)

    def weight(n, experts=None, stride=4 * unit, g=g):
        return F.FP4Weight(kind, 200, 130, experts, torch.zeros(n, dtype=torch.uint8), stride, g)

    full = 4 * 2 * b
    x, w, ws, off = mat(full), weight(4 * unit), weight(12 * unit, 3, g=None), torch.zeros(4, dtype=torch.int32)
    for bad, match in ((mat(full - 1), "bytes"), (mat(full, torch.int8), "bytes"), (x, "CUDA")):
        for call in (lambda: F.dequantize_fp4(bad), bad.to_checkpoint, lambda: F.FP4Weight.from_quantized(bad),
                     lambda: F.FP4Weight.from_quantized([bad, bad])):
            with pytest.raises(ValueError, match=match):
                call()
    bad = mat(2 * full)
    bad.data = bad.data[::2]
    with pytest.raises(ValueError, match="bytes"):
        F.dequantize_fp4(bad)
    with pytest.raises(ValueError, match="CUDA"):
        F.fp4_matmul(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        F.fp4_grouped_matmul(x, ws, off)
    for bad, match in ((weight(4 * unit - 1), "bytes"), (weight(12 * unit - 1, 3), "bytes"), (weight(12 * unit, 3, 4 * unit - 16), "stride"),
                       (weight(12 * unit, 3, 5 * unit), "bytes"), (weight(4 * unit), "CUDA")):
        with pytest.raises(ValueError, match=match):
            F._mm_args(bad, bad.experts or 0, 0, 1, 0, 0, 0, 4, 0, 200)
    for t in (torch.ones(2), torch.ones(1, dtype=torch.float64), torch.ones(1, device="meta")):
        with pytest.raises(ValueError, match="global.scale"):
            F.dequantize_fp4(mat(full, g=t))
        with pytest.raises(ValueError, match="global.scale"):
            F._mm_args(weight(4 * unit, g=t), 0, 0, 1, 0, 0, 0, 4, 0, 200)
    with pytest.raises(ValueError, match="global.scale"):
        F._mm_args(weight(12 * unit, 3, g=torch.ones(6)[::2]), 3, 0, 1, 0, 0, 0, 4, 0, 200)
    m = F._new_matrix(kind, 4, 130, torch.zeros(1), g)
    assert m.data.numel() == full and m._operand()[0] == m.data.data_ptr()  # made to measure: taken as it is, until something is assigned
    for again in (copy.copy(m), copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        assert (again.kind, again.rows, again.cols) == (kind, 4, 130) and torch.equal(again.data, m.data)
        with pytest.raises(ValueError, match="CUDA"):
            again._operand()
    with pytest.raises(AttributeError):
        m.codes = m.data
    m.rows = 5
    with pytest.raises(ValueError, match="bytes"):
        m._operand()
    with pytest.raises(ValueError, match="stack"):
        F.fp4_grouped_matmul(x, weight(4 * unit, 0), off[:1])


def test_linear_attributes():
    """What is assigned after construction is checked like the constructor's arguments, and is what sizes go by."""
    w = F.FP4Weight("nvfp4", 128, 64, None, torch.zeros(9216, dtype=torch.uint8), 9216, torch.ones(1))
    ws = F.FP4Weight("nvfp4", 128, 64, 2, torch.zeros(2 * 9216, dtype=torch.uint8), 9216, torch.ones(2))
    lin = F.FP4Linear(w, 0.5)
    lin.weight = F.FP4Weight("nvfp4", 256, 32, None, torch.zeros(2 * 9216, dtype=torch.uint8), 9216, torch.ones(1))
    assert (lin.rows, lin.cols) == (256, 32)
    with pytest.raises(ValueError, match="x must be"):
        lin(torch.zeros(4, 64))
    with pytest.raises(ValueError, match="single"):
        lin.weight = ws
    for g in (0.0, float("nan"), torch.ones(2), torch.ones(1, dtype=torch.float64)):
        with pytest.raises(ValueError, match="act_scale"):
            lin.act_scale = g
    assert float(lin.act_scale) == 0.5 and lin.rows == 256
    lin.act_scale = None
    assert lin.act_scale is None
    # the workspace goes by whether a scale is given, not by what an earlier call of as many rows had
    assert F._linear_ws("nvfp4", 256, 32, 3, True) == 0 and F._linear_ws("nvfp4", 256, 32, 3, False) == 256
    with pytest.raises(ValueError, match="rows in one product"):
        F._linear_ws("nvfp4", 256, 32, F.MAX_ROWS + 1, True)


def test_overlap():
    """Against the bytes themselves, where pitches differ at least never missed."""
    r = torch.Generator().manual_seed(3)

    def draw(lo, hi):
        return int(torch.randint(lo, hi, (1,), generator=r))

    def taken(a, pitch, width, rows):
        return {a + i * pitch + j for i in range(rows) for j in range(width)}

    seen = [0, 0]
    for _ in range(3000):
        rows, pa = draw(1, 5), draw(4, 20)
        pb = pa if draw(0, 2) else draw(4, 20)
        wa, wb = draw(1, min(pa, pb) + 1), draw(1, pb + 1)
        a, b = draw(0, 60), draw(0, 60)
        shares = bool(taken(a, pa, wa, rows) & taken(b, pb, wb, rows))
        got = F._overlap(rows, a, pa, wa, b, pb, wb)
        assert got == shares if pa == pb or rows == 1 else got >= shares
        seen[got] += 1
    assert min(seen) > 300
