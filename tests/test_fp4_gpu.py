"""The 4-bit microscaled operators on the GPU against their float64 restatement."""
import pytest
import torch

from tests import _fp4_ref as R

pytestmark = pytest.mark.gpu

KINDS = ["nvfp4", "mxfp4"]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def fp4():
    from block_lut_b200 import fp4 as F
    return F


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(rows, cols, dtype, seed=0, spread=2.0):
    r = gen(seed)
    x = torch.randn(rows, cols, generator=r, device="cuda") * torch.exp(spread * torch.randn(rows, cols, generator=r, device="cuda"))
    return x.to(dtype)


def g_of(kind, x, pow2=False):
    if kind == "mxfp4":
        return None
    a = x.double().abs().max().clamp(min=1e-20) / 2688
    g = torch.exp2(torch.log2(a).ceil()) if pow2 else a * 1.07
    return g.float().reshape(1)


def assert_same_codes(q, ref, what=""):
    codes, scales = q.to_checkpoint()
    assert torch.equal(scales, ref[1]), f"{what}: {int((scales != ref[1]).sum())} scales differ"
    assert torch.equal(codes, ref[0]), f"{what}: {int((codes != ref[0]).sum())} code bytes differ"


# --------------------------------------------------------------------- quantisation --
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 16), (1, 1), (3, 15), (8, 33), (9, 127), (17, 128), (5, 129), (2, 500), (7, 513),
                                       (40, 1408), (1, 2048), (33, 2056)])
@pytest.mark.parametrize("pow2", [False, True])
def test_quantize_bits(kind, dtype, rows, cols, pow2):
    F = fp4()
    x = rand(rows, cols, dtype, rows * 7 + cols)
    g = g_of(kind, x, pow2)
    q = F.quantize_fp4(x, kind, global_scale=g)
    ref = R.quantize(x, kind, 1.0 if g is None else g)
    assert_same_codes(q, ref)
    # the way back is q * s * g, one float32 rounding and one to the output type
    v = R.values(*ref, kind, cols, 1.0 if g is None else g)
    for out in DTYPES:
        assert torch.equal(F.dequantize_fp4(q, out), v.float().to(out))
    # columns past the matrix are zero in the layout
    assert int(q.codes.view(-1, rows, 16)[-(-cols // 32):].count_nonzero()) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_ties(dtype):
    """Every border of e2m1 times every e4m3 mantissa, exactly on the border and next to it on both sides."""
    F = fp4()
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda", dtype=torch.float64)
    rows = []
    for m in range(8):
        s = (1 + m / 8) * 2.0 ** 3
        row = torch.zeros(16, device="cuda", dtype=torch.float64)
        row[0] = 6 * s  # its block's maximum: the scale is s for g = 1
        row[1:8] = border * s
        row[8:15] = -border * s
        rows.append(row)
    x = torch.stack(rows).to(dtype)
    bits = {2: torch.int16, 4: torch.int32}[x.element_size()]
    near = []
    for step in (-1, 0, 1):
        y = (x.view(bits) + step).view(dtype)
        y[:, 0], y[:, 15] = x[:, 0], 0
        near.append(y)
    x = torch.cat(near)
    for g in (1.0, 0.25, 3.0, 0.7):
        gt = torch.tensor([g], device="cuda")
        assert_same_codes(F.quantize_fp4(x, "nvfp4", global_scale=gt), R.quantize(x, "nvfp4", gt), f"g={g}")
        assert_same_codes(F.quantize_fp4(x, "nvfp4", global_scale=g), R.quantize(x, "nvfp4", gt), f"g={g}")
    assert_same_codes(F.quantize_fp4(x, "mxfp4"), R.quantize(x, "mxfp4"))


def test_scale_borders():
    """Block maxima on and next to every border between two e4m3 scales."""
    F = fp4()
    t = R.e4m3_values("cuda")
    mid = ((t[1:] + t[:-1]) / 2 * 6).float()
    a = torch.cat([(mid.view(torch.int32) + d).view(torch.float32) for d in (-1, 0, 1)])
    x = torch.zeros(a.numel(), 16, device="cuda")
    x[:, 3] = a
    x[:, 5] = -a / 3
    for g in (1.0, 0.5, 0.3):
        gt = torch.tensor([g], device="cuda")
        assert_same_codes(F.quantize_fp4(x * g if g != 0.3 else x, "nvfp4", global_scale=gt),
                          R.quantize(x * g if g != 0.3 else x, "nvfp4", gt))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_extremes(kind, dtype):
    F = fp4()
    fi = torch.finfo(dtype)
    vals = [0.0, -0.0, fi.max, -fi.max, fi.smallest_normal, fi.smallest_normal / 4, 1.0, 3e-3]
    x = torch.zeros(len(vals) + 1, 64, device="cuda", dtype=dtype)
    for i, v in enumerate(vals):
        x[i, 5] = v
        x[i, 40:] = v / 3
    x[-1] = torch.linspace(-1, 1, 64).to(dtype)
    for g in ([1.0, 2.0 ** -100, 2.0 ** 100] if kind == "nvfp4" else [None]):
        gt = None if g is None else torch.tensor([g], device="cuda")
        q = F.quantize_fp4(x, kind, global_scale=gt)
        assert_same_codes(q, R.quantize(x, kind, 1.0 if g is None else gt), f"g={g}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_not_finite(kind, dtype):
    """A block with an infinity or a NaN stands for NaN; its neighbours are untouched."""
    F = fp4()
    x = rand(6, 256, dtype, 3, 0.5)
    x[0, 3], x[1, 40], x[2, 255], x[3, 128] = float("nan"), float("inf"), float("-inf"), float("nan")
    g = None if kind == "mxfp4" else torch.tensor([0.01], device="cuda")
    q = F.quantize_fp4(x, kind, global_scale=g)
    assert_same_codes(q, R.quantize(x, kind, 1.0 if g is None else g))
    v = F.dequantize_fp4(q, torch.float32)
    b = R.BLOCK[kind]
    want = torch.zeros(6, 256, dtype=torch.bool, device="cuda")
    for r, c in ((0, 3), (1, 40), (2, 255), (3, 128)):
        want[r, c // b * b: c // b * b + b] = True
    assert torch.equal(v.isnan(), want) and not v.isinf().any()
    if kind == "nvfp4":  # the maximum is taken over the finite values
        f = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).double().abs().max()
        assert torch.equal(F.fp4_global_scale(x), (f / 2688).float().reshape(1))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_strides_and_gather(kind, dtype):
    F = fp4()
    big = rand(70, 3 * 160 + 5, dtype, 5)
    g = g_of(kind, big)
    gr = 1.0 if g is None else g
    for x in (big[:, 160:320], big[::3, 1:200], big[5:6, 3:40], big[:, :32].t(), big[:1].expand(9, -1)[:, :48]):
        assert_same_codes(F.quantize_fp4(x, kind, global_scale=g), R.quantize(x, kind, gr))
    x = big[:, 8:200]
    idx = torch.tensor([3, 3, 69, 0, -1, 70, 1 << 30, -(1 << 31), 12], dtype=torch.int32, device="cuda")
    want = torch.zeros(9, 192, dtype=dtype, device="cuda")
    for i, j in enumerate(idx.tolist()):
        if 0 <= j < 70:
            want[i] = x[j]
    assert_same_codes(F.quantize_fp4(x, kind, global_scale=g, row_index=idx), R.quantize(want, kind, gr))
    assert F.quantize_fp4(x, kind, global_scale=g, row_index=idx[:0]).codes.numel() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_gather_from_no_rows(kind):
    """Every index is outside an x without rows: rows of zeros."""
    F = fp4()
    x = torch.empty(0, 200, device="cuda")
    idx = torch.tensor([0, -1, 5], dtype=torch.int32, device="cuda")
    for g in (None, 0.5) if kind == "nvfp4" else (None,):
        q = F.quantize_fp4(x, kind, global_scale=g, row_index=idx)
        assert (q.rows, q.cols) == (3, 200) and int(q.data.count_nonzero()) == 0
        assert torch.equal(F.dequantize_fp4(q, torch.float32), torch.zeros(3, 200, device="cuda"))
        q = F.quantize_fp4(x, kind, global_scale=g, row_index=idx[:0])
        assert q.rows == 0 and q.codes.numel() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 7), (5, 2048), (300, 1400), (77, 2319), (1, 9001)])
def test_global_scale(dtype, rows, cols):
    F = fp4()
    x = rand(rows, cols, dtype, 11)
    want = (x.double().abs().max() / 2688).float().reshape(1)  # 53 bits: rounding twice changes nothing
    assert torch.equal(F.fp4_global_scale(x), want)
    q = F.quantize_fp4(x)
    assert torch.equal(q.global_scale, want)
    assert_same_codes(q, R.quantize(x, "nvfp4", want))
    assert int(q.to_checkpoint()[1].max()) == 0x7E  # the largest block has the last scale
    for at in ((0, 0), (rows - 1, cols - 1), (rows // 2, cols // 2), (rows - 1, 0)):  # found wherever it is, any row pitch
        big = torch.zeros(rows, cols + 3, dtype=dtype, device="cuda")
        for y in (big[:, :cols], big[:, 1:cols + 1], torch.zeros(rows, cols, dtype=dtype, device="cuda")):
            y.zero_()
            y[at] = -42.0
            assert float(F.fp4_global_scale(y)) == float(torch.tensor(42 / 2688, dtype=torch.float32))
    zero = torch.zeros(rows, cols, dtype=dtype, device="cuda")
    assert float(F.fp4_global_scale(zero)) == 2.0 ** -100
    assert int(F.quantize_fp4(zero).codes.count_nonzero()) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 7), (5, 1024), (300, 700), (77, 1159), (2000, 1408)])
def test_global_scale_of_silu(dtype, rows, cols):
    """The largest product to the last bit, though most are only estimated; next to what is not finite, and where the
    gates are far below zero."""
    F = fp4()

    def want(gu):
        h = R.silu_mul(gu).float().abs()  # past float32 is infinite
        h = torch.where(torch.isfinite(h), h, torch.zeros_like(h)).max().double()
        return (h / 2688).float().clamp(min=2.0 ** -100).reshape(1)

    for seed in range(3):
        r = gen(seed)
        gu = (torch.randn(rows, 2 * cols, generator=r, device="cuda") * 2).to(dtype)
        assert torch.equal(F.fp4_global_scale(gu, silu_mul=True), want(gu))
        q = F.silu_mul_quantize_fp4(gu)
        assert torch.equal(q.global_scale, want(gu))
        assert_same_codes(q, R.quantize(R.silu_mul(gu), "nvfp4", want(gu)))
        many = gu.clone()
        many[:, cols:] = many[:, cols:].clamp(-1, 1)  # products near one another
        many[:, :cols] = many[:, :cols].clamp(max=1.0)
        assert torch.equal(F.fp4_global_scale(many, silu_mul=True), want(many))
        gu[0, 0], gu[rows - 1, 2 * cols - 1] = float("nan"), float("inf")
        assert torch.equal(F.fp4_global_scale(gu, silu_mul=True), want(gu))
    low = torch.full((rows, 2 * cols), -90.0, device="cuda", dtype=dtype)
    low[:, cols:] = 3e4
    low[rows // 2, 0] = -85.0
    assert torch.equal(F.fp4_global_scale(low, silu_mul=True), want(low))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 16), (3, 15), (9, 130), (64, 1408), (700, 768)])
def test_silu_mul_bits(kind, dtype, rows, cols):
    F = fp4()
    r = gen(rows + cols)
    gu = (torch.randn(rows, 2 * cols, generator=r, device="cuda") * 2).to(dtype)
    h = R.silu_mul(gu)
    g = g_of(kind, h)
    assert_same_codes(F.silu_mul_quantize_fp4(gu, kind, global_scale=g), R.quantize(h, kind, 1.0 if g is None else g))


@pytest.mark.parametrize("kind", KINDS)
def test_silu_mul_range(kind):
    """Gates far from zero on both sides, zeros, ties (up = 0), and what is not finite."""
    F = fp4()
    gate = torch.tensor([-300.0, -100, -89, -88, -85, -80, -60, -20, -1, 0, 1, 20, 88, 100, 300, 1e4], device="cuda")
    up = torch.tensor([0.0, 1, -1, 1e-3, 3e4, 1e20, -1e30, 1e35], device="cuda")
    rows = []
    for u in up:
        for c in range(0, 16, 4):
            rows.append(torch.cat((gate.roll(c), gate, gate[:4].repeat(8)[:32], u.repeat(64))))
    for gt in gate:
        rows.append(torch.cat((gt.repeat(64), up.repeat(8))))
    gu = torch.stack(rows)
    h = R.silu_mul(gu)
    over = h.abs() > torch.finfo(torch.float32).max  # past float32: not finite
    href = torch.where(over, torch.full_like(h, float("inf")), h)
    for g in ([1.0, 2.0 ** -90] if kind == "nvfp4" else [None]):
        gt = None if g is None else torch.tensor([g], device="cuda")
        assert_same_codes(F.silu_mul_quantize_fp4(gu, kind, global_scale=gt), R.quantize(href, kind, 1.0 if g is None else gt))
    gu[0, 3], gu[1, 70], gu[2, 5] = float("nan"), float("inf"), float("inf")
    gt = None if kind == "mxfp4" else torch.tensor([1.0], device="cuda")
    s = F.silu_mul_quantize_fp4(gu, kind, global_scale=gt).to_checkpoint()[1]
    nan = 127 if kind == "nvfp4" else 255
    b = R.BLOCK[kind]
    assert s[0, 3 // b] == nan and s[1, 6 // b] == nan and s[2, 5 // b] == nan


# Several rows a warp from rows * ceil(cols / 512) >= 18944 on: as many rows as leave the last CTA a few, for rows on
# 32-byte and on 16-byte boundaries (columns or padding), and on any other (one row a warp, many CTAs).
MANY = [(6401, 1408), (6403, 1392), (18977, 500), (6405, 1399)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", MANY)
def test_many_rows(kind, dtype, rows, cols):
    """Bit for bit, the quantiser and the way back, at the boundaries of x's rows that the kernels tell apart."""
    F = fp4()
    per16 = 16 // dtype.itemsize
    for pad, lo in ((-cols % (2 * per16), 0), (-cols % (2 * per16) + per16, per16), (0, 0)):
        big = rand(rows, cols + pad + lo, dtype, rows)
        x = big[:, lo:lo + cols]
        finite = torch.where(torch.isfinite(x), x, torch.zeros_like(x))  # (some float16 values are past its end)
        g = g_of(kind, finite, pow2=lo > 0)
        gr = 1.0 if g is None else g
        q = F.quantize_fp4(x, kind, global_scale=g)
        ref = R.quantize(x, kind, gr)
        assert_same_codes(q, ref, f"pad {pad}")
        v = R.values(*ref, kind, cols, gr).float().to(dtype)
        assert torch.allclose(F.dequantize_fp4(q, dtype), v, rtol=0, atol=0, equal_nan=True)
        assert int(v.isnan().sum()) <= 10 * R.BLOCK[kind]
        if kind == "nvfp4":
            assert torch.equal(F.fp4_global_scale(x), (finite.double().abs().max() / 2688).float().reshape(1))
        idx = torch.randint(-3, rows + 3, (rows,), generator=gen(cols), device="cuda", dtype=torch.int32)
        inside = (idx >= 0) & (idx < rows)
        want = torch.where(inside[:, None], x[idx.clamp(0, rows - 1).long()], torch.zeros((), dtype=dtype, device="cuda"))
        assert_same_codes(F.quantize_fp4(x, kind, global_scale=g, row_index=idx), R.quantize(want, kind, gr), "gathered")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", MANY)
def test_silu_mul_many_rows(kind, dtype, rows, cols):
    """The same of the SiLU form, with gates that only the float64 redo holds in the last rows and here and there."""
    F = fp4()
    per16 = 16 // dtype.itemsize
    r = gen(rows)
    for pad, lo in ((-2 * cols % (2 * per16), 0), (-2 * cols % (2 * per16) + per16, per16)):
        big = (torch.randn(rows, 2 * cols + pad + lo, generator=r, device="cuda") * 2).to(dtype)
        gu = big[:, lo:lo + 2 * cols]
        far = torch.rand(rows, cols, generator=r, device="cuda") < 0.002
        far[-20:] |= torch.rand(20, cols, generator=r, device="cuda") < 0.3
        far[-1] = True
        gate, up = gu[:, :cols], gu[:, cols:]
        gate.copy_(torch.where(far, -60 - 40 * torch.rand(rows, cols, generator=r, device="cuda"), gate.float()))
        up.copy_(torch.where(far, up.float() * 3e3, up.float()))
        h = R.silu_mul(gu)
        g = g_of(kind, h, pow2=lo > 0)
        gr = 1.0 if g is None else g
        q = F.silu_mul_quantize_fp4(gu, kind, global_scale=g)
        assert_same_codes(q, R.quantize(h, kind, gr), f"pad {pad}")
        assert torch.equal(F.dequantize_fp4(q), F.dequantize_fp4(F.silu_mul_quantize_fp4(gu.contiguous(), kind, global_scale=g)))
        if kind == "nvfp4":
            assert torch.equal(F.fp4_global_scale(gu, silu_mul=True), (h.abs().max().float().double() / 2688).float().reshape(1))
            tiny = torch.tensor([2.0 ** -100], device="cuda")  # the far gates' products are the ones that have digits
            assert_same_codes(F.silu_mul_quantize_fp4(gu[-40:], kind, global_scale=tiny), R.quantize(h[-40:], kind, tiny))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_silu_mul_smallest_gates(kind, dtype):
    """Gates below float32's normal range times an up that brings the product back into it."""
    F = fp4()
    r = gen(17)
    least = {torch.bfloat16: -133, torch.float32: -149}[dtype]  # gates are small multiples of the smallest one
    k = torch.randint(1, 200, (40, 64), generator=r, device="cuda").double()
    k[:20] = torch.randint(1, 9, (20, 64), generator=r, device="cuda").double()
    gate = k * 2.0 ** least * torch.where(torch.rand(40, 64, generator=r, device="cuda") < 0.5, -1, 1)
    up = torch.exp2(torch.randint(95, 126, (40, 1), generator=r, device="cuda").double()).expand(-1, 64)
    gu = torch.cat((gate, up), 1).to(dtype)
    h = R.silu_mul(gu)
    assert (gu[:20, :64].float().abs() < 2.0 ** -126).all() and gu[:, :64].count_nonzero() == gu[:, :64].numel()
    for row in (slice(0, 40), slice(3, 4)):
        gr = None if kind == "mxfp4" else (h[row].abs().max() / 2688).float().clamp(min=2.0 ** -100).reshape(1)
        assert_same_codes(F.silu_mul_quantize_fp4(gu[row], kind, global_scale=gr), R.quantize(h[row], kind, 1.0 if gr is None else gr))
        if kind == "nvfp4":
            assert torch.equal(F.fp4_global_scale(gu[row], silu_mul=True), gr)


@pytest.mark.parametrize("kind", KINDS)
def test_silu_mul_end_of_range(kind):
    """Products next to the largest float32: a block is finite exactly where its products round to finite float32."""
    F = fp4()
    top = torch.finfo(torch.float32).max
    r = gen(23)
    cols = 64
    gate = 1.5 + 12 * torch.rand(1800, 1, generator=r, device="cuda").expand(-1, cols)
    silu = gate.double() / (1 + torch.exp(-gate.double()))
    at = (torch.rand(1800, 1, generator=r, device="cuda").double() - 0.5) * 2.0 ** -15  # within 2^-16 of the end, both sides,
    at[::3] *= 2.0 ** -7  # and within a few of its last digits
    at[1::3] *= 2.0 ** -8
    up = (top / silu * (1 + at)).clamp(max=top).float()
    up[:, 1::2] *= 0.3
    up[1200:, cols - 1] = float("nan")
    gu = torch.cat((gate, up), 1)
    h = R.silu_mul(gu)
    href = torch.where(torch.isinf(h.float()), torch.full_like(h, float("inf")), h)
    finite = torch.isfinite(href[:1200]).all(1)
    assert 200 < int(finite.sum()) < 1000
    g = None if kind == "mxfp4" else torch.tensor([2.0 ** 100], device="cuda")
    assert_same_codes(F.silu_mul_quantize_fp4(gu, kind, global_scale=g), R.quantize(href, kind, 1.0 if g is None else g))
    one = gu[:1200][finite]
    if kind == "nvfp4":
        want = (R.silu_mul(one).abs().max().float().double() / 2688).float().reshape(1)
        assert torch.equal(F.fp4_global_scale(one.contiguous(), silu_mul=True), want)


@pytest.mark.parametrize("low,high", [(-80, -60), (-64, -46), (-80, -1)])
def test_global_scale_of_near_products(low, high):
    """Products within float32's rounding of one another, at gates whose estimates are least exact: the largest is found."""
    F = fp4()
    rows, cols = 400, 512
    r = gen(-low)
    for seed in range(4):
        gate = (low + (high - low) * torch.rand(rows, cols, generator=r, device="cuda")).clamp(min=-80.0)
        silu = R.silu_mul(torch.cat((gate, torch.ones_like(gate)), 1))
        near = 1 + torch.rand(rows, cols, generator=r, device="cuda").double() * 2.0 ** (-17 - seed)
        gu = torch.cat((gate, (1000 * near / silu).float()), 1)
        h = R.silu_mul(gu)
        want = (h.abs().max().float().double() / 2688).float().reshape(1)
        assert torch.equal(F.fp4_global_scale(gu, silu_mul=True), want)
        at = int(h.abs().argmax())  # that value alone among the smallest of the others
        gu[:, cols:] *= 1 - 2.0 ** -18
        gu.view(-1)[at // cols * 2 * cols + cols + at % cols] /= 1 - 2.0 ** -18
        want = (R.silu_mul(gu).abs().max().float().double() / 2688).float().reshape(1)
        assert torch.equal(F.fp4_global_scale(gu, silu_mul=True), want)


@pytest.mark.parametrize("kind", KINDS)
def test_checkpoint_round_trip(kind):
    F = fp4()
    for rows, cols in ((1, 5), (130, 200), (33, 1408)):
        x = rand(rows, cols, torch.bfloat16, 9)
        g = g_of(kind, x)
        ref = R.quantize(x, kind, 1.0 if g is None else g)
        codes, scales = ref
        m = F.FP4Matrix.from_checkpoint(kind, codes, scales, cols, global_scale=g)
        assert_same_codes(m, ref)
        q = F.quantize_fp4(x, kind, global_scale=g)
        assert torch.equal(m.codes, q.codes) and torch.equal(m.scales, q.scales)
        if kind == "nvfp4":
            f8 = F.FP4Matrix.from_checkpoint(kind, codes, scales.view(torch.float8_e4m3fn), cols, global_scale=g)
            assert torch.equal(f8.scales, q.scales)


@pytest.mark.parametrize("rows", [0, 1, 3])
def test_odd_gate_width_refused(rows):
    F = fp4()
    x = torch.ones(rows, 33, device="cuda")
    with pytest.raises(ValueError, match="even width"):
        F.fp4_global_scale(x, silu_mul=True)
    with pytest.raises(ValueError, match="even width"):
        F.silu_mul_quantize_fp4(x)
