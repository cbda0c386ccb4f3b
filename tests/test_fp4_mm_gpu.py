"""Products of 4-bit microscaled matrices on the GPU against float64."""
import pytest
import torch

from tests import _fp4_ref as R

pytestmark = pytest.mark.gpu

KINDS = ["nvfp4", "mxfp4"]


def fp4():
    from block_lut_b200 import fp4 as F
    return F


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def operand(rows, cols, kind, seed, scale=1.0):
    """Quantised rows and the float64 values they stand for."""
    F = fp4()
    x = torch.randn(rows, cols, generator=gen(seed), device="cuda") * scale
    q = F.quantize_fp4(x, kind)
    g = 1.0 if q.global_scale is None else q.global_scale
    return q, R.values(*R.quantize(x, kind, g), kind, cols, g)


def check(y, x, w, what=""):
    ref, tol = R.product_bound(x, w, y.dtype)
    d = (y.double() - ref).abs()
    assert torch.isfinite(y).all() and (d <= tol).all(), f"{what}: off by up to {float((d / tol).max()):.3g} of the bound"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(1, 128, 128), (1, 1, 16), (5, 130, 200), (16, 128, 64), (17, 256, 1408), (32, 640, 2048),
                                   (33, 129, 256), (64, 384, 500), (65, 128, 2048), (128, 200, 1024), (129, 300, 640),
                                   (192, 128, 128), (193, 257, 2048), (500, 640, 1408), (1000, 1000, 1000)])
def test_matmul(kind, m, n, k):
    F = fp4()
    xq, x = operand(m, k, kind, 1)
    wq, w = operand(n, k, kind, 2, 0.05)
    W = F.FP4Weight.from_quantized(wq)
    y = F.fp4_matmul(xq, W, out_dtype=torch.float32)
    check(y, x, w, "float32")
    check(F.fp4_matmul(xq, W), x, w, "bfloat16")
    check(F.fp4_matmul(xq, W, out_dtype=torch.float16), x, w, "float16")
    assert torch.equal(y, F.fp4_matmul(xq, W, out_dtype=torch.float32))  # the same bits every time
    F.fp4_check_status()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(3, 60000, 640), (40, 50000, 384), (100, 30000, 1408), (700, 20000, 640), (1500, 9000, 2048)])
def test_matmul_many_items(kind, m, n, k):
    """More tiles than CTAs run at once: the rings and the accumulator go on from one to the next."""
    F = fp4()
    xq, x = operand(m, k, kind, 1)
    wq, w = operand(n, k, kind, 2, 0.05)
    W = F.FP4Weight.from_quantized(wq)
    check(F.fp4_matmul(xq, W, out_dtype=torch.float32), x, w, "float32")
    check(F.fp4_matmul(xq, W), x, w, "bfloat16")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(40000, 264, 64), (40000, 328, 128), (5000, 5000, 128), (30000, 1160, 256), (50000, 296, 128)])
def test_cut_row_tile_after_a_full_one(kind, dtype, m, n, k):
    """CTAs go from full row tiles, which leave by bulk stores, to one that the matrix cuts, which does not, with next to
    no K between: no row of y holds another tile's values.  (The row tiles' number does not divide the CTAs', so that
    a CTA meets both kinds.)  The float32 output takes neither way, and rounding it is the
    16-bit output to the bit (one accumulator, one factor)."""
    F = fp4()
    xq, x = operand(m, k, kind, 1)
    wq, w = operand(n, k, kind, 2, 0.05)
    W = F.FP4Weight.from_quantized(wq)
    wide = F.fp4_matmul(xq, W, out_dtype=torch.float32)
    check(wide, x, w, "float32")
    want = wide.to(dtype)
    outs = [torch.empty(m, n, device="cuda", dtype=dtype) for _ in range(8)]
    for out in outs:  # back to back: the stores meet a busy memory
        out.fill_(7.0)
        F.fp4_matmul(xq, W, out=out)
    for out in outs:
        assert torch.equal(out, want)
    F.fp4_check_status()


@pytest.mark.parametrize("n", [264, 1160])
def test_cut_row_tile_after_a_full_one_grouped(n):
    """The same for runs of rows, some of which end inside a stretch."""
    F = fp4()
    counts = [9000, 0, 8001, 1, 7777, 4095]
    m, xq, x, W, ws, off = runs_case(len(counts), counts, 3, 5, n, 128, "nvfp4")
    wide = F.fp4_grouped_matmul(xq, W, off, out=torch.full((m, n), 7.0, device="cuda"))
    at = off.tolist()
    for e in range(len(counts)):
        if counts[e]:
            check(wide[at[e]:at[e + 1]], x[at[e]:at[e + 1]], ws[e], f"run {e}")
    outs = [torch.full((m, n), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(8)]
    for out in outs:
        F.fp4_grouped_matmul(xq, W, off, out=out)
    for out in outs:
        assert torch.equal(out, wide.bfloat16())
    F.fp4_check_status()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,k", [(200, 500), (1000, 4096), (60000, 1408), (129, 33)])
def test_linear_is_quantize_then_matmul(kind, dtype, n, k):
    """Bit for bit, on both sides of the number of rows that the product quantises itself, for any row pitch."""
    F = fp4()
    W = F.FP4Weight.quantize(torch.randn(n, k, generator=gen(5), device="cuda") * 0.05, kind)
    for scale in (None, 0.0025) if kind == "nvfp4" else (None,):
        lin = F.FP4Linear(W, scale)
        for m in (1, 2, 7, 8, 9, 33):
            big = torch.randn(m, k + 11, generator=gen(m), device="cuda").to(dtype)
            for x in (big[:, :k].contiguous(), big[:, 3:3 + k]):
                want = F.fp4_matmul(F.quantize_fp4(x, kind, scale), W, out_dtype=dtype)
                assert torch.equal(lin(x), want), (m, scale)
    F.fp4_check_status()


@pytest.mark.parametrize("kind", KINDS)
def test_every_element_has_its_place(kind):
    """One nonzero weight column and one nonzero token at a time would take long; a rank-one pattern of distinct
    powers shows a swapped row, token, block or half just as well."""
    F = fp4()
    for m, n, k in ((40, 256, 384), (200, 128, 256)):
        xv = torch.zeros(m, k, device="cuda")
        for t in range(m):
            xv[t, (t * 37) % k] = [1.0, 2.0, 3.0, 4.0, 6.0][t % 5]
        wv = torch.zeros(n, k, device="cuda")
        r = torch.arange(n, device="cuda")[:, None]
        c = torch.arange(k, device="cuda")[None]
        lv = R.LEVELS.float().cuda()
        wv = lv[(r * 5 + c * 3) % 8] * torch.where((r + c) % 3 == 0, -1.0, 1.0) * torch.exp2(((r + c // 32) % 5).float())
        g = None if kind == "mxfp4" else 1.0
        xq, wq = F.quantize_fp4(xv, kind, global_scale=g), F.quantize_fp4(wv, kind, global_scale=g)
        x = F.dequantize_fp4(xq, torch.float32).double()
        w = F.dequantize_fp4(wq, torch.float32).double()
        y = F.fp4_matmul(xq, F.FP4Weight.from_quantized(wq), out_dtype=torch.float32)
        assert torch.equal(y.double(), x @ w.T)  # single products: exact


@pytest.mark.parametrize("kind", KINDS)
def test_not_finite_blocks_stay_in_their_rows(kind):
    F = fp4()
    x = torch.randn(40, 256, generator=gen(0), device="cuda")
    w = torch.randn(200, 256, generator=gen(1), device="cuda")
    clean = F.fp4_matmul(F.quantize_fp4(x, kind, 0.01 if kind == "nvfp4" else None),
                         F.FP4Weight.from_quantized(F.quantize_fp4(w, kind, 0.01 if kind == "nvfp4" else None)))
    x[7, 100], w[130, 5] = float("nan"), float("inf")
    y = F.fp4_matmul(F.quantize_fp4(x, kind, 0.01 if kind == "nvfp4" else None),
                     F.FP4Weight.from_quantized(F.quantize_fp4(w, kind, 0.01 if kind == "nvfp4" else None)))
    bad = torch.zeros(40, 200, dtype=torch.bool, device="cuda")
    bad[7], bad[:, 130] = True, True
    assert torch.equal(y.isnan(), bad)
    assert torch.equal(y[~bad], clean[~bad])


@pytest.mark.parametrize("kind", KINDS)
def test_output_pitch(kind):
    F = fp4()
    xq, x = operand(21, 256, kind, 1)
    wq, w = operand(200, 256, kind, 2)
    W = F.FP4Weight.from_quantized(wq)
    big = torch.full((21, 333), 7.0, device="cuda", dtype=torch.bfloat16)
    y = F.fp4_matmul(xq, W, out=big[:, 11:211])
    assert y.data_ptr() == big[:, 11:211].data_ptr()
    check(y, x, w)
    assert (big[:, :11] == 7).all() and (big[:, 211:] == 7).all()
    assert F.fp4_matmul(F.quantize_fp4(torch.zeros(0, 256, device="cuda"), kind), W).shape == (0, 200)
    # many tokens, on 16-byte boundaries and off them, the columns beside y as they were
    xq, x = operand(333, 256, kind, 3)
    for n, lo in ((200, 8), (200, 11), (129, 16), (40, 24)):
        W2 = F.FP4Weight.from_quantized(operand(n, 256, kind, 4)[0])
        w2 = operand(n, 256, kind, 4)[1]
        big = torch.full((333 + 40, 304), 7.0, device="cuda", dtype=torch.float16)
        check(F.fp4_matmul(xq, W2, out=big[:333, lo:lo + n]), x, w2)
        assert (big[:333, :lo] == 7).all() and (big[:333, lo + n:] == 7).all() and (big[333:] == 7).all(), (n, lo)


def runs_case(E, counts, lead, tail, n, k, kind, seed=0):
    F = fp4()
    m = lead + sum(counts) + tail
    xq, x = operand(m, k, kind, seed)
    ws = [operand(n, k, kind, 100 + seed * 1000 + e, 0.05 * (1 + e % 3)) for e in range(E)]
    off = torch.tensor([lead] + [lead + sum(counts[: e + 1]) for e in range(E)], dtype=torch.int32, device="cuda")
    return m, xq, x, F.FP4Weight.from_quantized([q for q, _ in ws]), [w for _, w in ws], off


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("counts,lead,tail", [
    ([1], 0, 0), ([0, 0, 5, 0], 0, 0), ([3, 0, 1, 40, 0, 33], 2, 7), ([0] * 7, 0, 9), ([200, 1, 0, 65], 1, 1),
    ([1] * 8 + [0] * 120, 0, 0), ([2, 0, 1] * 43, 3, 64), ([300, 300, 5], 0, 0), ([0, 700, 0, 1], 17, 0), ([90, 100, 80], 0, 3)])
def test_grouped(kind, counts, lead, tail):
    F = fp4()
    n, k = 200, 384
    E = len(counts)
    m, xq, x, W, ws, off = runs_case(E, counts, lead, tail, n, k, kind)
    for dt in (torch.bfloat16, torch.float32):
        out = torch.full((m, n), 7.0, device="cuda", dtype=dt)
        y = F.fp4_grouped_matmul(xq, W, off, out=out)
        assert y.data_ptr() == out.data_ptr()
        at = off.tolist()
        for e in range(E):
            if at[e + 1] > at[e]:
                check(y[at[e]:at[e + 1]], x[at[e]:at[e + 1]], ws[e], f"run {e}")
        assert (y[:lead] == 7).all() and (y[m - tail:] == 7).all()
    again = F.fp4_grouped_matmul(xq, W, off, out=torch.full_like(out, 7.0))
    assert torch.equal(again, out)
    F.fp4_check_status()


def test_grouped_many_experts():
    F = fp4()
    counts = [(e * 7) % 4 for e in range(300)]
    m, xq, x, W, ws, off = runs_case(300, counts, 0, 0, 128, 128, "nvfp4")
    y = F.fp4_grouped_matmul(xq, W, off, out_dtype=torch.float32)
    at = off.tolist()
    for e in range(300):
        if counts[e]:
            check(y[at[e]:at[e + 1]], x[at[e]:at[e + 1]], ws[e], f"run {e}")


def test_offsets_stay_in_the_buffer():
    """Offsets outside [0, rows] are clamped by the kernel: no row outside the buffers is read or written."""
    F = fp4()
    m, xq, x, W, ws, off = runs_case(3, [4, 5, 6], 0, 0, 130, 128, "nvfp4")
    guard = torch.full((m + 8, 130), 7.0, device="cuda", dtype=torch.float32)
    out = guard[4:4 + m]
    F.fp4_grouped_matmul(xq, W, torch.tensor([-5, 4, 9, 1 << 30], dtype=torch.int32, device="cuda"), out=out)
    check(out[:4], x[:4], ws[0])
    check(out[4:9], x[4:9], ws[1])
    check(out[9:], x[9:], ws[2])
    assert (guard[:4] == 7).all() and (guard[4 + m:] == 7).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear(kind, dtype):
    F = fp4()
    w = torch.randn(300, 500, generator=gen(5), device="cuda") * 0.05
    W = F.FP4Weight.quantize(w, kind)
    gw = 1.0 if W.global_scale is None else W.global_scale
    wv = R.values(*R.quantize(w, kind, gw), kind, 500, gw)
    for shape, scale in (((3, 500), None), ((2, 5, 500), 0.004), ((500,), None), ((0, 500), None), ((1, 1, 500), 0.01)):
        x = torch.randn(*shape, generator=gen(6), device="cuda").to(dtype)
        lin = F.FP4Linear(W, None if kind == "mxfp4" else scale)
        y = lin(x)
        assert y.shape == x.shape[:-1] + (300,) and y.dtype == dtype
        x2 = x.reshape(-1, 500)
        if x2.shape[0]:
            g = 1.0 if kind == "mxfp4" else torch.tensor([scale], device="cuda") if scale else (x2.double().abs().max() / 2688).float()
            check(y.reshape(-1, 300), R.values(*R.quantize(x2, kind, g), kind, 500, g), wv)
            out = torch.empty_like(y)
            assert lin(x, out=out) is out and torch.equal(out, y)


def test_streams_and_graphs():
    """A side stream, and two captured graphs replayed beside each other and beside eager calls: no shared state."""
    F = fp4()
    xq, x = operand(24, 2048, "nvfp4", 1)
    wq, w = operand(640, 2048, "nvfp4", 2)
    W = F.FP4Weight.from_quantized(wq)
    want = F.fp4_matmul(xq, W)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    y = F.fp4_matmul(xq, W, stream=s)
    s.synchronize()
    assert torch.equal(y, want)
    lin = F.FP4Linear(W)
    xs = [torch.randn(24, 2048, generator=gen(i), device="cuda").bfloat16() for i in range(2)]
    want = [lin(v) for v in xs]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for v in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(lin(v))
        graphs.append(g)
    side = torch.cuda.Stream()
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        eager = lin(xs[0])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])


@pytest.mark.parametrize("kind", KINDS)
def test_expert_layer(kind):
    """The operators as a layer of routed experts runs them: gather + quantise, gate/up, SiLU + quantise, down.  Each
    step is held to its own bound on the rows that the step before it gave."""
    F = fp4()
    T, k, E, H, I = 37, 2, 6, 256, 200
    r = gen(8)
    x = torch.randn(T, H, generator=r, device="cuda").bfloat16()
    ids = torch.rand(T, E, generator=r, device="cuda").topk(k).indices
    order = ids.flatten().argsort(stable=True)
    off = torch.searchsorted(ids.flatten()[order].contiguous(), torch.arange(E + 1, device="cuda")).int()
    w13 = torch.randn(E, 2 * I, H, generator=r, device="cuda") * 0.08
    w2 = torch.randn(E, H, I, generator=r, device="cuda") * 0.08
    W13, W2 = F.FP4Weight.quantize(w13, kind), F.FP4Weight.quantize(w2, kind)
    tok = (order // k).int()
    xq = F.quantize_fp4(x, kind, row_index=tok)
    gx = 1.0 if kind == "mxfp4" else xq.global_scale
    gu = F.fp4_grouped_matmul(xq, W13, off)
    hq = F.silu_mul_quantize_fp4(gu, kind)
    y = F.fp4_grouped_matmul(hq, W2, off, out_dtype=torch.float32)
    xv = R.values(*R.quantize(x[tok.long()], kind, gx), kind, H, gx)
    gh = 1.0 if kind == "mxfp4" else hq.global_scale
    hv = R.values(*R.quantize(R.silu_mul(gu), kind, gh), kind, I, gh)
    at = off.tolist()
    for e in range(E):
        lo, hi = at[e], at[e + 1]
        if hi == lo:
            continue
        g13 = 1.0 if kind == "mxfp4" else W13.global_scale[e]
        g2 = 1.0 if kind == "mxfp4" else W2.global_scale[e]
        check(gu[lo:hi], xv[lo:hi], R.values(*R.quantize(w13[e], kind, g13), kind, H, g13))
        check(y[lo:hi], hv[lo:hi], R.values(*R.quantize(w2[e], kind, g2), kind, I, g2))
    # the layer's result is near the unquantised one: 4-bit noise, not a wrong expert
    full = torch.zeros(T * k, H, dtype=torch.float64, device="cuda")
    for i, (t, e) in enumerate(zip(tok.tolist(), ids.flatten()[order].tolist())):
        full[i] = R.silu_mul(x[t].double() @ w13[e].double().T) @ w2[e].double().T
    # noise of a 4-bit value: at most a quarter of it between two levels, in rms about 0.1; five such factors
    # (x twice through the product of gate and up, two weights, h) stay below 0.5 of the result in the 2-norm
    assert float((y.double() - full).norm() / full.norm()) < 0.5


def test_linear_follows_its_attributes():
    """A scale or a weight assigned after construction is the one used, on both sides of the rows that the product
    quantises itself; the old tensors stay alive here, so that a stale pointer gives a wrong result and no fault."""
    F = fp4()
    ws = [torch.randn(n, 384, generator=gen(n), device="cuda") * 0.05 for n in (256, 256, 200)]
    Ws = [F.FP4Weight.quantize(w) for w in ws]
    mx = F.FP4Weight.quantize(ws[2], "mxfp4")
    scales = [None, torch.tensor([0.002], device="cuda"), torch.tensor([0.003], device="cuda"), 0.004]
    lin = F.FP4Linear(Ws[0], scales[1])
    for m in (3, 20):
        x = torch.randn(m, 384, generator=gen(m), device="cuda").bfloat16()

        def want(W, scale):
            return F.fp4_matmul(F.quantize_fp4(x, W.kind, scale), W)

        for W in Ws:
            lin.weight = W
            assert (lin.rows, lin.cols) == (W.rows, W.cols)
            for scale in scales + scales[::-1]:
                lin.act_scale = scale
                assert torch.equal(lin(x), want(W, scale)), (m, W.rows, scale)
        lin.act_scale = scales[1]
        lin.weight = mx
        with pytest.raises(ValueError, match="no global scale"):
            lin(x)
        lin.act_scale = None
        assert torch.equal(lin(x), want(mx, None))
        lin.weight = own = F.FP4Weight.from_quantized(F.quantize_fp4(ws[0]))  # a weight whose parts are replaced
        assert torch.equal(lin(x), want(Ws[0], None))
        old = own.tiled, own.global_scale
        own.tiled, own.global_scale = Ws[1].tiled.clone(), Ws[1].global_scale * 2
        assert torch.equal(lin(x), want(own, None)) and not torch.equal(lin(x), want(Ws[0], None))
        own.tiled, own.global_scale = old
    with pytest.raises(ValueError, match="single"):
        lin.weight = F.FP4Weight.from_quantized([F.quantize_fp4(w) for w in ws[:2]])
    with pytest.raises(ValueError, match="act_scale"):
        lin.act_scale = -1.0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens", [1, 50])
def test_routed_layer_in_a_graph(kind, tokens):
    """From the router to the weighted sum without a word from the host: captured, and replayed on other tokens."""
    from block_lut_b200 import router
    F = fp4()
    k, E, H, I = 3, 12, 256, 136
    r = gen(4)
    w_router = torch.randn(E, H, generator=r, device="cuda").bfloat16()
    W13 = F.FP4Weight.quantize(torch.randn(E, 2 * I, H, generator=r, device="cuda") * 0.08, kind)
    W2 = F.FP4Weight.quantize(torch.randn(E, H, I, generator=r, device="cuda") * 0.08, kind)
    every = torch.arange(E + 1, dtype=torch.int32, device="cuda")

    def layer(x):
        ids, weights, _ = router(x, w_router, k)
        expert_of_row, order = ids.flatten().sort(stable=True)
        offsets = torch.searchsorted(expert_of_row, every, out_int32=True)
        xq = F.quantize_fp4(x, kind, row_index=(order // k).int())
        h = F.silu_mul_quantize_fp4(F.fp4_grouped_matmul(xq, W13, offsets), kind)
        y = F.fp4_grouped_matmul(h, W2, offsets)
        rows = torch.empty_like(y).index_copy_(0, order, y)
        return (rows.view(len(x), k, -1) * weights[..., None]).sum(1), ids, weights, xq.global_scale

    x = torch.randn(tokens, H, generator=r, device="cuda").bfloat16()
    for _ in range(2):
        layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(x)
    for seed in range(3):
        x.copy_(torch.randn(tokens, H, generator=gen(seed), device="cuda"))
        graph.replay()
        want = layer(x)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        out, ids, weights, g = want
        xq = F.quantize_fp4(x, kind, global_scale=g)
        per = []  # every expert on every row, without sorting: rows and matrix scales are the same
        for e in range(E):
            off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
            off[e + 1:] = tokens
            per.append(F.fp4_grouped_matmul(xq, W13, off))
        gu = torch.stack(per)[ids.long(), torch.arange(tokens, device="cuda")[:, None]]  # [tokens, k, 2 I]
        h = F.silu_mul_quantize_fp4(gu.view(tokens * k, -1), kind)
        per = []
        for e in range(E):
            off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
            off[e + 1:] = tokens * k
            per.append(F.fp4_grouped_matmul(h, W2, off).view(tokens, k, H))
        y = torch.stack(per).gather(0, ids.long()[None, :, :, None].expand(1, -1, -1, H))[0]
        assert torch.equal(out, (y * weights[..., None]).sum(1))  # a row's product does not depend on its run


def test_linear_in_place():
    """An output that overlaps the input is written from the input as it was."""
    F = fp4()
    W = F.FP4Weight.quantize(torch.randn(1024, 1024, generator=gen(1), device="cuda") * 0.05)
    lin = F.FP4Linear(W, 0.002)
    for m in (3, 20):
        x = torch.randn(m, 1024, generator=gen(2), device="cuda").bfloat16()
        want = lin(x)
        assert lin(x, out=x) is x and torch.equal(x, want)


@pytest.mark.parametrize("m", [3, 20])
def test_linear_beside_its_input(m):
    """An output next to the input in one array is no overlap; one that reaches into it is written from it as it was."""
    F = fp4()
    W = F.FP4Weight.quantize(torch.randn(640, 512, generator=gen(1), device="cuda") * 0.05)
    lin = F.FP4Linear(W, 0.002)
    for x_at, y_at, fresh in ((0, 512, False), (640, 0, False), (0, 500, True), (600, 0, True), (128, 128, True)):
        arena = torch.randn(2 * m, 1152, generator=gen(2), device="cuda").bfloat16()
        x, out = arena[:m, x_at:x_at + 512], arena[:m, y_at:y_at + 640]
        want, rest = lin(x), arena.clone()
        rest[:m, y_at:y_at + 640] = want
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        lin(x, out=out)
        after = torch.cuda.memory_stats()["allocation.all.allocated"]
        assert torch.equal(arena, rest), (x_at, y_at)
        assert after - before == fresh + (m > 8)  # the copy of x, and the workspace
        below = arena[m:, 64:64 + 640]  # rows behind x's
        x.normal_(generator=gen(3))
        want = lin(x)
        assert torch.equal(lin(x, out=below), want)


@pytest.mark.parametrize("m,n,k", [(3, 256, 2048), (40, 256, 2048), (500, 3000, 2048)])
def test_a_wait_that_runs_out_is_reported(m, n, k):
    """With a limit of 1 ns the kernels' waits give up: the call ends, the status says so once, the next call is right."""
    from block_lut_b200 import _lib
    F = fp4()
    xq, x = operand(m, k, "nvfp4", 1)
    wq, w = operand(n, k, "nvfp4", 2)
    W = F.FP4Weight.from_quantized(wq)
    F.fp4_check_status()
    _lib.lib().blut_debug_set_wait_limit(1)
    try:
        F.fp4_matmul(xq, W)
        torch.cuda.synchronize()
    finally:
        _lib.lib().blut_debug_set_wait_limit(0)
    with pytest.raises(RuntimeError, match="timed out"):
        F.fp4_check_status()
    F.fp4_check_status()
    check(F.fp4_matmul(xq, W), x, w)
    F.fp4_check_status()


@pytest.mark.parametrize("kind", KINDS)
def test_no_global_scale_is_one(kind):
    """A matrix without a global scale stands for g = 1 as an operand, on the way back, and as a weight."""
    F = fp4()
    for rows in (20, 130):
        xq, x = operand(rows, 200, kind, 1)
        bare = F.FP4Matrix(kind, rows, 200, xq.data)
        one = F.FP4Matrix(kind, rows, 200, xq.data, None if kind == "mxfp4" else torch.ones(1, device="cuda"))
        assert torch.equal(F.dequantize_fp4(bare), F.dequantize_fp4(one))
        W, W1 = F.FP4Weight.from_quantized(bare), F.FP4Weight.from_quantized(one)
        assert torch.equal(F.fp4_matmul(bare, W), F.fp4_matmul(one, W1))
        E, E1 = F.FP4Weight.from_quantized([bare, xq]), F.FP4Weight.from_quantized([one, xq])
        off = torch.tensor([0, 7, rows], dtype=torch.int32, device="cuda")
        assert torch.equal(F.fp4_grouped_matmul(bare, E, off), F.fp4_grouped_matmul(one, E1, off))


@pytest.mark.parametrize("kind", KINDS)
def test_operands_made_by_hand(kind):
    """What a kernel would read past its end or on the host is refused before a launch; buffers that hold enough work."""
    F = fp4()
    xq, x = operand(20, 200, kind, 1)
    wq, w = operand(130, 200, kind, 2)
    W = F.FP4Weight.from_quantized(wq)
    lin = F.FP4Linear(W)
    xf = torch.randn(20, 200, generator=gen(3), device="cuda")
    want, wl = F.fp4_matmul(xq, W), lin(xf)

    def calls(q, v):
        own = F.FP4Linear(v)
        return ((q, lambda: F.dequantize_fp4(q)), (q, q.to_checkpoint), (q, lambda: F.FP4Weight.from_quantized(q)),
                (q, lambda: F.fp4_matmul(q, W)), (v, lambda: F.fp4_matmul(xq, v)), (v, lambda: own(xf)), (v, lambda: own(xf[:2])))

    def like(q=xq, v=W, **kw):
        return (F.FP4Matrix(q.kind, q.rows, q.cols, kw.get("data", q.data), kw.get("gx", q.global_scale)),
                F.FP4Weight(v.kind, v.rows, v.cols, None, kw.get("tiled", v.tiled), v.stride, kw.get("gw", v.global_scale)))

    for kw in (dict(data=xq.data[:-16], tiled=W.tiled[:-16]), dict(data=xq.data.cpu(), tiled=W.tiled.cpu()),
               dict(data=xq.data.view(torch.int8), tiled=W.tiled.view(torch.int8)), dict(gx=torch.ones(1), gw=torch.ones(1)),
               dict(gx=torch.ones(2, device="cuda"), gw=torch.ones(2, device="cuda"))):
        for _, call in calls(*like(**kw)):
            with pytest.raises(ValueError):
                call()
    more, moreW = like(data=torch.cat((xq.data, xq.data)), tiled=torch.cat((W.tiled, W.tiled)))
    assert torch.equal(F.fp4_matmul(more, moreW), want)
    one, oneW = like(gx=None, gw=None)  # no scale: 1
    if kind == "nvfp4":
        gg = xq.global_scale * W.global_scale
        assert torch.equal(F.fp4_matmul(one, oneW, out_dtype=torch.float32) * gg, F.fp4_matmul(xq, W, out_dtype=torch.float32))
        lin.act_scale = torch.ones(1, device="cuda")
        lin._act_scale = torch.ones(1)
        for rows in (2, 20):
            with pytest.raises(ValueError, match="act_scale"):
                lin(xf[:rows])
        lin.act_scale = None
    assert torch.equal(lin(xf), wl) and torch.equal(F.fp4_matmul(xq, W), want)


def test_first_call_in_a_capture():
    """A process whose first product is captured: the launch set-up works inside a capture."""
    import subprocess
    import sys
    code = (
        "import torch\n"
        "from block_lut_b200 import fp4 as F\n"
        "w = torch.randn(256, 512, device='cuda'); x = torch.randn(20, 512, device='cuda').bfloat16()\n"
        "W = F.FP4Weight.quantize(w); lin = F.FP4Linear(W)\n"
        "torch.cuda.synchronize(); g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g): y = lin(x); z = lin(x[:2])\n"
        "g.replay(); torch.cuda.synchronize()\n"
        "assert torch.equal(y, lin(x)) and torch.equal(z, lin(x[:2]))\n"
        "print('captured')\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("kind", KINDS)
def test_large_codes_offset(kind):
    """Rows and columns whose codes pass 2^31 bytes, and an output past 2^31 elements: spot checks on both ends."""
    F = fp4()
    m, k, n = 1 << 21, 2304, 1152
    x = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16)
    at = [0, 1, m // 2, m - 2, m - 1]
    x[at] = torch.randn(5, k, generator=gen(1), device="cuda").bfloat16()
    g = None if kind == "mxfp4" else 0.002
    xq = F.quantize_fp4(x, kind, g)
    wq, w = operand(n, k, kind, 2, 0.05)
    y = F.fp4_matmul(xq, F.FP4Weight.from_quantized(wq))
    gv = 1.0 if g is None else torch.tensor([g], device="cuda")
    check(y[at], R.values(*R.quantize(x[at], kind, gv), kind, k, gv), w)
    assert int(y.count_nonzero()) <= 5 * n and m * n > 2 ** 31 and xq.codes.numel() > 2 ** 31
    d = F.dequantize_fp4(xq)
    assert torch.equal(d[at], R.values(*R.quantize(x[at], kind, gv), kind, k, gv).float().bfloat16())


def test_beside_other_work():
    """Products of every variant, and a LUT matmul, on streams of their own at the same time: they share the SMs' tensor
    memory and shared memory, and nothing else."""
    from block_lut_b200.formats import LUTFormat, encode
    from block_lut_b200.linear import LUTLinear
    F = fp4()
    jobs = []
    for m, n, k, kind in ((1, 2048, 2048, "nvfp4"), (12, 1024, 4096, "mxfp4"), (60, 512, 2048, "nvfp4"), (100, 256, 2048, "mxfp4"),
                          (700, 3000, 1024, "nvfp4"), (300, 20000, 512, "nvfp4")):
        xq, _ = operand(m, k, kind, m)
        W = F.FP4Weight.from_quantized(operand(n, k, kind, n)[0])
        jobs.append(lambda xq=xq, W=W: F.fp4_matmul(xq, W))
    m, xq, x, WE, ws, off = runs_case(5, [3, 0, 40, 7, 100], 1, 2, 640, 1024, "nvfp4")
    jobs.append(lambda: F.fp4_grouped_matmul(xq, WE, off, out=torch.zeros(m, 640, device="cuda", dtype=torch.float16)))
    lin = F.FP4Linear(F.FP4Weight.quantize(torch.randn(1024, 1024, generator=gen(3), device="cuda")))
    xs = torch.randn(20, 1024, generator=gen(4), device="cuda").bfloat16()
    jobs.append(lambda: lin(xs))
    lut = LUTLinear(encode(torch.randn(1024, 1024, generator=gen(5), device="cuda"), LUTFormat("b", 4, 64)))
    xl = torch.randn(64, 1024, generator=gen(6), device="cuda").half()
    jobs.append(lambda: lut(xl))
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(20):
        got = []
        for j, s in zip(jobs, streams):
            with torch.cuda.stream(s):
                for _ in range(3):
                    out = j()
                got.append(out)
        torch.cuda.synchronize()
        for i, (g, w) in enumerate(zip(got, want)):
            assert torch.equal(g, w), i
    F.fp4_check_status()
