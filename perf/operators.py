"""The 4-bit microscaled operators: plain forms, inputs and cases.

Formulas.  A row of K values is cut into blocks of B columns (nvfp4: B = 16, mxfp4: B = 32; the last block may be
short).  A block has one 8-bit scale s and a 4-bit value q per column, q in +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} (e2m1), and
stands for q * s * g, with one float32 g per matrix:

    nvfp4   s = e4m3(max|x| / (6 g)), round to nearest even, at most 448; g is given or max|x| of the matrix / 2688
    mxfp4   s = 2^(floor(log2 max|x|) - 2), within 2^-127 .. 2^127; g = 1
    q = e2m1(x / (s g)), round to nearest even, at most 6 in magnitude (q = 0 where s = 0)

"quantize" is that map and its way back, "silu" the same map of silu(gate) * up, "linear" quantises the rows x and
multiplies them with a matrix held in 4 bits, y = x W^T, and "grouped" multiplies runs of quantised rows, one run for
each expert, with that expert's matrix.  What is rounded to 4 or 8 bits goes by the exact quotient, so the plain form
forms quotients in 64 bits: a 32-bit quotient can fall on the wrong side of a border.
"""
import math

import torch

own = False

BLOCK = {"nvfp4": 16, "mxfp4": 32}
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------ plain form --
def _to_step(v, step):
    return torch.round(v / step) * step  # torch.round: ties to even


def _e4m3(v):
    """Non-negative float64 values rounded to e4m3."""
    _, e = torch.frexp(v)
    return _to_step(v, torch.exp2((e - 1).clamp(min=-6).double() - 3)).clamp(max=448.0)


def _e2m1(v):
    """Non-negative float64 values rounded to e2m1."""
    _, e = torch.frexp(v)
    return _to_step(v, torch.exp2((e - 1).clamp(0, 2).double() - 1)).clamp(max=6.0)


def _global_scale(x):
    top = x.abs().amax().float()
    return (top / torch.full_like(top, 2688.0)).clamp(min=2.0 ** -100)  # by a number, torch multiplies with its reciprocal


def _quantize(v, kind, g):
    """float64 rows -> (q, s) as float64: signed e2m1 values [rows, blocks, B] and scales [rows, blocks, 1]."""
    rows, cols = v.shape
    b = BLOCK[kind]
    v = torch.nn.functional.pad(v, (0, -cols % b)).reshape(rows, -1, b)
    a = v.abs().amax(-1, keepdim=True)
    if kind == "nvfp4":
        s = _e4m3(a / (6.0 * g.double()))
    else:
        _, e = torch.frexp(a)
        s = torch.exp2((e - 3).clamp(-127, 127).double())
        s = torch.where(a > 0, s, torch.full_like(s, 2.0 ** -127))
    q = torch.where(s > 0, _e2m1(v.abs() / (s * g.double())), 0.0)
    return torch.copysign(q, v), s


def _values(q, s, g, cols):
    """float64 q, s -> the float64 values they stand for, [rows, cols]."""
    return (q * (s * g.double())).flatten(1)[:, :cols]


def _codes(q):
    """Signed e2m1 values [rows, blocks, B] -> bytes [rows, blocks * B / 2], the even column in the low half."""
    code = torch.bucketize(q.abs().float(), torch.tensor(LEVELS, device=q.device)).to(torch.uint8)
    code = (code | (torch.signbit(q).to(torch.uint8) << 3)).flatten(1)
    return code[:, 0::2] | (code[:, 1::2] << 4)


def _scale_bytes(s, kind):
    s = s.squeeze(-1)
    return s.float().to(torch.float8_e4m3fn).view(torch.uint8) if kind == "nvfp4" else (torch.log2(s) + 127).to(torch.uint8)


def _dense(codes, scales, kind, cols):
    """Checkpoint bytes [..., rows, *] -> float32 q * s [..., rows, cols] (exact), without the matrix' g."""
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    q = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).flatten(-2)
    s = scales.view(torch.float8_e4m3fn).float() if kind == "nvfp4" else torch.exp2(scales.float() - 127)
    return (q.unflatten(-1, (-1, BLOCK[kind])) * s[..., None]).flatten(-2)[..., :cols]


def _silu_mul(gu):
    gate, up = gu.double().chunk(2, -1)
    return gate / (1 + torch.exp(-gate)) * up


def _padded(offsets, longest):
    """Row of each (expert, place) and whether that place has one."""
    row = offsets[:-1, None].long() + torch.arange(longest, device=offsets.device)
    return row, row < offsets[1:, None]


# ----------------------------------------------------------------------- inputs --
def _activations(gen, rows, cols, dtype):
    """Rows of unit scale whose columns differ in scale, as after a norm with its weight."""
    channel = torch.exp(0.5 * torch.randn(cols, generator=gen, device="cuda"))
    return (torch.randn(rows, cols, generator=gen, device="cuda") * channel).to(dtype)


def _checkpoint(gen, rows, cols, kind, std):
    """One matrix as a checkpoint holds it: bytes of codes and scales, and g."""
    w = torch.randn(rows, cols, generator=gen, device="cuda") * std
    g = _global_scale(w) if kind == "nvfp4" else torch.ones((), device="cuda")
    q, s = _quantize(w.double(), kind, g)
    return _codes(q), _scale_bytes(s, kind), g


def _stack(gen, n, rows, cols, kind, std):
    one = [_checkpoint(gen, rows, cols, kind, std) for _ in range(n)]
    return [torch.stack(t) for t in zip(*one)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, kind, dtype = case["op"], case["kind"], DTYPE[case["dtype"]]
    st = {"case": case}
    if op in ("quantize", "silu"):
        rows, cols = case["rows"], case["cols"]
        st["x"] = _activations(gen, rows, cols if op == "quantize" else 2 * cols, dtype)
        st["g"] = None
        if kind == "nvfp4" and not case["dynamic"]:  # the layer's calibrated scale: a little above this batch's own
            top = st["x"] if op == "quantize" else _silu_mul(st["x"])
            st["g"] = _global_scale(top).reshape(1) * 1.07
    elif op == "linear":
        m, rows, cols = case["m"], case["rows"], case["cols"]
        st["x"] = _activations(gen, m, cols, dtype)
        st["g"] = _global_scale(st["x"]).reshape(1) * 1.07 if kind == "nvfp4" else None
        st["w"] = _checkpoint(gen, rows, cols, kind, cols ** -0.5)
        if own:
            from block_lut_b200 import fp4
            codes, scales, g = st["w"]
            st["layer"] = fp4.FP4Linear(fp4.FP4Weight.from_checkpoint(kind, codes, scales, cols, global_scale=g if kind == "nvfp4" else None),
                                        act_scale=st["g"])
    else:
        tokens, k, n, rows, cols = case["tokens"], case["top_k"], case["experts"], case["rows"], case["cols"]
        logits = torch.randn(tokens, n, generator=gen, device="cuda") + 0.4 * torch.randn(n, generator=gen, device="cuda")
        counts = torch.bincount(logits.topk(k).indices.flatten(), minlength=n)
        m = tokens * k + case["spare"]  # the buffer's rows: those past the last run stay as they are
        st["offsets"] = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).int()
        st["longest"] = int(counts.max())
        x = _activations(gen, m, cols, torch.float32)
        st["gx"] = _global_scale(x).reshape(1) if kind == "nvfp4" else None
        q, s = _quantize(x.double(), kind, st["gx"] if kind == "nvfp4" else torch.ones((), device="cuda"))
        st["xq"] = _codes(q), _scale_bytes(s, kind)
        del x, q, s
        st["w"] = _stack(gen, n, rows, cols, kind, cols ** -0.5)
        st["out"] = torch.zeros(m, rows, dtype=dtype, device="cuda")
        if own:
            from block_lut_b200 import fp4
            codes, scales, g = st["w"]
            st["weight"] = fp4.FP4Weight.from_checkpoint(kind, codes, scales, cols, global_scale=g if kind == "nvfp4" else None)
            st["rows"] = fp4.FP4Matrix.from_checkpoint(kind, *st["xq"], cols, global_scale=st["gx"])
    return st


# ----------------------------------------------------------------------- passes --
def _one(st):
    return torch.ones((), device="cuda")


def run(st):
    case = st["case"]
    op, kind, dtype = case["op"], case["kind"], DTYPE[case["dtype"]]
    if own:
        from block_lut_b200 import fp4
        if op == "quantize":
            return fp4.dequantize_fp4(fp4.quantize_fp4(st["x"], kind, global_scale=st["g"]), dtype)
        if op == "silu":
            return fp4.dequantize_fp4(fp4.silu_mul_quantize_fp4(st["x"], kind, global_scale=st["g"]), dtype)
        if op == "linear":
            return st["layer"](st["x"])
        return fp4.fp4_grouped_matmul(st["rows"], st["weight"], st["offsets"], out=st["out"])
    if op in ("quantize", "silu"):
        v = st["x"].double() if op == "quantize" else _silu_mul(st["x"])
        g = (_global_scale(v) if st["g"] is None else st["g"]) if kind == "nvfp4" else _one(st)
        return _values(*_quantize(v, kind, g), g, case["cols"]).to(dtype)
    if op == "linear":
        codes, scales, gw = st["w"]
        gx = st["g"] if kind == "nvfp4" else _one(st)
        q, s = _quantize(st["x"].double(), kind, gx)
        x = (q * s).flatten(1)[:, : case["cols"]].float()  # exact: 2 + 4 bits
        return (x @ _dense(codes, scales, kind, case["cols"]).T * (gx * gw)).to(dtype)
    codes, scales, gw = st["w"]
    row, there = _padded(st["offsets"], st["longest"])
    x = _dense(*st["xq"], kind, case["cols"])[row.clamp(max=st["out"].shape[0] - 1)]
    y = torch.bmm(x, _dense(codes, scales, kind, case["cols"]).mT)
    if kind == "nvfp4":
        y = y * (st["gx"] * gw)[:, None, None]
    st["out"][row[there]] = y[there].to(dtype)
    return st["out"]


# ------------------------------------------------------------- definition, 64 bits --
def _exact_levels(v, kind, g):
    """What the rows' 4-bit form stands for, by search among the borders between neighbours: float64 [rows, cols]."""
    rows, cols = v.shape
    b = BLOCK[kind]
    nb = -(-cols // b)
    full = torch.zeros(rows, nb * b, dtype=torch.float64, device=v.device)
    full[:, :cols] = v
    a = full.view(rows, nb, b).abs().max(-1).values

    def nearest(t, table):
        """Index of the entry of an ascending table next to t >= 0; a tie goes to the even index."""
        mid = (table[1:] + table[:-1]) / 2
        lo, hi = torch.searchsorted(mid, t, right=False), torch.searchsorted(mid, t, right=True)
        return torch.where(lo % 2 == 0, lo, hi)

    if kind == "nvfp4":
        byte = torch.arange(127, dtype=torch.uint8, device=v.device)
        table = byte.view(torch.float8_e4m3fn).double()
        s = table[nearest(a / (6 * g.double()), table)]
    else:
        powers = torch.ldexp(torch.ones(255, dtype=torch.float64, device=v.device), torch.arange(-127, 128, device=v.device))
        s = powers[(torch.searchsorted(powers * 4, a, right=True) - 1).clamp(min=0)]
    unit = (s * g.double())[..., None]
    table = torch.tensor(LEVELS, dtype=torch.float64, device=v.device)
    t = full.view(rows, nb, b)
    q = table[nearest((t.abs() / unit.clamp(min=1e-300)).contiguous(), table)] * torch.sign(t)
    return (q * unit).reshape(rows, -1)[:, :cols]


def _exact_dense(codes, scales, kind, cols):
    q = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
    table = torch.tensor(LEVELS, dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        c = (codes >> (4 * half)) & 15
        q[..., half::2] = table[(c & 7).long()] * (1 - 2 * (c >> 3).double())
    if kind == "nvfp4":
        s = scales.view(torch.float8_e4m3fn).double()
    else:
        s = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 127)
    return (q * s.repeat_interleave(BLOCK[kind], -1))[..., :cols]


def exact(case, seed):
    st = prepare(case, seed)
    op, kind, cols = case["op"], case["kind"], case["cols"]
    one = torch.ones((), dtype=torch.float64, device="cuda")
    if op in ("quantize", "silu"):
        v = st["x"].double()
        if op == "silu":
            v = v[:, cols:] * v[:, :cols] * torch.special.expit(v[:, :cols])
        g = one
        if kind == "nvfp4":
            g = st["g"] if st["g"] is not None else (v.abs().max().float().double() / 2688).float().clamp(min=2.0 ** -100)
        return _exact_levels(v, kind, g)
    if op == "linear":
        codes, scales, gw = st["w"]
        x = _exact_levels(st["x"].double(), kind, st["g"] if kind == "nvfp4" else one)
        return x @ _exact_dense(codes, scales, kind, cols).T * gw.double()
    codes, scales, gw = st["w"]
    at = st["offsets"].tolist()
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
    gx = st["gx"].double() if kind == "nvfp4" else one
    for e in range(case["experts"]):
        lo, hi = at[e], at[e + 1]
        if hi > lo:
            w = _exact_dense(codes[e], scales[e], kind, cols) * gw[e].double()
            out[lo:hi] = _exact_dense(st["xq"][0][lo:hi], st["xq"][1][lo:hi], kind, cols) @ w.T * gx
    return out


# ------------------------------------------------------------------------- cases --
def _packed(n, cols, kind):
    return n * (cols / 2 + -(-cols // BLOCK[kind]))


def work(case):
    op, kind, size = case["op"], case["kind"], DTYPE[case["dtype"]].itemsize
    cols, rows = case["cols"], case["rows"]
    if op in ("quantize", "silu"):
        wide = 2 if op == "silu" else 1
        return {"bytes": rows * cols * (wide + 1) * size + 2 * _packed(rows, cols, kind), "flops": 0}
    if op == "linear":
        m = case["m"]
        return {"bytes": m * cols * size + _packed(rows, cols, kind) + m * rows * size, "flops": 2 * m * rows * cols}
    n, m = case["experts"], case["tokens"] * case["top_k"]
    active = n * (1 - (1 - case["top_k"] / n) ** case["tokens"])  # experts that get a row
    return {"bytes": _packed(m, cols, kind) + active * _packed(rows, cols, kind) + m * rows * size, "flops": 2 * m * rows * cols}


def _rows_case(name, op, kind, dtype, rows, cols, dynamic=False):
    return {"name": name, "op": op, "kind": kind, "dtype": dtype, "rows": rows, "cols": cols, "dynamic": dynamic}


def _linear_case(name, kind, dtype, m, rows, cols):
    return {"name": name, "op": "linear", "kind": kind, "dtype": dtype, "m": m, "rows": rows, "cols": cols}


def _grouped_case(name, kind, dtype, tokens, top_k, experts, rows, cols, spare=0):
    return {"name": name, "op": "grouped", "kind": kind, "dtype": dtype, "tokens": tokens, "top_k": top_k, "experts": experts,
            "rows": rows, "cols": cols, "spare": spare}


def listed():
    return [
        # a decode batch of 32 hidden rows, a scale from calibration
        _rows_case("quantize decode", "quantize", "nvfp4", "bf16", 32, 2048),
        # an uneven prefill chunk, rows that are no multiple of a tile and end inside a block
        _rows_case("quantize ragged", "quantize", "mxfp4", "fp16", 1999, 1400),
        # the prefill of 8 x 4096 tokens, its scale taken from the batch itself
        _rows_case("quantize prefill", "quantize", "nvfp4", "bf16", 32768, 2048, True),
        # the routed rows of a decode batch of 32 tokens with 4 experts each, between the experts' two products
        _rows_case("silu decode", "silu", "nvfp4", "bf16", 128, 1408),
        # those of a prefill of 8 x 4096 tokens with 6 experts each
        _rows_case("silu prefill", "silu", "mxfp4", "fp16", 196608, 1408),
        # one token through the down projection of a shared expert
        _linear_case("linear one token", "nvfp4", "bf16", 1, 2048, 5632),
        # a decode batch through its gate and up projections
        _linear_case("linear decode", "nvfp4", "bf16", 32, 11264, 2048),
        # an uneven prefill chunk, an output width and a depth that are no multiples of a tile
        _linear_case("linear ragged", "mxfp4", "fp16", 1999, 5000, 1400),
        # the prefill of 8 x 4096 tokens
        _linear_case("linear prefill", "nvfp4", "bf16", 32768, 11264, 2048),
        # one token, 8 of 128 experts, gate and up
        _grouped_case("grouped one token", "mxfp4", "bf16", 1, 8, 128, 1536, 2048),
        # a decode batch of 32 tokens, 4 of 60 experts, in a buffer with room for more rows
        _grouped_case("grouped decode", "nvfp4", "bf16", 32, 4, 60, 2816, 2048, 64),
        # the prefill of 8 x 4096 tokens, 6 of 64 experts
        _grouped_case("grouped prefill", "nvfp4", "fp16", 32768, 6, 64, 2816, 2048),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("quantize", "silu", "linear", "grouped"))
    kind, dtype = rng.choice(tuple(BLOCK)), rng.choice(("bf16", "fp16"))
    cols = spread(192, 8192)
    cols = rng.choice((cols, cols, -(-cols // 128) * 128, -(-cols // 128) * 128, -(-cols // 16) * 16))
    if op in ("quantize", "silu"):
        if op == "quantize" and rng.random() < 0.2:
            dtype = "fp32"  # weights of a checkpoint
        return _unnamed(_rows_case("", op, kind, dtype, spread(1, 6e7 / cols), cols, rng.random() < 0.3))
    rows = spread(128, 12288)
    if rng.random() < 0.6:
        rows = -(-rows // 128) * 128
    if op == "linear":
        return _unnamed(_linear_case("", kind, dtype, spread(1, min(32768, 7e11 / (rows * cols))), rows, cols))
    experts = rng.choice((8, 16, 60, 64, 128))
    top_k = rng.randint(1, 8)
    rows = max(128, min(rows, int(3.6e8 / (experts * cols))))
    tokens = spread(1, max(1.0, min(32768, 1e12 / (rows * cols * top_k))))
    return _unnamed(_grouped_case("", kind, dtype, tokens, top_k, experts, rows, cols, rng.choice((0, 0, 37))))


def _unnamed(case):
    del case["name"]
    return case
