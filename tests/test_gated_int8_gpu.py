"""GPU: the gated feed-forward block and the 8-bit products against the same formulas in 64 bits.

Tolerances, fixed before the first run.  A rounding to type t is off by at most eps(t) / 2 relative to
the value (bf16 2^-8, fp16 2^-11, TF32 operands 2^-11); one element is a sum of many such errors of
either sign.
  forward   h is rounded once and y once: |error| <= e * (|h| . |Wd|^T + |y|), e = eps / 2, every error at
            its bound and of one sign.  The FP32 sums add K * 2^-24 of the sums of magnitudes, far less.
  backward  the same with the rounded operands of each product: dgate, dup and h.
  8 bits    the integer sum is exact; scales, bias and activation are a few FP32 roundings and the output
            one of its own type.
FP32 operands are multiplied as TF32 (both operands of each product rounded: 2 e with e = 2^-10 covers
truncation), a bound on the sums of magnitudes again.
"""
import pytest

pytestmark = pytest.mark.gpu

EPS2 = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -10}
ACTS = ("ACT_SILU", "ACT_GELU", "ACT_RELU", "ACT_NONE")


def _act64(v, act):
    import torch
    if act == "ACT_SILU":
        p = torch.sigmoid(v)
        return v * p, p * (1 + v * (1 - p))
    if act == "ACT_GELU":
        c = torch.special.ndtr(v)
        return v * c, c + v * torch.exp(-0.5 * v * v) * 0.3989422804014327
    if act == "ACT_RELU":
        return v.clamp(min=0), (v > 0).double()
    return v, torch.ones_like(v)


def _ffn_inputs(rows, d, f, dtype, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(getattr(torch, dtype))
    return t(rows, d), t(f, d, std=d ** -0.5), t(f, d, std=d ** -0.5), t(d, f, std=f ** -0.5), t(rows, d, std=0.1)


def _close(got, want, bound, what):
    import torch
    assert got.shape == want.shape, what
    g = got.double()
    assert torch.isfinite(g).all(), what
    over = ((g - want).abs() - bound).max().item()
    assert over <= 0, f"{what}: {over} above the bound"
    if want.numel() > 64:
        rel = ((g - want).norm() / want.norm().clamp(min=1e-30)).item()
        # far below the bound at which every rounding has one sign; catches a lost tile or k-block
        assert rel <= 4 * EPS2[str(got.dtype).split(".")[1]], f"{what}: relative error {rel}"


# one row, below / at / above a tile, odd sizes (rows that are no multiple of 16 bytes), a K split
SHAPES = [(1, 64, 64), (1, 256, 1024), (2, 129, 65), (17, 72, 264), (33, 1, 1), (64, 256, 512), (127, 200, 328),
          (256, 128, 256), (257, 264, 130), (300, 511, 1023), (513, 1024, 640), (1000, 96, 2050), (40, 2048, 4096)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,d,f", SHAPES)
def test_forward_matches_64_bits(gpu, rows, d, f, dtype):
    import torch
    act = ACTS[(rows + d + f) % 4]
    x, wg, wu, wd, _ = _ffn_inputs(rows, d, f, dtype, seed=rows + d)
    y, gate, up = gpu.gated_ffn_forward(x, wg, wu, wd, act=getattr(gpu, act), return_pre=True)
    plain = gpu.gated_ffn_forward(x, wg, wu, wd, act=getattr(gpu, act))
    torch.cuda.synchronize()
    assert torch.equal(y, plain)
    e = EPS2[dtype]
    tf = 2 * e if dtype == "float32" else 0.0           # operands of the FP32 form are rounded too
    X, G, U, D = x.double(), wg.double(), wu.double(), wd.double()
    g64, u64 = X @ G.t(), X @ U.t()
    mag_g, mag_u = X.abs() @ G.abs().t(), X.abs() @ U.abs().t()
    small = (d + 8) * 2.0 ** -24
    _close(gate, g64, e * g64.abs() + (tf + small) * mag_g + 1e-7, "gate")
    _close(up, u64, e * u64.abs() + (tf + small) * mag_u + 1e-7, "up")
    a, da = _act64(g64, act)
    h = a * u64
    # |act'| <= 1.13 for all four
    dh = 1.13 * (tf + small) * mag_g * u64.abs() + (tf + small) * mag_u * a.abs() + (e + 2.0 ** -20) * h.abs() + 1e-7
    want = h @ D.t()
    bound = dh @ D.abs().t() + (tf + (f + 8) * 2.0 ** -24) * (h.abs() @ D.abs().t()) + e * want.abs() + 1e-6
    _close(y, want, 1.01 * bound, "y")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,d,f", SHAPES)
def test_backward_matches_64_bits(gpu, rows, d, f, dtype):
    import torch
    act = ACTS[(rows + d + f) % 4]
    x, wg, wu, wd, dy = _ffn_inputs(rows, d, f, dtype, seed=rows + 7 * d)
    gate = (x.double() @ wg.double().t()).to(x.dtype)
    up = (x.double() @ wu.double().t()).to(x.dtype)
    got = gpu.gated_ffn_backward(dy, x, gate, up, wg, wu, wd, act=getattr(gpu, act))
    again = gpu.gated_ffn_backward(dy, x, gate, up, wg, wu, wd, act=getattr(gpu, act))
    torch.cuda.synchronize()
    for p, q in zip(got, again):
        assert torch.equal(p, q)
    e = EPS2[dtype]
    tf = 2 * e if dtype == "float32" else 0.0
    X, G, U, D, DY = (t.double() for t in (x, wg, wu, wd, dy))
    a, da = _act64(gate.double(), act)
    u = up.double()
    dh = DY @ D
    r = tf + (d + 16) * 2.0 ** -24
    ddh = r * (DY.abs() @ D.abs())                       # error of dh before the epilogue
    dg, du, h = dh * u * da, dh * a, a * u
    near = e + 2.0 ** -18                                # operand rounding and the epilogue's own arithmetic
    floor = 1e-7 if dtype == "float16" else 0.0          # fp16 below 2^-14 rounds in absolute steps of 2^-24
    edg = ddh * (u * da).abs() + near * dg.abs() + 2.0 ** -18 * (dh * u).abs() + floor
    edu = ddh * a.abs() + near * du.abs() + 2.0 ** -18 * dh.abs() + floor
    eh = near * h.abs() + 2.0 ** -18 * u.abs() + floor
    k = (max(rows, f) * 2 + 16) * 2.0 ** -24 + tf
    want = (dg @ G + du @ U, dg.t() @ X, du.t() @ X, DY.t() @ h)
    bound = (edg @ G.abs() + edu @ U.abs() + k * (dg.abs() @ G.abs() + du.abs() @ U.abs()),
             edg.t() @ X.abs() + k * (dg.abs().t() @ X.abs()),
             edu.t() @ X.abs() + k * (du.abs().t() @ X.abs()),
             DY.abs().t() @ eh + k * (DY.abs().t() @ h.abs()))
    for name, g, w, b in zip(("dx", "dw_gate", "dw_up", "dw_down"), got, want, bound):
        _close(g, w, 1.01 * b + e * w.abs() + floor, name)


# deep first products (the gradient's main loop covers its epilogue): odd widths, a K that ends inside a
# k-block, tiles past the last row and column, several tiles per CTA; same inputs and bounds as above
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,d,f", [(1, 1600, 130), (130, 1537, 517), (257, 1536, 1024), (700, 2056, 4100),
                                      (2050, 1664, 3001)])
def test_backward_of_deep_products_matches_64_bits(gpu, rows, d, f, dtype):
    test_backward_matches_64_bits(gpu, rows, d, f, dtype)


def _quant64(x):
    """The definition, in the 32-bit arithmetic it names."""
    import torch
    x = x.float()
    top = x.abs().amax(dim=-1, keepdim=True)
    finite = torch.isfinite(x).all(dim=-1, keepdim=True)
    live = finite & (top >= 2.0 ** -100)
    full = torch.full_like(top, 127.0)      # tensor by tensor: torch turns a scalar divisor into a product
    inv = torch.where(live, full / top, torch.zeros_like(top))
    q = torch.where(live, torch.round(x * inv), torch.zeros_like(x)).to(torch.int8)
    scale = torch.where(live, top / full, torch.zeros_like(top))
    scale = torch.where(finite, scale, torch.full_like(top, float("nan")))
    return q, scale[..., 0]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (9, 16), (5, 1000), (1, 4096), (33, 4104), (2, 8192), (3, 9001),
                                       (4, 20000)])
def test_quantize_rows_is_the_definition(gpu, rows, cols, dtype):
    import torch
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(rows + 6, cols + 8, generator=g, device="cuda")
    x *= torch.exp2(torch.randint(-6, 7, (rows + 6, 1), generator=g, device="cuda").float())
    x[rows] = 0.0
    x[rows + 1, cols // 2] = float("inf")
    x[rows + 2, cols - 1] = float("nan")
    x[rows + 3] = 2.0 ** -110
    x[rows + 4, :cols] = torch.where(torch.arange(cols, device="cuda") % 2 == 0, 1.0, -0.5)      # a tie
    x = x.to(getattr(torch, dtype))
    for view in (x[:, :cols], x[:, :cols].contiguous(), x[:, 1:cols + 1]):
        q, scale = gpu.quantize_rows(view)
        wq, ws = _quant64(view)
        torch.cuda.synchronize()
        assert torch.equal(q, wq)
        assert torch.equal(torch.nan_to_num(scale, nan=-1.0), torch.nan_to_num(ws, nan=-1.0))


INT8_SHAPES = [(1, 16, 16), (1, 4096, 512), (2, 1, 1), (7, 33, 65), (16, 128, 130), (57, 1024, 333), (64, 500, 64),
               (128, 256, 256), (255, 144, 513), (300, 1000, 768), (600, 2048, 200)]


@pytest.mark.parametrize("out", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("rows,k,n", INT8_SHAPES)
def test_int8_products(gpu, rows, k, n, gated, out):
    import torch
    act = ACTS[(rows + k + n) % 4]
    g = torch.Generator(device="cuda").manual_seed(rows + k + n)

    def q(*shape):
        return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)

    def s(*shape):
        return (torch.rand(*shape, generator=g, device="cuda") + 0.5) * (0.02 / k ** 0.5)
    x, w, w2, xs, ws, ws2 = q(rows, k), q(n, k), q(n, k), s(rows), s(n), s(n)
    xs *= 100.0
    bias = torch.randn(n, generator=g, device="cuda")
    dt = getattr(torch, out)
    e = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[out]
    p = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
    if gated:
        got = gpu.int8_gated_forward(x, xs, w, ws, w2, ws2, act=getattr(gpu, act), out_dtype=dt)
        p2 = (x.double() @ w2.double().t()) * xs.double()[:, None] * ws2.double()
        want = _act64(p, act)[0] * p2
        inner = (p.abs() + 1.0) * p2.abs()
    else:
        got = gpu.int8_linear_forward(x, xs, w, ws, bias=bias, act=getattr(gpu, act), out_dtype=dt)
        want = _act64(p + bias.double(), act)[0]
        inner = p.abs() + bias.double().abs() + 1.0
        none = gpu.int8_linear_forward(x, xs, w, ws, out_dtype=dt)
        assert ((none.double() - p).abs() <= (e + 2.0 ** -21) * p.abs() + 1e-7).all()
    torch.cuda.synchronize()
    # a handful of FP32 roundings (2^-24 each) and the special functions' few units
    bound = e * want.abs() + 2.0 ** -19 * inner + (6e-8 if out == "float16" else 0.0)
    assert ((got.double() - want).abs() <= bound).all()
