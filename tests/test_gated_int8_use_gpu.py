"""GPU: the gated feed-forward and 8-bit entries as programs use them: strided and unaligned operands, other
streams, captured graphs, every kernel form, neighbours of the outputs, refusals, a run of all together.

The reference is the same formula in 64 bits; tolerances as derived in test_gated_int8_gpu.py, here as a
relative error in the 2-norm: two roundings to the type in a row (hidden, output) are at most
2 * eps / 2 each in any element, so in the norm at most eps of the sums' magnitudes; 4 * eps / 2 covers
cancellation in random sums.
"""
import pytest

pytestmark = pytest.mark.gpu


def _rel(got, want):
    want = want.double()
    return ((got.double() - want).norm() / want.norm().clamp(min=1e-30)).item()


def _tol(t):
    import torch
    return 4 * torch.finfo(t.dtype).eps / 2 if t.dtype != torch.float32 else 4e-3


def _inputs(rows, d, f, dtype, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)

    def t(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)
    return t(rows, d), t(f, d, std=d ** -0.5), t(f, d, std=d ** -0.5), t(d, f, std=f ** -0.5)


def _block64(x, wg, wu, wd):
    import torch
    g = x.double() @ wg.double().t()
    return (g * torch.sigmoid(g) * (x.double() @ wu.double().t())) @ wd.double().t()


@pytest.mark.parametrize("rows,d,f", [(5, 72, 136), (140, 136, 264), (700, 136, 264)])
def test_strided_unaligned_and_batched_operands(gpu, rows, d, f):
    import torch
    x, wg, wu, wd = _inputs(rows, d, f, torch.bfloat16)
    want = _block64(x, wg, wu, wd)
    wide = torch.zeros(rows, d + 24, device="cuda", dtype=torch.bfloat16)
    for off in (0, 8, 3):                                    # aligned rows, an offset of 16 bytes, of 6
        view = wide[:, off:off + d]
        view.copy_(x)
        y, gate, up = gpu.gated_ffn_forward(view, wg, wu, wd, return_pre=True)
        assert y.is_contiguous() and _rel(y, want) <= _tol(y)
        dx = gpu.gated_ffn_backward(view, view, gate, up, wg, wu, wd)
        ref = gpu.gated_ffn_backward(x, x, gate, up, wg, wu, wd)
        for a, b in zip(dx, ref):
            assert torch.equal(a, b)
    fused = torch.cat([wg, wu])                              # halves of one matrix
    assert torch.equal(gpu.gated_ffn_forward(x, fused[:f], fused[f:], wd), gpu.gated_ffn_forward(x, wg, wu, wd))
    flat = torch.zeros(wg.numel() + 1, device="cuda", dtype=torch.bfloat16)
    odd = flat[1:].view(f, d)                                # a base off by one element
    odd.copy_(wg)
    assert torch.equal(gpu.gated_ffn_forward(x, odd, wu, wd), gpu.gated_ffn_forward(x, wg, wu, wd))
    if rows % 5 == 0:
        x3 = x.view(5, rows // 5, d)
        y3 = gpu.gated_ffn_forward(x3, wg, wu, wd)
        assert y3.shape == x3.shape and torch.equal(y3.view(rows, d), gpu.gated_ffn_forward(x, wg, wu, wd))
        q3, s3 = gpu.quantize_rows(x3)
        assert q3.shape == x3.shape and s3.shape == (5, rows // 5)
    y1 = gpu.gated_ffn_forward(x[0], wg, wu, wd)             # a single row without a batch dimension
    assert y1.shape == (d,) and _rel(y1, want[0]) <= _tol(y1)


@pytest.mark.parametrize("policy,block_n,split", [(3, 0, 0), (3, 0, 1), (3, 0, 2), (3, 0, 8), (4, 64, 1), (4, 128, 1),
                                                  (4, 256, 1), (4, 512, 1), (4, 128, 3), (4, 256, 5), (4, 512, 2)])
def test_every_kernel_form(gpu, policy, block_n, split):
    import torch
    rows, d, f = 330, 456, 1032
    for dtype in (torch.bfloat16, torch.float32):
        x, wg, wu, wd = _inputs(rows, d, f, dtype, seed=3)
        want = _block64(x, wg, wu, wd)
        plain = gpu.gated_ffn_forward(x, wg, wu, wd, return_pre=True)
        ref = gpu.gated_ffn_backward(x, x, plain[1], plain[2], wg, wu, wd)
        q, s = gpu.quantize_rows(x)
        wq, ws = gpu.quantize_rows(wg)
        uq, us = gpu.quantize_rows(wu)
        y8 = gpu.int8_linear_forward(q, s, wq, ws, out_dtype=dtype)
        h8 = gpu.int8_gated_forward(q, s, wq, ws, uq, us, out_dtype=dtype)
        gpu.set_policy(policy, block_n, split)
        try:
            y, gate, up = gpu.gated_ffn_forward(x, wg, wu, wd, return_pre=True)
            assert gpu.last_path()["path"] == (13 if policy == 3 else 12)
            grads = gpu.gated_ffn_backward(x, x, plain[1], plain[2], wg, wu, wd)
            assert _rel(y, want) <= _tol(y)
            assert _rel(gate, plain[1]) <= _tol(y) and _rel(up, plain[2]) <= _tol(y)
            for a, b in zip(grads, ref):
                assert _rel(a, b) <= _tol(a)
            # the integer sums are exact in every form
            assert torch.equal(gpu.int8_linear_forward(q, s, wq, ws, out_dtype=dtype), y8)
            assert torch.equal(gpu.int8_gated_forward(q, s, wq, ws, uq, us, out_dtype=dtype), h8)
        finally:
            gpu.set_policy(0, 0, 0)


def test_empty_batches(gpu):
    import torch
    x, wg, wu, wd = _inputs(0, 64, 128, torch.float16)
    y, gate, up = gpu.gated_ffn_forward(x, wg, wu, wd, return_pre=True)
    assert y.shape == (0, 64) and gate.shape == (0, 128)
    dx, dwg, dwu, dwd = gpu.gated_ffn_backward(x, x, gate, up, wg, wu, wd)
    assert dx.shape == (0, 64) and not dwg.any() and not dwu.any() and not dwd.any()
    q, s = gpu.quantize_rows(x)
    assert q.shape == (0, 64) and s.shape == (0,)
    wq, ws = gpu.quantize_rows(wg)
    assert gpu.int8_linear_forward(q, s, wq, ws).shape == (0, 128)


@pytest.mark.parametrize("rows", [3, 200, 400])
@pytest.mark.parametrize("d,f", [(64, 72), (65, 77)])
def test_neighbours_of_the_outputs_are_left_alone(gpu, rows, d, f):
    import torch
    x, wg, wu, wd = _inputs(rows, d, f, torch.bfloat16)
    pad = 512

    def guarded(n, dtype):
        return torch.full((n + 2 * pad,), 77, device="cuda", dtype=dtype)

    buf = guarded(rows * d, torch.bfloat16)
    y = gpu.gated_ffn_forward(x, wg, wu, wd, out=buf[pad:pad + rows * d].view(rows, d))
    assert _rel(y, _block64(x, wg, wu, wd)) <= _tol(y)
    assert (buf[:pad] == 77).all() and (buf[pad + rows * d:] == 77).all()
    q, s = gpu.quantize_rows(x)
    wq, ws = gpu.quantize_rows(wg)
    for dtype in (torch.float32, torch.float16):
        buf = guarded(rows * f, dtype)
        gpu.int8_linear_forward(q, s, wq, ws, out_dtype=dtype, out=buf[pad:pad + rows * f].view(rows, f))
        gpu.int8_gated_forward(q, s, wq, ws, wq, ws, out_dtype=dtype, out=buf[pad:pad + rows * f].view(rows, f))
        assert (buf[:pad] == 77).all() and (buf[pad + rows * f:] == 77).all()
    # the raw backward entry, every output between guards
    es = 2
    outs = [guarded(n, torch.bfloat16) for n in (rows * d, f * d, f * d, d * f)]
    _, gate, up = gpu.gated_ffn_forward(x, wg, wu, wd, return_pre=True)
    lib = gpu.lib()
    nbytes = lib.fastnn_b200_gated_ffn_workspace(2, rows, d, f, 1, 0)
    ws = torch.full((nbytes + 2 * pad,), 7, device="cuda", dtype=torch.uint8)
    rc = lib.fastnn_b200_gated_ffn_backward(2, x.data_ptr(), d, x.data_ptr(), d, gate.data_ptr(), up.data_ptr(),
                                            wg.data_ptr(), wu.data_ptr(), wd.data_ptr(),
                                            *[o.data_ptr() + es * pad for o in outs], rows, d, f, 5,
                                            ws.data_ptr() + pad, nbytes, gpu.current_stream_ptr())
    assert rc == 0
    for o in outs:
        assert (o[:pad] == 77).all() and (o[-pad:] == 77).all()
    assert (ws[:pad] == 7).all() and (ws[-pad:] == 7).all()
    for o, r in zip(outs, gpu.gated_ffn_backward(x, x, gate, up, wg, wu, wd)):
        assert torch.equal(o[pad:-pad].view(r.shape), r)


def test_a_short_workspace_is_refused(gpu):
    import torch
    x, wg, wu, wd = _inputs(4, 64, 128, torch.bfloat16)
    y = torch.zeros_like(x)
    lib = gpu.lib()
    nbytes = lib.fastnn_b200_gated_ffn_workspace(2, 4, 64, 128, 0, 0)
    ws = torch.zeros(nbytes, device="cuda", dtype=torch.uint8)
    call = lambda p, n: lib.fastnn_b200_gated_ffn_forward(2, x.data_ptr(), 64, wg.data_ptr(), wu.data_ptr(),  # noqa: E731
                                                          wd.data_ptr(), y.data_ptr(), 0, 0, 4, 64, 128, 5, p, n,
                                                          gpu.current_stream_ptr())
    assert call(ws.data_ptr(), nbytes - 1) == -1 and call(0, nbytes) == -1 and call(ws.data_ptr() + 8, nbytes) == -1
    torch.cuda.synchronize()
    assert not y.any()
    assert call(ws.data_ptr(), nbytes) == 0


def test_python_refusals(gpu):
    import torch
    x, wg, wu, wd = _inputs(4, 64, 128, torch.bfloat16)
    bad = [dict(x=x.half()), dict(x=x[:, :63]), dict(x=x.t()), dict(x=x[:1].expand(4, 64)), dict(wu=wu[:64]), dict(wd=wg),
           dict(wg=wg.t().contiguous().t()), dict(x=x.cpu()), dict(wg=wg.cpu()), dict(act=3), dict(act=99),
           dict(out=torch.empty(4, 65, device="cuda", dtype=torch.bfloat16)), dict(out=x.float())]
    for change in bad:
        a = dict(x=x, wg=wg, wu=wu, wd=wd, act=gpu.ACT_SILU, out=None)
        a.update(change)
        with pytest.raises(ValueError):
            gpu.gated_ffn_forward(a["x"], a["wg"], a["wu"], a["wd"], act=a["act"], out=a["out"])
    _, gate, up = gpu.gated_ffn_forward(x, wg, wu, wd, return_pre=True)
    for args in ((x[:2], x, gate, up), (x.half(), x, gate, up), (x, x, gate[:2], up), (x, x, gate, up.float()),
                 (x, x, gate.t().contiguous().t(), up)):
        with pytest.raises(ValueError):
            gpu.gated_ffn_backward(*args, wg, wu, wd)
    q, s = gpu.quantize_rows(x)
    wq, ws = gpu.quantize_rows(wg)
    with pytest.raises(ValueError):
        gpu.quantize_rows(x.to(torch.int32))
    with pytest.raises(ValueError):
        gpu.quantize_rows(x[:, ::2])
    for args, kw in (((q.float(), s, wq, ws), {}), ((q, s[:2], wq, ws), {}), ((q, s, wq[:, :32], ws), {}),
                     ((q, s, wq, ws[:3]), {}), ((q, s.double(), wq, ws), {}), ((q, s, wq, ws), dict(bias=s)),
                     ((q, s, wq, ws), dict(out_dtype=torch.int8)), ((q, s, wq, ws), dict(act=4)),
                     ((q.t().contiguous().t(), s, wq, ws), {})):
        with pytest.raises(ValueError):
            gpu.int8_linear_forward(*args, **kw)
    with pytest.raises(ValueError):
        gpu.int8_gated_forward(q, s, wq, ws, wq[:64], ws[:64])
    wide = torch.zeros(2, 131072, device="cuda", dtype=torch.int8)
    with pytest.raises(ValueError):
        gpu.int8_linear_forward(wide, s[:2].contiguous(), wide, s[:2].contiguous())


def test_the_longest_integer_sum_is_exact(gpu):
    import torch
    k = 131071
    for rows in (2, 600):                                    # both kernels; rows of an odd length
        x = torch.full((rows, k), -128, device="cuda", dtype=torch.int8)
        w = torch.full((20, k), -128, device="cuda", dtype=torch.int8)
        one = torch.ones(rows, device="cuda"), torch.ones(20, device="cuda")
        y = gpu.int8_linear_forward(x, one[0], w, one[1])
        assert (y == float(k * 128 * 128)).all()             # 2147467264 = 131071 * 2^14: exact in FP32 too


def test_special_values_stay_in_their_rows(gpu):
    import torch
    for rows in (40, 600):
        x, wg, wu, wd = _inputs(rows, 128, 256, torch.bfloat16)
        clean = gpu.gated_ffn_forward(x, wg, wu, wd)
        bad = x.clone()
        bad[3, 5] = float("nan")
        bad[rows - 1, 0] = float("inf")
        y = gpu.gated_ffn_forward(bad, wg, wu, wd)
        keep = torch.ones(rows, dtype=torch.bool, device="cuda")
        keep[[3, rows - 1]] = False
        assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[3]).all() and not torch.isfinite(y[rows - 1]).any()
        q, s = gpu.quantize_rows(bad)
        wq, ws = gpu.quantize_rows(wg)
        y8 = gpu.int8_linear_forward(q, s, wq, ws, out_dtype=torch.bfloat16)
        assert torch.isnan(y8[~keep]).all() and torch.isfinite(y8[keep]).all()
    # far out on both sides of every activation: finite, and the limits
    big = torch.tensor([[-3.0e38, -1e30, -200.0, -90.0, -20.0, 0.0, 20.0, 90.0]], device="cuda")
    eye = torch.eye(8, device="cuda")
    for act, name in ((gpu.ACT_SILU, "silu"), (gpu.ACT_GELU, "gelu"), (gpu.ACT_RELU, "relu")):
        h = gpu.gated_ffn_forward(big, eye, torch.zeros_like(eye), eye, act=act, return_pre=True)
        assert torch.isfinite(h[0]).all(), name
        grads = gpu.gated_ffn_backward(torch.ones_like(big), big, big, torch.ones_like(big), eye, eye, eye, act=act)
        assert torch.isfinite(grads[0]).all(), name
        assert (grads[0][0, :3].abs() <= 1e-6).all(), name


def test_side_stream_and_named_stream(gpu):
    import torch
    x, wg, wu, wd = _inputs(300, 256, 512, torch.bfloat16)
    want = gpu.gated_ffn_forward(x, wg, wu, wd, return_pre=True)
    grads = gpu.gated_ffn_backward(x, x, want[1], want[2], wg, wu, wd)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    late = torch.zeros_like(x)
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late.copy_(x)                                        # the call must see what its stream wrote
        y = gpu.gated_ffn_forward(late, wg, wu, wd)
        q, s = gpu.quantize_rows(late)
    side.synchronize()
    assert torch.equal(y, want[0])
    got = gpu.gated_ffn_backward(x, x, want[1], want[2], wg, wu, wd, stream=side.cuda_stream)
    y2 = gpu.gated_ffn_forward(x, wg, wu, wd, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(y2, want[0]) and all(torch.equal(a, b) for a, b in zip(got, grads))
    # two streams at once, many calls: each call's workspace is its own
    other = torch.cuda.Stream()
    outs = []
    for i in range(20):
        for st in (side, other):
            with torch.cuda.stream(st):
                outs.append(gpu.gated_ffn_backward(x, x, want[1], want[2], wg, wu, wd))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, grads))


@pytest.mark.parametrize("rows,d,f", [(4, 256, 512), (300, 264, 520), (700, 129, 301)])
def test_captured_graphs(gpu, rows, d, f):
    import torch
    x, wg, wu, wd = _inputs(rows, d, f, torch.bfloat16)
    wq, ws = gpu.quantize_rows(wg)
    uq, us = gpu.quantize_rows(wu)

    def step(t):
        y, gate, up = gpu.gated_ffn_forward(t, wg, wu, wd, return_pre=True)
        q, s = gpu.quantize_rows(t)
        return (y,) + gpu.gated_ffn_backward(y, t, gate, up, wg, wu, wd) + \
            (gpu.int8_gated_forward(q, s, wq, ws, uq, us, out_dtype=torch.bfloat16),)
    graphs = []
    for i in range(2):
        static = x.clone()
        step(static)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(static)
        graphs.append((g, static, out, torch.cuda.Stream()))
    news = [_inputs(rows, d, f, torch.bfloat16, seed=9 + i)[0] for i in range(2)]
    wants = [step(n) for n in news]
    torch.cuda.synchronize()
    for (g, static, out, _), n in zip(graphs, news):
        static.copy_(n)
    torch.cuda.synchronize()
    for _ in range(5):                                       # both graphs in flight at once, replayed again
        for g, _, _, st in graphs:
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (_, _, out, _), want in zip(graphs, wants):
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_offsets_beyond_32_bits(gpu):
    import torch
    rows, n = 262_200, 8201                                  # 2^31 < rows * n; rows of an odd length
    q = torch.randint(-127, 128, (rows, 16), device="cuda", dtype=torch.int8)
    s = torch.rand(rows, device="cuda")
    w = torch.randint(-127, 128, (n, 16), device="cuda", dtype=torch.int8)
    ws = torch.rand(n, device="cuda")
    y = gpu.int8_linear_forward(q, s, w, ws, out_dtype=torch.bfloat16)
    for lo in (0, rows // 2, rows - 70):
        want = (q[lo:lo + 70].double() @ w.double().t()) * s[lo:lo + 70].double()[:, None] * ws.double()
        assert _rel(y[lo:lo + 70], want) <= _tol(y)
    top = y.view(rows, n)
    qq, ss = gpu.quantize_rows(top)                          # more than 2^31 elements in
    for lo in (0, rows - 5):
        part = top[lo:lo + 5].contiguous()
        pq, ps = gpu.quantize_rows(part)
        assert torch.equal(qq[lo:lo + 5], pq) and torch.equal(ss[lo:lo + 5], ps)


def test_gradients_against_differences(gpu):
    """<gradient, v> against the change of the 64-bit loss sum(y * r) along v.  A central difference with
    step 1e-4 in 64 bits is good to about 1e-8 relative here; what remains is the error e of the gradient
    itself, |e| <= 8 * 2^-11 |gradient| (the saved projections, the operands of its products and the
    result are rounded, twice the norm of each).  <e, v> with v of independent standard normals is |e| times a
    standard normal: four of those."""
    import torch
    rows, d, f = 96, 80, 144
    x, wg, wu, wd = _inputs(rows, d, f, torch.float16)
    g = torch.Generator(device="cuda").manual_seed(5)
    r = torch.randn(rows, d, generator=g, device="cuda").half()
    _, gate, up = gpu.gated_ffn_forward(x, wg, wu, wd, return_pre=True)
    grads = gpu.gated_ffn_backward(r, x, gate, up, wg, wu, wd)
    base = [t.double() for t in (x, wg, wu, wd)]
    for i, grad in enumerate(grads):
        v = torch.randn(grad.shape, generator=g, device="cuda", dtype=torch.float64)

        def loss(t):
            args = list(base)
            args[i] = base[i] + t * v
            return (_block64(*args) * r.double()).sum()
        slope = (loss(1e-4) - loss(-1e-4)) / 2e-4
        got = (grad.double() * v).sum()
        assert abs(got - slope) <= 8 * 2.0 ** -11 * grad.double().norm() * v.norm() / grad.numel() ** 0.5 * 4


def test_train_then_quantise_and_serve(gpu):
    """The operators together: steps of training in bf16, then the trained block's weights in 8 bits and
    its serving form for a prompt and for single tokens, against the 64-bit value of the same 8-bit block."""
    import torch
    rows, d, f = 512, 128, 384
    x, wg, wu, wd = _inputs(rows, d, f, torch.bfloat16, seed=1)
    target = _inputs(rows, d, f, torch.bfloat16, seed=2)[0]
    master = [w.float() for w in (wg, wu, wd)]
    for _ in range(3):
        ws = [m.bfloat16() for m in master]
        y, gate, up = gpu.gated_ffn_forward(x, *ws, return_pre=True)
        grads = gpu.gated_ffn_backward((y - target) / rows, x, gate, up, *ws)
        for m, gr in zip(master, grads[1:]):
            assert torch.isfinite(gr).all() and gr.any()
            m.sub_(gr.float())
    (gq, gs), (uq, us), (dq, ds) = [gpu.quantize_rows(m) for m in master]
    for t in (1, 7, rows):
        q, s = gpu.quantize_rows(x[:t].contiguous())
        h = gpu.int8_gated_forward(q, s, gq, gs, uq, us, out_dtype=torch.bfloat16)
        hq, hs = gpu.quantize_rows(h)
        y = gpu.int8_linear_forward(hq, hs, dq, ds, out_dtype=torch.bfloat16)
        g64 = (q.double() @ gq.double().t()) * s.double()[:, None] * gs.double()
        u64 = (q.double() @ uq.double().t()) * s.double()[:, None] * us.double()
        h64 = g64 * torch.sigmoid(g64) * u64
        assert _rel(h, h64) <= _tol(h)
        want = (hq.double() @ dq.double().t()) * hs.double()[:, None] * ds.double()
        assert _rel(y, want) <= _tol(y)
        # and near the block it came from: 127 steps to the largest value of a row, on both operands
        ref = _block64(x[:t], *[m.bfloat16() for m in master])
        assert _rel(y, ref) <= 0.05


def test_two_threads_on_two_streams(gpu):
    """Calls from two host threads, each on its own stream and with its own kernel-form override (which
    belongs to the calling thread), at the same time."""
    import threading
    import torch
    cases = [_inputs(300, 512, 1024, torch.bfloat16, seed=1), _inputs(20, 1000, 520, torch.float16, seed=2)]

    def work(x, wg, wu, wd):
        y, gate, up = gpu.gated_ffn_forward(x, wg, wu, wd, return_pre=True)
        q, s = gpu.quantize_rows(x)
        wq, ws = gpu.quantize_rows(wg)
        return (y,) + gpu.gated_ffn_backward(y, x, gate, up, wg, wu, wd) + (gpu.int8_linear_forward(q, s, wq, ws),)
    want = [work(*c) for c in cases]
    torch.cuda.synchronize()
    bad, errors = [], []

    def run(i):
        try:
            torch.cuda.set_device(0)
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(30):
                    got = work(*cases[i])
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        bad.append(i)
        except Exception as exc:                             # reported by the thread that asserts
            errors.append(exc)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and not bad


def test_a_weight_used_twice_and_views_of_one_buffer(gpu):
    import torch
    for rows in (4, 300):
        x, w, _, wd = _inputs(rows, 128, 256, torch.bfloat16)
        want = _block64(x, w, w, wd)
        assert _rel(gpu.gated_ffn_forward(x, w, w, wd), want) <= _tol(x)
        square = _inputs(128, 128, 128, torch.bfloat16, seed=4)[0]
        y, gate, up = gpu.gated_ffn_forward(square, square, square, square, return_pre=True)
        assert _rel(y, _block64(square, square, square, square)) <= _tol(x)
        dx, a, b, c = gpu.gated_ffn_backward(square, square, gate, up, square, square, square, act=gpu.ACT_SILU)
        again = gpu.gated_ffn_backward(square.clone(), square.clone(), gate, up, square.clone(), square.clone(),
                                       square.clone(), act=gpu.ACT_SILU)
        assert all(torch.equal(p, q) for p, q in zip((dx, a, b, c), again))
