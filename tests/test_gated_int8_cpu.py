"""CPU: what the gated feed-forward and 8-bit entries refuse, at the C ABI and in Python, before any launch."""
import ctypes

import pytest

P = ctypes.c_void_p(4096)
NULL = ctypes.c_void_p(0)


def _fwd(lib, dtype=2, ld=64, rows=4, d=64, f=128, act=5, x=P, y=P, gate=NULL, up=NULL, ws=P, nbytes=1 << 20):
    return lib.fastnn_b200_gated_ffn_forward(dtype, x, ld, P, P, P, y, gate, up, rows, d, f, act, ws, nbytes, NULL)


def _bwd(lib, dtype=2, ld_dy=64, ld_x=64, rows=4, d=64, f=128, act=5, dwd=P):
    return lib.fastnn_b200_gated_ffn_backward(dtype, P, ld_dy, P, ld_x, P, P, P, P, P, P, P, P, dwd, rows, d, f, act, P,
                                              1 << 20, NULL)


def test_c_abi_refuses_bad_arguments(built_library):
    import fastnn_b200 as f
    lib = f.lib()
    for bad in (dict(dtype=3), dict(dtype=-1), dict(ld=63), dict(rows=-1), dict(d=0), dict(f=0), dict(act=3), dict(act=4),
                dict(act=6), dict(gate=P), dict(up=P), dict(x=NULL), dict(y=NULL)):
        assert _fwd(lib, **bad) == -1, bad
    for bad in (dict(dtype=9), dict(ld_dy=1), dict(ld_x=0), dict(rows=-2), dict(d=0), dict(act=-1), dict(dwd=NULL)):
        assert _bwd(lib, **bad) == -1, bad
    q = lib.fastnn_b200_quantize_rows
    for args in ((4, P, 8, P, P, 2, 8, NULL), (0, P, 7, P, P, 2, 8, NULL), (0, P, 8, P, P, -1, 8, NULL),
                 (0, P, 8, P, P, 2, 0, NULL), (0, NULL, 8, P, P, 2, 8, NULL), (0, P, 8, NULL, P, 2, 8, NULL)):
        assert q(*args) == -1, args
    lin, gated = lib.fastnn_b200_int8_linear_forward, lib.fastnn_b200_int8_gated_forward
    for rows, k, n, act, out in ((-1, 16, 16, 0, 0), (1, 0, 16, 0, 0), (1, 16, 0, 0, 0), (1, 131072, 16, 0, 0),
                                 (1, 16, 16, 4, 0), (1, 16, 16, 0, 3)):
        assert lin(P, P, P, P, NULL, P, out, rows, k, n, act, NULL, 0, NULL) == -1
        assert gated(P, P, P, P, P, P, P, out, rows, k, n, act, NULL, 0, NULL) == -1
    assert lin(P, P, NULL, P, NULL, P, 0, 1, 16, 16, 0, NULL, 0, NULL) == -1
    assert gated(P, P, P, P, NULL, P, P, 0, 1, 16, 16, 0, NULL, 0, NULL) == -1


def test_c_abi_empty_calls_and_missing_device(built_library):
    import torch
    import fastnn_b200 as f
    lib = f.lib()
    assert _fwd(lib, rows=0) == 0
    assert lib.fastnn_b200_quantize_rows(0, P, 8, P, P, 0, 8, NULL) == 0
    assert lib.fastnn_b200_int8_linear_forward(P, P, P, P, NULL, P, 0, 0, 16, 16, 0, NULL, 0, NULL) == 0
    if torch.cuda.is_available():
        return
    assert _fwd(lib) == -1 and _bwd(lib) == -1          # no context: an error, no fallback
    assert lib.fastnn_b200_quantize_rows(0, P, 8, P, P, 2, 8, NULL) == -1
    assert lib.fastnn_b200_int8_linear_forward(P, P, P, P, NULL, P, 0, 2, 16, 16, 0, NULL, 0, NULL) == -1


def test_workspace_sizes(built_library):
    import fastnn_b200 as f
    lib = f.lib()
    ws, ws8 = lib.fastnn_b200_gated_ffn_workspace, lib.fastnn_b200_int8_workspace
    assert ws(3, 4, 64, 64, 0, 0) == 0 and ws(2, -1, 64, 64, 0, 0) == 0 and ws(2, 4, 0, 64, 0, 0) == 0
    assert ws(2, 0, 64, 64, 0, 1) == 0 and ws(2, 0, 64, 64, 1, 1) == 0 and ws8(0, 16, 16, 1, 1) == 0    # no rows, no work
    # the hidden rows, at least; copies of the operands only where they are needed
    assert ws(2, 8192, 256, 1024, 0, 0) >= 8192 * 1024 * 2
    aligned, packed = ws(2, 64, 1024, 4096, 0, 0), ws(2, 64, 1024, 4096, 0, 1)
    assert packed >= aligned + 3 * 1024 * 4096 * 2
    assert ws(2, 64, 1023, 4095, 0, 0) >= 64 * 4095 * 2 + 3 * 1023 * 4095 * 2
    assert ws(2, 8192, 256, 1024, 1, 0) >= 3 * 8192 * 1024 * 2
    assert ws8(64, 1024, 512, 0, 0) == 0 and ws8(64, 1024, 512, 1, 1) >= (64 + 2 * 512) * 1024
    assert ws8(64, 1001, 512, 0, 0) >= (64 + 512) * 1001


def test_python_refuses_bad_tensors(built_library):
    import torch
    import fastnn_b200 as f
    x, w, wd = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(128, 64, dtype=torch.bfloat16), torch.zeros(64, 128)
    with pytest.raises(ValueError):
        f.gated_ffn_forward(x, w, w, wd)                         # not on a GPU
    with pytest.raises(ValueError):
        f.gated_ffn_backward(x, x, x, x, w, w, wd)
    with pytest.raises(ValueError):
        f.quantize_rows(x)
    with pytest.raises(ValueError):
        f.quantize_rows(torch.zeros(4, 4, dtype=torch.int32))
    q, s = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)
    with pytest.raises(ValueError):
        f.int8_linear_forward(q, s, q, s)
    with pytest.raises(ValueError):
        f.int8_gated_forward(q, s, q, s, q, s)
