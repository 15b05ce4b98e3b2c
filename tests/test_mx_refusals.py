"""Refusals of the microscaled entry points that need no device: each is made before any device call."""
import ctypes

import pytest
import torch

import spconv_amd as sp

A = 0x10000  # an address that nothing reads


def p(v):
    return ctypes.c_void_p(v)


def refused(rc, word):
    lib = sp.load_library()
    assert rc == -1
    assert word in lib.spc_last_error().decode(), lib.spc_last_error()


def test_sizes():
    lib = sp.load_library()
    c, s = ctypes.c_int64(), ctypes.c_int64()
    for rows, cols, fmt, want in ((3, 32, 2, (48, 48)), (3, 512, 1, (1536, 48)), (3, 544, 2, (816, 96)), (0, 64, 1, (0, 0))):
        assert lib.spc_mx_sizes(rows, cols, fmt, ctypes.byref(c), ctypes.byref(s)) == 0 and (c.value, s.value) == want
    refused(lib.spc_mx_sizes(3, 33, 1, None, None), "cols=33")
    refused(lib.spc_mx_sizes(3, 32, 4, None, None), "format 4")
    refused(lib.spc_mx_sizes(1 << 31, 32, 1, None, None), "rows=2147483648")
    n = ctypes.c_int64()
    assert lib.spc_mx_linear_workspace(100, 64, 2, ctypes.byref(n)) == 0 and n.value >= 100 * 32 + 100 * 16
    assert lib.spc_convnext_mlp_mx_workspace(10, 64, 1, ctypes.byref(n)) == 0 and n.value >= 10 * (64 + 256) + 20 * 16
    for rows in (0, 16):  # few rows are quantised on the way
        assert lib.spc_mx_linear_workspace(rows, 64, 2, ctypes.byref(n)) == 0 and n.value == 0


def test_tail_in_one_kernel_by_rows():
    """The tail is one kernel, without a workspace, from the rows on where that is the faster form."""
    lib, n = sp.load_library(), ctypes.c_int64()
    for rows, c, fmt, one in ((128, 128, 1, False), (129, 128, 1, True), (129, 128, 2, False), (129, 256, 1, False), (4000, 256, 1, False),
                              (6145, 256, 1, True), (6145, 256, 2, False), (6145, 512, 1, False)):
        assert lib.spc_convnext_mlp_mx_workspace(rows, c, fmt, ctypes.byref(n)) == 0 and (n.value == 0) == one, (rows, c, fmt)


def test_quantize():
    lib = sp.load_library()
    refused(lib.spc_mx_quantize(p(A), 2, 4, 48, 1, p(2 * A), p(3 * A)), "multiple of 32")
    refused(lib.spc_mx_quantize(p(A), 2, 4, 64, 0, p(2 * A), p(3 * A)), "format 0")
    refused(lib.spc_mx_quantize(p(A), 3, 4, 64, 1, p(2 * A), p(3 * A)), "dtype code 3")
    refused(lib.spc_mx_quantize(p(A + 8), 2, 4, 64, 1, p(2 * A), p(3 * A)), "aligned")
    refused(lib.spc_mx_quantize(p(A), 2, 4, 64, 1, p(2 * A + 4), p(3 * A)), "aligned")
    refused(lib.spc_mx_quantize(p(A), 2, 4, 64, 1, None, p(3 * A)), "null")
    refused(lib.spc_mx_quantize(p(A), 2, 4, 64, 1, p(A + 64), p(3 * A)), "overlap")
    refused(lib.spc_mx_quantize(None, 2, 4, 64, 1, p(2 * A), p(3 * A)), "null")
    refused(lib.spc_mx_quantize(p(A), 2, -1, 64, 1, p(2 * A), p(3 * A)), "rows=-1")
    refused(lib.spc_mx_dequantize(p(A), p(2 * A), 4, 64, 1, 2, p(A + 16)), "overlap")
    assert lib.spc_mx_quantize(None, 2, 0, 64, 1, None, None) == 0


def test_norm():
    lib = sp.load_library()

    def call(x=A, r=2 * A, kind=0, dt=2, n=4, c=64, fmt=1, s=3 * A, codes=4 * A, scales=5 * A):
        return lib.spc_add_norm_mx(p(x), p(r), None, None, 0, 1e-6, kind, dt, n, c, fmt, p(s), p(codes), p(scales))

    refused(call(c=16416), "at most 16384")
    refused(call(c=40), "multiple of 32")
    refused(call(kind=2), "kind=2")
    refused(call(dt=0), "bf16/fp16")
    refused(call(s=None), "needs a sum")
    refused(call(s=A + 16), "apart")
    refused(call(s=2 * A + 16), "apart")
    refused(call(codes=3 * A), "overlap")
    refused(call(scales=A), "overlap")
    refused(call(x=None), "null")
    refused(call(x=A + 2), "aligned")
    assert call(n=0) == 0


def test_linear():
    lib = sp.load_library()

    def call(x=A, xs=2 * A, xdt=0, xf=1, w=3 * A, ws=4 * A, b=None, bdt=0, r=None, act=0, n=4, k=64, o=64, ot=2, y=6 * A,
             ys=None, work=None, nwork=0):
        return lib.spc_mx_linear(p(x), p(xs), xdt, xf, p(w), p(ws), p(b), bdt, p(r), act, n, k, o, ot, p(y), p(ys), p(work), nwork)

    refused(call(o=48), "multiple of 32")
    refused(call(k=48), "multiple of 32")
    refused(call(xf=5), "format 5")
    refused(call(act=3), "act=3")
    refused(call(ot=7), "dtype code 7")
    refused(call(ys=7 * A, ot=0), "format 0")
    refused(call(ys=7 * A, ot=1, r=8 * A), "no residual")
    refused(call(y=A), "overlap")
    refused(call(y=3 * A + 16), "overlap")
    refused(call(r=6 * A + 16), "apart")
    refused(call(y=6 * A + 4), "aligned")
    refused(call(y=None), "null")
    refused(call(w=None), "null")
    refused(call(b=6 * A), "overlap")
    refused(call(xs=None, xdt=5), "dtype code 5")
    refused(call(xs=None, xdt=2, xf=3), "x_fmt=3")
    refused(call(xs=None, xdt=2, y=A), "overlap")
    refused(call(xs=None, xdt=2, n=1000, work=9 * A, nwork=1), "workspace of 1 bytes")
    refused(call(xs=None, xdt=2, n=1000, y=16 * A, work=9 * A + 8, nwork=1 << 30), "16-byte aligned")
    refused(call(xs=None, xdt=2, n=1000, y=16 * A, work=16 * A, nwork=1 << 30), "overlap the workspace")
    refused(call(xs=None, xdt=2, n=1000, x=20 * A, y=16 * A, work=20 * A, nwork=1 << 30), "overlap the workspace")
    assert call(n=0, x=None, xs=None, y=None) == 0


def test_linear_tile():
    lib, r, c = sp.load_library(), ctypes.c_int(), ctypes.c_int()
    refused(lib.spc_mx_linear_tile(1, 48, 1, 2, 0, ctypes.byref(r), ctypes.byref(c)), "arguments")
    refused(lib.spc_mx_linear_tile(1, 64, 3, 2, 0, ctypes.byref(r), ctypes.byref(c)), "arguments")
    refused(lib.spc_mx_linear_tile(1, 64, 1, 2, 0, None, ctypes.byref(c)), "arguments")
    refused(lib.spc_mx_linear_tile(1, 64, 1, 9, 0, ctypes.byref(r), ctypes.byref(c)), "dtype code 9")


def test_tail():
    lib = sp.load_library()

    def call(h=A, x=2 * A, g=None, w1=3 * A, s1=4 * A, w2=5 * A, s2=6 * A, dt=2, pdt=0, fmt=1, n=4, c=64, y=7 * A, work=None, nwork=0):
        return lib.spc_convnext_mlp_mx(p(h), p(x), p(g), None, 1e-6, p(w1), p(s1), None, p(w2), p(s2), None, dt, pdt, fmt, n, c,
                                       p(y), p(work), nwork)

    refused(call(c=48), "multiple of 32")
    refused(call(c=4128), "at most 4096")
    refused(call(dt=0), "bf16/fp16")
    refused(call(fmt=4), "fmt=4")
    refused(call(y=A + 16), "apart")
    refused(call(y=3 * A), "overlap")
    refused(call(g=7 * A), "overlap")
    refused(call(h=None), "null")
    refused(call(work=9 * A, nwork=16), "workspace of 16 bytes")
    refused(call(work=7 * A, nwork=1 << 30), "overlap the workspace")
    assert call(n=0) == 0


@pytest.mark.parametrize("operand", range(8))
def test_tail_workspace_apart_from_weights_and_parameters(operand):
    """The three-pass tail writes its workspace while it still reads these."""
    lib, room = sp.load_library(), 1 << 24
    work = 16 * room
    for at in (work, work + 512):  # the same address, and one inside (200 rows of 64 and 256 columns take 64 KB and more)
        # gamma, beta, w1, s1, b1, w2, s2, b2
        ops = [(k + 1) * room for k in range(8)]
        ops[operand] = at
        g, b, w1, s1, b1, w2, s2, b2 = (p(v) for v in ops)
        refused(lib.spc_convnext_mlp_mx(p(9 * room), p(10 * room), g, b, 1e-6, w1, s1, b1, w2, s2, b2, 2, 0, 1, 200, 64, p(11 * room),
                                        p(work), room), "overlap the workspace")


@pytest.mark.parametrize("scales", [2 * A, 2 * A + 64, 2 * A - 16])
def test_codes_and_scales_apart(scales):
    """A call that writes both refuses buffers that share a byte (4 rows of 64 columns: 256 bytes of codes, 64 of scales)."""
    lib, c, s = sp.load_library(), p(2 * A), p(scales)
    refused(lib.spc_mx_quantize(p(A), 2, 4, 64, 1, c, s), "codes and scales must not overlap")
    refused(lib.spc_add_norm_mx(p(A), None, None, None, 0, 1e-6, 0, 2, 4, 64, 1, None, c, s), "codes and scales must not overlap")
    refused(lib.spc_mx_linear(p(4 * A), p(5 * A), 0, 1, p(6 * A), p(7 * A), None, 0, None, 0, 4, 64, 64, 1, c, s, None, 0),
            "codes and scales must not overlap")


def test_binding():
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    for call in (lambda: sp.mx_quantize(x[0]),
                 lambda: sp.MxTensor(x, x, 64, sp.MX_E4M3),
                 lambda: sp.MxTensor(torch.zeros((4, 64), dtype=torch.uint8), torch.zeros((4, 2), dtype=torch.uint8), 64, sp.MX_E4M3),
                 lambda: sp.MxTensor(torch.zeros((4, 64), dtype=torch.uint8), torch.zeros((4, 16), dtype=torch.uint8), 64, 0),
                 lambda: sp.MxTensor(torch.zeros((4, 48), dtype=torch.uint8), torch.zeros((4, 16), dtype=torch.uint8), 48, sp.MX_E4M3),
                 lambda: sp.mx_linear(x, x)):
        with pytest.raises(ValueError):
            call()
