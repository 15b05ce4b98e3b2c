"""Refusals of the entry points of linear layers with many weights that need no device: each is made before any device call."""
import ctypes

import pytest
import torch

import spconv_amd as sp

A = 0x100000  # addresses that nothing reads, 1 MB apart


def p(v):
    return ctypes.c_void_p(v)


def refused(rc, word):
    lib = sp.load_library()
    assert rc == -1
    assert word in lib.spc_last_error().decode(), lib.spc_last_error()


def test_forward():
    lib = sp.load_library()

    def call(x=A, w=2 * A, ends=3 * A, bias=None, dt=2, bdt=0, n=4, g=3, k=64, o=72, y=4 * A, work=None, nwork=0):
        return lib.spc_group_linear(p(x), p(w), p(ends), p(bias), dt, bdt, n, g, k, o, p(y), p(work), nwork)

    refused(call(k=60), "multiple of 8")
    refused(call(o=70), "multiple of 8")
    refused(call(k=(1 << 20) + 8), "2^20")
    refused(call(g=0), "G=0")
    refused(call(g=(1 << 16) + 1), "groups")
    refused(call(n=-1), "N=-1")
    refused(call(n=1 << 31), "rows")
    refused(call(dt=0), "bf16/fp16")
    refused(call(dt=5), "dtype code 5")
    refused(call(x=A + 2), "aligned")
    refused(call(y=4 * A + 8), "aligned")
    refused(call(x=None), "null")
    refused(call(w=None), "null")
    refused(call(ends=None), "null")
    refused(call(y=None), "null")
    refused(call(y=A), "overlap")
    refused(call(y=2 * A + 16), "overlap")
    refused(call(y=3 * A), "overlap")
    refused(call(bias=4 * A + 64), "overlap")
    refused(call(bias=5 * A, bdt=3), "dtype code 3")
    assert call(n=0, x=None, y=None) == 0
    # 600 rows of one group: few tiles, deep
    deep = dict(n=600, g=1, k=4096, o=128, x=0x10000000, w=0x20000000, y=0x30000000)
    refused(call(**deep, work=0x40000000, nwork=16), "workspace of 16 bytes")
    refused(call(**deep, work=0x40000008, nwork=1 << 30), "16-byte aligned")
    for over in ("x", "w", "y"):
        refused(call(**deep, work=deep[over], nwork=1 << 30), "overlap the workspace")


def test_gradients():
    lib = sp.load_library()

    def dx(dy=A, w=2 * A, ends=3 * A, dt=2, n=4, g=3, k=64, o=72, out=4 * A, work=None, nwork=0):
        return lib.spc_group_linear_dx(p(dy), p(w), p(ends), dt, n, g, k, o, p(out), p(work), nwork)

    def dw(dy=A, x=2 * A, ends=3 * A, dt=2, n=4, g=3, k=64, o=72, odt=0, out=4 * A, db=5 * A, work=None, nwork=0):
        return lib.spc_group_linear_dw(p(dy), p(x), p(ends), dt, n, g, k, o, odt, p(out), p(db), p(work), nwork)

    refused(dx(k=4), "multiple of 8")
    refused(dx(dt=0), "bf16/fp16")
    refused(dx(out=A + 16), "overlap")
    refused(dx(out=2 * A), "overlap")
    refused(dx(w=None), "null")
    refused(dx(ends=None), "null")
    assert dx(n=0, dy=None, out=None) == 0
    refused(dx(n=500, g=1, k=128, o=4096, dy=0x10000000, w=0x20000000, out=0x30000000, work=0x40000000, nwork=16), "workspace of 16 bytes")
    refused(dx(n=500, g=1, k=128, o=4096, dy=0x10000000, w=0x20000000, out=0x30000000, work=0x10000000, nwork=1 << 30), "overlap the workspace")
    deep = dict(n=9000, g=1, k=128, o=128, dy=0x10000000, x=0x20000000, out=0x30000000)
    refused(dw(**deep, work=0x40000000, nwork=16), "workspace of 16 bytes")
    refused(dw(**deep, work=5 * A, nwork=1 << 30), "overlap the workspace")
    refused(dw(o=12), "multiple of 8")
    refused(dw(odt=1), "fp32 or of dy's type")
    refused(dw(out=None), "null")
    refused(dw(out=A), "overlap")
    refused(dw(out=2 * A), "overlap")
    refused(dw(db=A), "overlap")
    refused(dw(db=4 * A + 64), "overlap")
    refused(dw(db=5 * A + 4), "aligned")
    refused(dw(x=None), "null")
    refused(dw(n=1 << 31), "rows")


def test_workspaces():
    """Zero unless a few tiles are deep; the adapters' also holds the first product, except a single row's."""
    lib, n = sp.load_library(), ctypes.c_int64()

    def group(*sizes):
        assert lib.spc_group_linear_workspace(*sizes, ctypes.byref(n)) == 0
        return n.value

    def adapter(*sizes):
        assert lib.spc_adapter_workspace(*sizes, ctypes.byref(n)) == 0
        return n.value

    assert group(sp.GROUP_FORWARD, 0, 1, 4096, 128) == group(sp.GROUP_FORWARD, 64, 1, 4096, 128) == group(sp.GROUP_FORWARD, 500, 1, 1024, 128) == 0
    assert group(sp.GROUP_FORWARD, 16000, 8, 4096, 4096) == 0
    assert group(sp.GROUP_FORWARD, 600, 1, 4096, 128) % (600 * 128 * 4) == 0 < n.value < 1 << 26
    assert group(sp.GROUP_DX, 500, 1, 128, 4096) % (500 * 128 * 4) == 0 < n.value < 1 << 26
    assert group(sp.GROUP_DW, 9000, 1, 128, 136) % (129 * 136 * 4) == 0 < n.value < 1 << 26
    assert group(sp.GROUP_DW, 1000, 1, 128, 128) == group(sp.GROUP_DW, 0, 1, 128, 128) == 0
    assert adapter(0, 8, 64, 64) == adapter(1, 16, 4096, 4096) == adapter(1, 16, 0, 4096) == 0
    assert adapter(7, 24, 0, 64) == 512 and adapter(500, 8, 64, 64) == 500 * 16 // 256 * 256 + 256
    assert adapter(600, 8, 4096, 128) > adapter(600, 8, 0, 128) > 0
    for bad in ((3, 4, 1, 64, 64), (-1, 4, 1, 64, 64), (0, 1 << 31, 1, 64, 64), (0, 4, 0, 64, 64), (0, 4, 1, 0, 64), (0, 4, 1, 64, 1 << 21)):
        refused(lib.spc_group_linear_workspace(*bad, ctypes.byref(n)), "arguments")
    refused(lib.spc_group_linear_workspace(0, 4, 1, 64, 64, None), "arguments")
    for bad in ((4, 0, 64, 64), (1 << 31, 8, 64, 64), (4, 264, 64, 64), (4, 8, -1, 64), (4, 8, 64, 0)):
        refused(lib.spc_adapter_workspace(*bad, ctypes.byref(n)), "arguments")
    refused(lib.spc_adapter_workspace(4, 8, 64, 64, None), "arguments")


def test_adapters():
    lib = sp.load_library()

    def linear(x=A, w=2 * A, a=3 * A, b=4 * A, slots=5 * A, scale=None, bias=None, dt=2, bdt=0, n=4, l=3, r=16, k=64, o=72, out=6 * A,
               work=None, nwork=0):
        return lib.spc_adapter_linear(p(x), p(w), p(a), p(b), p(slots), p(scale), p(bias), dt, bdt, n, l, r, k, o, p(out), p(work), nwork)

    def add(y=2 * A, x=A, a=3 * A, b=4 * A, slots=5 * A, scale=None, dt=2, n=4, l=3, r=16, k=64, o=72, out=6 * A, work=None, nwork=0):
        return lib.spc_adapter_add(p(y), p(x), p(a), p(b), p(slots), p(scale), dt, n, l, r, k, o, p(out), p(work), nwork)

    for call in (linear, add):
        refused(call(r=12), "multiple of 8")
        refused(call(r=264), "at most 256")
        refused(call(k=12), "multiple of 8")
        refused(call(o=12), "multiple of 8")
        refused(call(l=0), "L=0")
        refused(call(l=(1 << 16) + 1), "adapters")
        refused(call(dt=0), "bf16/fp16")
        refused(call(a=None), "null")
        refused(call(b=4 * A + 4), "aligned")
        refused(call(slots=None), "null")
        refused(call(out=None), "null")
        refused(call(out=A), "overlap")
        refused(call(out=3 * A), "overlap")
        refused(call(out=4 * A), "overlap")
        refused(call(out=5 * A), "overlap")
        refused(call(scale=6 * A), "overlap")
        refused(call(n=1 << 31), "rows")
        refused(call(n=(1 << 27) + 1, x=A, a=1 << 60, b=1 << 61), "2^27")
        assert call(n=0, x=None, slots=None, out=None, **({"y": None} if call is add else {})) == 0
    refused(linear(out=2 * A), "overlap")
    refused(linear(bias=6 * A), "overlap")
    refused(add(out=2 * A + 16), "apart")


def test_binding():
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((3, 72, 64), dtype=torch.bfloat16)
    ends, a, b = torch.zeros(3, dtype=torch.int32), torch.zeros((2, 8, 64), dtype=torch.bfloat16), torch.zeros((2, 72, 8), dtype=torch.bfloat16)
    slots, dy = torch.zeros(4, dtype=torch.int32), torch.zeros((4, 72), dtype=torch.bfloat16)
    for call in (lambda: sp.group_linear(x, w, ends),  # on the CPU
                 lambda: sp.group_linear(x, w[0], ends), lambda: sp.group_linear(x, w, ends.long()), lambda: sp.group_linear(x.half(), w, ends),
                 lambda: sp.group_linear(x, w, ends, bias=dy), lambda: sp.group_linear_dx(x, w, ends),
                 lambda: sp.group_linear_dw(dy, x[:3], ends), lambda: sp.group_linear_dw(dy, x, ends, out=w, out_dtype=torch.float32),
                 lambda: sp.adapter_linear(x, w[0], a, b, slots.long()), lambda: sp.adapter_linear(x, w[0], a, b[:1], slots),
                 lambda: sp.adapter_linear(x, w[0], a, b, slots, scale=torch.ones(3)), lambda: sp.adapter_add(x, x, a, b, slots)):
        with pytest.raises((ValueError, RuntimeError)):
            call()


def test_adapter_workspace_borders():
    """Nothing for up to 4 rows and 32 products of rows and ranks, which are one kernel; else half of the rows' inner products, and at least one row's."""
    lib, n = sp.load_library(), ctypes.c_int64()

    def adapter(rows, rank, k=0, o=64):
        assert lib.spc_adapter_workspace(rows, rank, k, o, ctypes.byref(n)) == 0
        return n.value

    for rows, rank in ((1, 8), (1, 32), (2, 16), (4, 8), (1, 24)):
        assert adapter(rows, rank) == adapter(rows, rank, 4096, 4096) == 0
    for rows, rank in ((5, 8), (1, 40), (3, 16), (2, 24), (1, 256), (2, 256), (1000, 64), (1 << 27, 256)):
        assert adapter(rows, rank) % 256 == 0 and adapter(rows, rank) >= max((rows + 1) // 2 * rank * 4, rank * 4 + (rank + 63) // 64 * 4)
        assert adapter(rows, rank, 64) == adapter(rows, rank)
    # with 3 N R bytes more there is room for every row's ranks and factors
    for rows in (1, 3, 5, 17, 1001):
        for rank in range(8, 264, 8):
            least = adapter(rows, rank)
            assert least == 0 or least + 3 * rows * rank >= (rows * (rank * 4 + (rank + 63) // 64 * 4) + 15) // 16 * 16
