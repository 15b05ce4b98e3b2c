"""Linear layers with many weights on the GPU against their definitions in 64 bits.

Whole numbers: operands are small integers, every product and sum is exact in fp32 (below 2^24) and what is held in 16 bits
between the two products of an adapter too, so the results have to be the exact ones, rounded once, bit for bit. Other values: a sum
of K products in fp32, in any order, is off by at most K 2^-23 of the sum of their magnitudes (each of its additions by 2^-23 of a
partial sum, whether the unit rounds or cuts), the result's rounding by finfo.eps / 2 of it, or half of the type's smallest step.
An adapter's inner product is rounded once more (scaled, to 16 bits): that, and its own sum's error, reach the result through |b|.
"""
import pytest
import torch

import spconv_amd as sp

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(g, *shape, most=3, dt=torch.bfloat16):
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(dt)


def values(g, *shape, dt=torch.bfloat16):
    return torch.randn(shape, generator=g, device="cuda").to(dt)


def ends_of(lengths):
    return torch.tensor(lengths, device="cuda").cumsum(0).int()


def spans(ends, n):
    """Each group's rows."""
    e = [0] + [min(max(v, 0), n) for v in ends.tolist()]
    return [slice(s, max(s, t)) for s, t in zip(e, e[1:])]


def forward64(x, w, ends, bias, into):
    y = into.double()
    for g, s in enumerate(spans(ends, len(x))):
        y[s] = x[s].double() @ w[g].double().T + (0 if bias is None else bias[g].double())
    return y


def dx64(dy, w, ends, into):
    dx = into.double()
    for g, s in enumerate(spans(ends, len(dy))):
        dx[s] = dy[s].double() @ w[g].double()
    return dx


def dw64(dy, x, ends):
    at = spans(ends, len(x))
    return torch.stack([dy[s].double().T @ x[s].double() for s in at]), torch.stack([dy[s].double().sum(0) for s in at])


def near(got, want, size, depth, what=""):
    """size: the sums of the magnitudes."""
    t = torch.finfo(got.dtype)
    tol = depth * 2.0 ** -23 * size
    tol = tol + t.eps / 2 * (want.abs() + tol) + t.tiny * t.eps / 2
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


# lengths of the groups, rows behind them, K, O: each size of tile and beyond, one row to many, empty groups, widths that no tile divides
SHAPES = [
    ([1], 0, 8, 8), ([0, 1, 0], 0, 64, 64), ([0, 0], 3, 32, 16), ([2, 0, 1, 5], 2, 72, 136), ([1] * 40, 0, 1024, 264),
    ([16, 17, 15, 33], 0, 512, 96), ([64, 65, 63, 1, 0], 7, 256, 256), ([100], 0, 1032, 520), ([127, 128, 129], 1, 320, 392),
    ([300, 0, 513, 255], 40, 264, 1032), ([5, 1000, 2], 0, 128, 2056), ([256, 256, 257], 0, 1416, 264), ([2500, 70, 1900], 13, 136, 520),
    # rounds of whole tiles and quartered ones behind them, in each product; more than 64 groups; one stage of depth; deep gradients
    ([2000, 700, 1500, 300], 5, 136, 8200), ([1300, 700, 1500, 300], 5, 8200, 136), ([900, 300, 0, 2000], 7, 2056, 2104), ([300] * 130, 3, 72, 520),
    ([20] * 70, 0, 520, 776), ([6000], 0, 8, 4104), ([700] * 40, 0, 264, 1032), ([9000, 4000], 0, 520, 1544),
    # few tiles of long sums, in parts
    ([1500, 0, 530], 9, 2056, 136), ([500, 0, 130], 9, 136, 2056), ([600], 0, 4104, 40), ([300], 0, 4104, 40), ([3000, 0, 2500, 7000], 20, 72, 200),
    ([3] * 130, 0, 200, 328), ([40] * 70, 9, 72, 72), ([4100], 0, 72, 1096), ([40, 25, 60, 33], 0, 4096, 1024), ([700] * 9, 0, 512, 512),
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lengths,spare,k,o", SHAPES)
def test_group_bits(gpu, lengths, spare, k, o, dt):
    g = gen(len(lengths) + k + o)
    n, ends = sum(lengths) + spare, ends_of(lengths)
    most = 3 if max(k, o) <= 2100 else 2
    x, w, dy = ints(g, n, k, most=most, dt=dt), ints(g, len(lengths), o, k, most=2, dt=dt), ints(g, n, o, most=2, dt=dt)
    if spare:  # rows of no group are not read
        x[-spare:], dy[-spare:] = float("nan"), float("inf")
    bias = ints(g, len(lengths), o, most=9, dt=torch.float32)
    for b in (None, bias, bias.to(dt)):
        out = ints(g, n, o, most=100, dt=dt)
        want = forward64(x, w, ends, b, out)
        assert sp.group_linear(x, w, ends, bias=b, out=out) is out
        assert torch.equal(out, want.to(dt))
    out = ints(g, n, k, most=100, dt=dt)
    want = dx64(dy, w, ends, out)
    assert sp.group_linear_dx(dy, w, ends, out=out) is out
    assert torch.equal(out, want.to(dt))
    dw, db = dw64(dy, x, ends)
    for odt in (None, torch.float32):
        got, gb = sp.group_linear_dw(dy, x, ends, out_dtype=odt, bias=True)
        assert got.dtype == gb.dtype == (odt or dt)
        assert torch.equal(got, dw.to(got.dtype)) and torch.equal(gb, db.to(got.dtype))
    out = torch.full_like(got, 7.0)
    assert sp.group_linear_dw(dy, x, ends, out=out) is out and torch.equal(out, got)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lengths,spare,k,o", [SHAPES[i] for i in (3, 4, 9, 11, 14, 19, 20, 21, 23)])
def test_group_values(gpu, lengths, spare, k, o, dt):
    g = gen(7)
    n, ends = sum(lengths) + spare, ends_of(lengths)
    x, w, dy, bias = values(g, n, k, dt=dt), values(g, len(lengths), o, k, dt=dt), values(g, n, o, dt=dt), values(g, len(lengths), o, dt=dt)
    zero = torch.zeros((n, o), dtype=dt, device=gpu)
    near(sp.group_linear(x, w, ends, bias=bias, out=zero.clone()), forward64(x, w, ends, bias, zero),
         forward64(x.abs(), w.abs(), ends, bias.abs(), zero), k + 1, "y")
    zero = torch.zeros((n, k), dtype=dt, device=gpu)
    near(sp.group_linear_dx(dy, w, ends, out=zero.clone()), dx64(dy, w, ends, zero), dx64(dy.abs(), w.abs(), ends, zero), o, "dx")
    want, size = dw64(dy, x, ends), dw64(dy.abs(), x.abs(), ends)
    for odt in (dt, torch.float32):
        for got, ref, s in zip(sp.group_linear_dw(dy, x, ends, out_dtype=odt, bias=True), want, size):
            near(got, ref, s, max(lengths), "dw")


def test_gradients_against_differences(gpu):
    """<dy, y(x + e) - y(x)> = <dx, e>, and the same for w and the bias: exact in whole numbers."""
    g, dt = gen(11), torch.float16
    lengths, k, o = [70, 0, 130, 9], 136, 264
    n, ends = sum(lengths), ends_of(lengths)
    x, w, dy, bias = ints(g, n, k, most=1, dt=dt), ints(g, 4, o, k, most=1, dt=dt), ints(g, n, o, most=1, dt=dt), ints(g, 4, o, dt=dt)
    ex, ew, eb = ints(g, n, k, most=1, dt=dt), ints(g, 4, o, k, most=1, dt=dt), ints(g, 4, o, most=1, dt=dt)
    y = sp.group_linear(x, w, ends, bias=bias).long()
    dx, (dw, db) = sp.group_linear_dx(dy, w, ends).long(), sp.group_linear_dw(dy, x, ends, out_dtype=torch.float32, bias=True)
    d = dy.long()
    assert ((sp.group_linear(x + ex, w, ends, bias=bias).long() - y) * d).sum() == (dx * ex.long()).sum()
    assert ((sp.group_linear(x, w + ew, ends, bias=bias).long() - y) * d).sum() == (dw.long() * ew.long()).sum()
    assert ((sp.group_linear(x, w, ends, bias=bias + eb).long() - y) * d).sum() == (db.long() * eb.long()).sum()


@pytest.mark.parametrize("lengths", [[3, 5], [300, 400]])
def test_group_not_finite(gpu, lengths):
    """An infinity or NaN stays in its row, its group's weights and its columns."""
    g, (k, o) = gen(5), (136, 200)
    n, ends = sum(lengths), ends_of(lengths)
    x, w, dy = ints(g, n, k), ints(g, 2, o, k), ints(g, n, o)
    last = lengths[0] - 1
    x[last, 3], dy[last, 7] = float("nan"), float("inf")
    y = sp.group_linear(x, w, ends)
    assert y[last].isnan().all() and torch.isfinite(y).all(1).logical_not().sum() == 1
    dx = sp.group_linear_dx(dy, w, ends)
    assert torch.isfinite(dx).all(1).logical_not().sum() == 1 and not torch.isfinite(dx[last]).all()
    dw, db = sp.group_linear_dw(dy, x, ends, bias=True)
    bad = torch.zeros((2, o, k), dtype=torch.bool, device=gpu)
    bad[0, 7, :], bad[0, :, 3] = True, True
    assert not (~torch.isfinite(dw) & ~bad).any() and dw[0, :, 3].isnan().all() and not torch.isfinite(dw[0, 7]).any()
    assert torch.isfinite(db[0, 7]).logical_not() and torch.isfinite(db).sum() == 2 * o - 1


def test_ends_outside_the_rows(gpu):
    """Ends before the first row or past the last are taken as those."""
    g, dt = gen(6), torch.float16
    x, w, dy = ints(g, 100, 64, dt=dt), ints(g, 4, 72, 64, dt=dt), ints(g, 100, 72, dt=dt)
    ends = torch.tensor([-5, 30, 1 << 30, 2 ** 31 - 1], dtype=torch.int32, device=gpu)
    same = torch.tensor([0, 30, 100, 100], dtype=torch.int32, device=gpu)
    for e in (ends, same):
        assert torch.equal(sp.group_linear(x, w, e), forward64(x, w, same, None, dy).to(dt))
        assert torch.equal(sp.group_linear_dx(dy, w, e), dx64(dy, w, same, x).to(dt))
        assert torch.equal(sp.group_linear_dw(dy, x, e), dw64(dy, x, same)[0].to(dt))


def test_falling_ends(gpu):
    """Not allowed, and what the rows get is anything; but the call ends as soon as others, and what lies behind the rows stays."""
    g, dt, n, groups = gen(14), torch.bfloat16, 1 << 20, 4096
    ends = torch.tensor([n, 0] * (groups // 2), dtype=torch.int32, device=gpu)  # 2^31 rows, were they all taken
    x, w = ints(g, n, 8, dt=dt), ints(g, groups, 8, 8, dt=dt)
    for call in (sp.group_linear, sp.group_linear_dx):
        whole = torch.full((n + 300, 8), 7.0, dtype=dt, device=gpu)
        call(x, w, ends, out=whole[:n])
        assert (whole[n:] == 7).all()


def test_group_past_four_gigabytes(gpu):
    """Rows and weights whose offsets pass 32 bits: the last ones, beside their neighbours."""
    dt, n, k = torch.bfloat16, (1 << 20) + 300, 2112
    x = torch.zeros((n, k), dtype=dt, device=gpu)
    g = gen(3)
    x[-700:], w = ints(g, 700, k), ints(g, 3, 16, k, most=2)
    ends = torch.tensor([n - 600, n - 590, n], dtype=torch.int32, device=gpu)
    y = sp.group_linear(x, w, ends)
    assert torch.equal(y[-700:], forward64(x[-700:], w, ends - (n - 700), None, y[-700:]).to(dt))
    dy = torch.zeros((n, 16), dtype=dt, device=gpu)
    dy[-700:] = ints(g, 700, 16)
    assert torch.equal(sp.group_linear_dx(dy, w, ends)[-700:], dx64(dy[-700:], w, ends - (n - 700), x[-700:]).to(dt))
    assert torch.equal(sp.group_linear_dw(dy, x, ends), dw64(dy[-700:], x[-700:], ends - (n - 700))[0].to(dt))
    del x, y, dy
    o = k = 24576
    w = torch.zeros((5, o, k), dtype=dt, device=gpu)  # 1.2 GB each
    w[4, -300:], w[4, :10] = ints(g, 300, k, most=1), ints(g, 10, k, most=1)
    for few, ends in ((7, [0, 0, 0, 0, 7]), (70, [0, 0, 2, 2, 70])):
        x, ends = ints(g, few, k, most=1), torch.tensor(ends, dtype=torch.int32, device=gpu)
        wide = x[int(ends[3]):].float() @ w[4].float().T
        assert torch.equal(sp.group_linear(x, w, ends)[int(ends[3]):], wide.to(dt))
        assert torch.equal(sp.group_linear_dx(x, w, ends)[int(ends[3]):], (x[int(ends[3]):].float() @ w[4].float()).to(dt))
        del wide
    x, dy = ints(g, 33, k), ints(g, 33, o)
    ends = torch.tensor([0, 0, 0, 0, 33], dtype=torch.int32, device=gpu)
    dw = sp.group_linear_dw(dy, x, ends, out=w)
    assert torch.equal(dw[4, -100:], (dy[:, -100:].float().T @ x.float()).to(dt)) and not dw[:4].any()


# ---- adapters --------------------------------------------------------------------------------------------------


def adapter64(y, x, a, b, slots, scale, dt):
    """(the exact sum with the inner product as it is, and held in dt)."""
    plain, held = y.clone(), y.clone()
    for s in range(len(a)):
        r = (slots == s).nonzero().squeeze(1)
        h = x[r].double() @ a[s].double().T * (1.0 if scale is None else float(scale[s]))
        plain[r] += h @ b[s].double().T
        held[r] += h.to(dt).double() @ b[s].double().T
    return plain, held


def slots_of(g, n, count, how):
    if how == "mixed":  # any order, some without an adapter
        return torch.randint(-1, count, (n,), generator=g, device="cuda").int()
    if how == "runs":
        cuts = torch.randint(0, n + 1, (max(1, n // 50),), generator=g, device="cuda").sort()[0]
        return torch.randint(-1, count, (len(cuts) + 1,), generator=g, device="cuda")[torch.searchsorted(cuts, torch.arange(n, device="cuda"), right=True)].int()
    if how == "none":
        return torch.tensor([-1, count, -2 ** 31, 2 ** 31 - 1], device="cuda")[torch.arange(n, device="cuda") % 4].int()
    return torch.full((n,), count - 1, dtype=torch.int32, device="cuda")


ADAPTERS = [  # n, adapters, rank, k, o, order
    (1, 1, 8, 8, 8, "one"), (1, 8, 16, 4096, 1024, "mixed"), (2, 3, 24, 72, 136, "mixed"), (16, 16, 16, 512, 96, "mixed"),
    (17, 5, 32, 264, 520, "mixed"), (33, 64, 64, 1032, 264, "mixed"), (64, 4, 128, 256, 2056, "mixed"), (77, 32, 16, 2048, 1416, "mixed"),
    (128, 128, 8, 72, 72, "mixed"), (129, 3, 256, 136, 392, "mixed"), (300, 7, 40, 520, 264, "runs"), (1000, 2, 16, 1416, 1032, "runs"),
    (2600, 9, 64, 320, 1096, "runs"), (700, 70, 16, 512, 512, "mixed"), (50, 4, 16, 128, 64, "none"), (600, 4, 16, 128, 256, "none"),
    (4099, 6, 24, 136, 8200, "runs"), (2000, 40, 72, 72, 8200, "mixed"), (3, 5, 8, 520, 264, "mixed"), (2, 2, 16, 4104, 72, "mixed"),
    (1, 2, 32, 1416, 200, "one"), (40, 3, 256, 264, 136, "mixed"), (600, 4, 16, 4104, 136, "runs"), (500, 4, 16, 136, 136, "mixed"), (20000, 5, 48, 72, 136, "runs"), (4099, 1, 24, 136, 264, "one"), (513, 6, 200, 64, 40, "runs"), (9, 4, 16, 16384, 64, "mixed"), (300, 4, 16, 16384, 64, "runs"), (2500, 5, 16, 136, 264, "mixed"),
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,count,rank,k,o,order", ADAPTERS)
def test_adapter_bits(gpu, n, count, rank, k, o, order, dt):
    g = gen(n + k + rank)
    slots = slots_of(g, n, count, order)
    x = ints(g, n, k, most=1, dt=dt) * (torch.rand((n, k), generator=g, device=gpu) < 20.0 / k).to(dt)  # some 20 of a row's values
    x[:, 0] += 1
    w, a, b = ints(g, o, k, most=2, dt=dt), ints(g, count, rank, k, most=2, dt=dt), ints(g, count, o, rank, most=1, dt=dt)
    scale = 2.0 ** torch.randint(-1, 3, (count,), generator=g, device=gpu).float()
    bias, y = ints(g, o, most=9, dt=torch.float32), ints(g, n, o, most=20, dt=dt)
    base = x.double() @ w.double().T
    for sc, bi in ((scale, None), (None, bias), (scale, bias.to(dt))):
        want, held = adapter64(base + (0 if bi is None else bi.double()), x, a, b, slots, sc, dt)
        assert torch.equal(want, held)  # the inner products fit
        assert torch.equal(sp.adapter_linear(x, w, a, b, slots, scale=sc, bias=bi), want.to(dt))
        want = adapter64(y.double(), x, a, b, slots, sc, dt)[0].to(dt)
        assert torch.equal(sp.adapter_add(y, x, a, b, slots, scale=sc), want)
        z = y.clone()
        assert sp.adapter_add(z, x, a, b, slots, scale=sc, out=z) is z and torch.equal(z, want)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,count,rank,k,o,order", [ADAPTERS[i] for i in (1, 4, 7, 9, 11, 12, 17)])
def test_adapter_values(gpu, n, count, rank, k, o, order, dt):
    g = gen(n)
    slots = slots_of(g, n, count, order)
    x, w, a, b = values(g, n, k, dt=dt), values(g, o, k, dt=dt), values(g, count, rank, k, dt=dt), values(g, count, o, rank, dt=dt)
    scale, y = torch.rand(count, generator=g, device=gpu) + 0.5, values(g, n, o, dt=dt)
    a = (a.float() / 64).to(dt)
    zero = torch.zeros((n, o), dtype=torch.float64, device=gpu)
    part = adapter64(zero, x, a, b, slots, scale, dt)[0]
    size = adapter64(zero, x.abs(), a.abs(), b.abs(), slots, scale, dt)[0]
    # |b| |scale a x|: what the inner product's rounding is relative to
    inner = zero.clone()
    for s in range(count):
        r = (slots == s).nonzero().squeeze(1)
        inner[r] = (x[r].double() @ a[s].double().T * float(scale[s])).abs() @ b[s].double().abs().T
    eps = torch.finfo(dt).eps
    for got, base, bs in ((sp.adapter_linear(x, w, a, b, slots, scale=scale), x.double() @ w.double().T, x.double().abs() @ w.double().abs().T),
                          (sp.adapter_add(y, x, a, b, slots, scale=scale), y.double(), y.double().abs())):
        want = base + part
        tol = (k + rank + 2) * 2.0 ** -23 * (bs + 2 * size) + eps / 2 * 1.01 * inner + rank * 2.0 ** -24 * b.abs().max().double()
        tol = tol + eps / 2 * (want.abs() + tol) + 2.0 ** -24
        assert ((got.double() - want).abs() <= tol).all(), float(((got.double() - want).abs() / tol).max())


def test_adapter_not_finite(gpu):
    """NaN and infinities in a row, in an adapter that a row beside it does not have, and in rows without an adapter."""
    g, dt = gen(9), torch.bfloat16
    for n in (12, 300):
        x, w, a, b = ints(g, n, 64), ints(g, 72, 64), ints(g, 3, 16, 64), ints(g, 3, 72, 16)
        slots = (torch.arange(n, device=gpu) % 4 - 1).int()
        y = ints(g, n, 72)
        a[1, 5, 7], b[2, 4, 3] = float("nan"), float("inf")
        x[0, 0] = float("inf")  # no adapter
        for got in (sp.adapter_linear(x, w, a, b, slots), sp.adapter_add(y, x, a, b, slots)):
            fine = torch.isfinite(got)
            want = torch.ones((n, 72), dtype=torch.bool, device=gpu)
            want[slots == 1] = False
            want[slots == 2, 4] = False
            assert torch.equal(fine[1:], want[1:])
        assert torch.isfinite(got[0]).all()  # adapter_add's y of a row without an adapter does not read x


def test_more_tiles_than_a_launch_holds(gpu):
    """So many groups of a row each by so many channels that a workgroup for each would be past 2^32 threads."""
    g, dt, n, k, o = gen(12), torch.bfloat16, 8192, 8, 32776
    x, w = ints(g, n, k, dt=dt, most=1), torch.zeros((n, o, k), dtype=dt, device=gpu)
    w[:, -40:], w[:, :40] = ints(g, n, 40, k, dt=dt, most=1), ints(g, n, 40, k, dt=dt, most=1)
    y = sp.group_linear(x, w, torch.arange(1, n + 1, dtype=torch.int32, device=gpu))
    for part in (slice(0, 40), slice(o - 40, o)):
        assert torch.equal(y[:, part], (w[:, part].float() * x[:, None].float()).sum(-1).to(dt))
    assert not y[:, 40:-40].any()


def test_as_many_rows_as_there_may_be(gpu):
    """Row numbers up to the largest of 31 bits, in the last stage of the longest sum among them."""
    dt, n, last = torch.float16, 2 ** 31 - 1, 70
    g = gen(13)
    x, dy = (torch.zeros((n, 8), dtype=dt, device=gpu) for _ in range(2))  # 34 GB each
    x[-last:], dy[-last:] = ints(g, last, 8, dt=dt), ints(g, last, 8, dt=dt)
    w, ends = ints(g, 2, 8, 8, dt=dt), torch.tensor([n - 3, n], dtype=torch.int32, device=gpu)
    for e, which in ((ends, w), (ends[1:], w[:1])):
        tail = (e - (n - last)).clamp(min=0)
        assert torch.equal(sp.group_linear_dw(dy, x, e), dw64(dy[-last:], x[-last:], tail)[0].to(dt))
        y = sp.group_linear(x, which, e)
        assert torch.equal(y[-last:], forward64(x[-last:], which, tail, None, y[-last:]).to(dt))
        del y
        dx = sp.group_linear_dx(dy, which, e)
        assert torch.equal(dx[-last:], dx64(dy[-last:], which, tail, x[-last:]).to(dt))
        del dx
    del x, dy
    torch.cuda.empty_cache()


def test_adapters_of_as_many_rows_as_there_may_be(gpu):
    dt, n, last = torch.float16, 1 << 27, 70
    g = gen(15)
    x = torch.zeros((n, 8), dtype=dt, device=gpu)
    x[-last:] = ints(g, last, 8, dt=dt, most=1)
    slots = torch.zeros(n, dtype=torch.int32, device=gpu)
    for rank in (8, 72):
        a, b, w = ints(g, 2, rank, 8, dt=dt, most=1), ints(g, 2, 8, rank, dt=dt, most=1), ints(g, 8, 8, dt=dt, most=1)
        low = x[-last:].double() @ a[0].double().T @ b[0].double().T
        y = sp.adapter_add(x, x, a, b, slots)
        assert torch.equal(y[-last:], (x[-last:].double() + low).to(dt)) and not y[-n:-last].any()
        y = sp.adapter_linear(x, w, a, b, slots)
        assert torch.equal(y[-last:], (x[-last:].double() @ w.double().T + low).to(dt)) and not y[-n:-last].any()


def test_adapter_past_four_gigabytes(gpu):
    """Offsets past 32 bits: in the rows, the result and the adapters."""
    g, dt = gen(4), torch.bfloat16
    n, k, o = (1 << 20) + 70, 2112, 2056
    x, y = torch.zeros((n, k), dtype=dt, device=gpu), torch.zeros((n, o), dtype=dt, device=gpu)
    x[-90:], y[-90:] = ints(g, 90, k, most=1), ints(g, 90, o)
    x[:, 40:] = 0
    a, b, slots = ints(g, 2, 8, k, most=1), ints(g, 2, o, 8, most=1), (torch.arange(n, device=gpu) % 2).int()
    want = adapter64(y[-90:].double(), x[-90:], a, b, slots[-90:], None, dt)[0].to(dt)
    assert torch.equal(sp.adapter_add(y, x, a, b, slots, out=y)[-90:], want)
    w = ints(g, 16, k, most=1)
    assert torch.equal(sp.adapter_linear(x, w, a, b[:, :16].contiguous(), slots)[-90:],
                       adapter64(x[-90:].double() @ w.double().T, x[-90:], a, b[:, :16], slots[-90:], None, dt)[0].to(dt))
    del x, y
    count, k = 1025, 16384
    a = torch.zeros((count, 256, k), dtype=dt, device=gpu)  # 8 MB each
    a[1024] = ints(g, 256, k, most=1)
    b = ints(g, count, 16, 256, most=1)
    for n in (3, 200):
        x = ints(g, n, k, most=1) * (torch.rand((n, k), generator=g, device=gpu) < 0.002).to(dt)
        slots, y = torch.full((n,), 1024, dtype=torch.int32, device=gpu), ints(g, n, 16)
        assert torch.equal(sp.adapter_add(y, x, a, b, slots),
                           adapter64(y.double(), x, a[1024:], b[1024:], torch.zeros_like(slots), None, dt)[0].to(dt))


# ---- together, and as the framework runs them --------------------------------------------------------------------


def silu64(v):
    return v * torch.sigmoid(v)


def test_experts_block_trains(gpu):
    """x + W2[g] silu(W1[g] x + b1[g]) forward and backward from the operators, against autograd in 64 bits."""
    g, dt = gen(21), torch.bfloat16
    lengths, c = [130, 0, 301, 77, 4], 256
    n, ends = sum(lengths), ends_of(lengths)
    x, dy = values(g, n, c, dt=dt), values(g, n, c, dt=dt)
    w1, w2, b1 = (values(g, 5, 4 * c, c) / 16).to(dt), (values(g, 5, c, 4 * c) / 32).to(dt), values(g, 5, 4 * c, dt=dt)
    z = sp.group_linear(x, w1, ends, bias=b1)
    h = torch.nn.functional.silu(z)
    y = x + sp.group_linear(h, w2, ends)
    dh, dw2 = sp.group_linear_dx(dy, w2, ends), sp.group_linear_dw(dy, h, ends, out_dtype=torch.float32)
    sig = torch.sigmoid(z.float())
    dz = (dh.float() * sig * (1 + z.float() * (1 - sig))).to(dt)
    dx = dy + sp.group_linear_dx(dz, w1, ends)
    dw1, db1 = sp.group_linear_dw(dz, x, ends, out_dtype=torch.float32, bias=True)
    leaves = [t.double().requires_grad_() for t in (x, w1, b1, w2)]
    X, W1, B1, W2 = leaves
    parts = [X[s] + silu64(X[s] @ W1[i].T + B1[i]) @ W2[i].T for i, s in enumerate(spans(ends, n))]
    Y = torch.cat(parts)
    Y.backward(dy.double())
    # each result passes up to four roundings of 2^-8 relative 2-norm at most; they add as their squares or below, 4 x 2^-8 in any case
    for got, want in ((y, Y), (dx, X.grad), (dw1, W1.grad), (db1, B1.grad), (dw2, W2.grad)):
        want = want.detach()
        assert (got.double() - want).norm() <= 4 * 2.0 ** -8 * want.norm()
    assert not dw1[1].any() and not db1[1].any() and not dw2[1].any()


def test_adapters_beside_a_4_bit_layer(gpu):
    """mx_linear's projection with adapters added in place, and the same adapters as groups of rows sorted by request."""
    g, dt, n, k, o = gen(22), torch.float16, 90, 512, 1024
    x, w = values(g, n, k, dt=dt), sp.mx_quantize(values(g, o, k, dt=torch.float32) / 16)
    a, b = (values(g, 4, 16, k) / 32).to(dt), (values(g, 4, o, 16) / 4).to(dt)
    slots = torch.arange(n, device=gpu).mul(4).div(n, rounding_mode="floor").int()
    y = sp.mx_linear(x, w)
    want = adapter64(y.double(), x, a, b, slots, None, dt)[0]
    got = sp.adapter_add(y, x, a, b, slots, out=y)
    assert (got.double() - want).norm() <= 2 * 2.0 ** -11 * want.norm()
    ends = torch.bincount(slots, minlength=4).cumsum(0).int()
    again = sp.mx_linear(x, w, residual=sp.group_linear(sp.group_linear(x, a, ends), b, ends))
    assert (again.double() - want).norm() <= 4 * 2.0 ** -11 * want.norm()


def calls(g, dt=torch.bfloat16):
    lengths = [60, 3, 0, 200]
    n, ends = sum(lengths), ends_of(lengths)
    x, w, dy = values(g, n, 264, dt=dt), values(g, 4, 136, 264, dt=dt), values(g, n, 136, dt=dt)
    a, b, w1 = values(g, 3, 16, 264, dt=dt), values(g, 3, 136, 16, dt=dt), values(g, 136, 264, dt=dt)
    slots = torch.randint(-1, 3, (n,), generator=g, device="cuda").int()
    few = torch.tensor([2, 3, 3, 9], dtype=torch.int32, device="cuda")
    return [lambda: sp.group_linear(x, w, ends), lambda: sp.group_linear(x[:9], w, few), lambda: sp.group_linear_dx(dy, w, ends),
            lambda: sp.group_linear_dw(dy, x, ends, out_dtype=torch.float32), lambda: sp.adapter_linear(x, w1, a, b, slots),
            lambda: sp.adapter_linear(x[:5], w1, a, b, slots[:5]), lambda: sp.adapter_add(dy, x, a, b, slots),
            lambda: sp.adapter_add(dy[:5], x[:5], a, b, slots[:5])]


def test_same_bits_every_time(gpu):
    todo = calls(gen(31))
    first = [c() for c in todo]
    for _ in range(3):
        for c, want in zip(todo, first):
            assert torch.equal(c(), want)


def test_graph_replays(gpu):
    """Captured calls, replayed in turn with eager work between, give the eager results on every replay; other groups and slots in
    the same buffers are those of the replay."""
    todo = calls(gen(32))
    want = [c() for c in todo]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    try:
        for c in todo:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                sp.set_stream(torch.cuda.current_stream())
                outs.append(c())
            graphs.append(graph)
    finally:
        torch.cuda.synchronize()
        sp.set_stream(torch.cuda.current_stream())
    for _ in range(4):
        for out in outs:
            out.fill_(3.0)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, ref in zip(outs, want):
            assert torch.equal(out, ref)
        for c, ref in zip(todo, want):
            assert torch.equal(c(), ref)


def test_graph_follows_ends_and_slots(gpu):
    g, dt = gen(33), torch.float16
    x, w, a, b = ints(g, 300, 64, dt=dt), ints(g, 3, 72, 64, dt=dt), ints(g, 3, 8, 64, most=1, dt=dt), ints(g, 3, 72, 8, most=1, dt=dt)
    ends, slots = ends_of([100, 100, 100]), slots_of(g, 300, 3, "mixed")
    y = ints(g, 300, 72, dt=dt)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=s):
            sp.set_stream(torch.cuda.current_stream())
            out, add = sp.group_linear(x, w, ends), sp.adapter_add(y, x, a, b, slots)
    finally:
        torch.cuda.synchronize()
        sp.set_stream(torch.cuda.current_stream())
    for lengths in ([300, 0, 0], [1, 298, 1], [0, 0, 300], [17, 200, 83]):
        ends.copy_(ends_of(lengths))
        slots.copy_(slots_of(g, 300, 3, "mixed"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, forward64(x, w, ends, None, out).to(dt))
        assert torch.equal(add, adapter64(y.double(), x, a, b, slots, None, dt)[0].to(dt))


def test_other_streams(gpu):
    """The library on another stream than torch's current one; and both on it."""
    todo = calls(gen(34))
    want = [c() for c in todo]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    try:
        sp.set_stream(s)
        for _ in range(2):
            got = [c() for c in todo]
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
        with torch.cuda.stream(s):
            got = [c() for c in todo]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    finally:
        torch.cuda.synchronize()
        sp.set_stream(torch.cuda.current_stream())


def test_nothing_to_do(gpu):
    dt = torch.float16
    x, w, ends = torch.empty((0, 64), dtype=dt, device=gpu), torch.ones((3, 72, 64), dtype=dt, device=gpu), torch.zeros(3, dtype=torch.int32, device=gpu)
    dy = torch.empty((0, 72), dtype=dt, device=gpu)
    assert sp.group_linear(x, w, ends).shape == (0, 72) and sp.group_linear_dx(dy, w, ends).shape == (0, 64)
    dw, db = sp.group_linear_dw(dy, x, ends, out=torch.ones_like(w), bias=True)
    assert not dw.any() and not db.any()
    a, b, slots = torch.ones((2, 8, 64), dtype=dt, device=gpu), torch.ones((2, 72, 8), dtype=dt, device=gpu), ends[:0]
    assert sp.adapter_linear(x, w[0], a, b, slots).shape == (0, 72) and sp.adapter_add(dy, x, a, b, slots).shape == (0, 72)


def test_refusals_on_the_device(gpu):
    dt = torch.float16
    x, w, ends = torch.ones((8, 64), dtype=dt, device=gpu), torch.ones((3, 72, 64), dtype=dt, device=gpu), torch.tensor([2, 4, 8], dtype=torch.int32, device=gpu)
    a, b, slots = torch.ones((2, 8, 64), dtype=dt, device=gpu), torch.ones((2, 72, 8), dtype=dt, device=gpu), torch.zeros(8, dtype=torch.int32, device=gpu)
    for call in (lambda: sp.group_linear(x, w, ends.cpu()), lambda: sp.group_linear(x.cpu(), w, ends), lambda: sp.group_linear(x, w, ends.long()),
                 lambda: sp.group_linear(torch.ones((8, 128), dtype=dt, device=gpu)[:, ::2], w, ends),
                 lambda: sp.group_linear(x, w, ends, out=torch.empty((8, 71), dtype=dt, device=gpu)),
                 lambda: sp.group_linear(x, w.bfloat16(), ends), lambda: sp.group_linear(x, w, ends[:2]),
                 lambda: sp.adapter_add(x, x, a, b, slots), lambda: sp.adapter_linear(x, w[0], a, b, slots[:4]),
                 lambda: sp.adapter_linear(x, w[0], a, b.transpose(0, 1), slots)):
        with pytest.raises(ValueError):
            call()
    room = torch.ones(1 << 14, dtype=dt, device=gpu)
    with pytest.raises(RuntimeError, match="overlap"):
        sp.group_linear(room[:512].view(8, 64), w, ends, out=room[256:256 + 576].view(8, 72))
    with pytest.raises(RuntimeError, match="aligned"):
        sp.group_linear(room[1:513].view(8, 64), w, ends)
    with pytest.raises(RuntimeError, match="apart"):
        sp.adapter_add(room[:576].view(8, 72), x, a, b, slots, out=room[64:640].view(8, 72))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,k,o", [(2100, 16384, 128), (1990, 16136, 8), (4100, 128, 16384), (2500, 104, 16264), (2100, 16640, 128), (2100, 16128, 128)])
def test_gradient_of_64_tiles_in_parts(gpu, n, k, o, dt):
    """A result of one tile across and some 64 along, which is as many as are shared out by XCD and few enough for parts of the depth."""
    g = gen(n + k)
    x, dy, ends = ints(g, n, k, most=2, dt=dt), ints(g, n, o, most=2, dt=dt), ends_of([n])
    dw, db = dw64(dy, x, ends)
    for odt in (None, torch.float32):
        got, gb = sp.group_linear_dw(dy, x, ends, out_dtype=odt, bias=True)
        assert torch.equal(got, dw.to(got.dtype)) and torch.equal(gb, db.to(got.dtype))


# x, a, b, w, y and scale times these: as they come; A x past fp16's largest value, B small; scaled A x below fp16's least normal one, B large;
# a scale past fp16's largest value
RANGES = {"one": (1, 2.0 ** -6, 1, 1, 1, 1), "large": (256, 64, 2.0 ** -16, 2.0 ** -13, 1, 1), "small": (1, 2.0 ** -6, 2.0 ** 12, 2.0 ** -16, 2.0 ** -10, 2.0 ** -22),
          "scale": (1, 2.0 ** -6, 2.0 ** -18, 1, 1, 2.0 ** 18)}


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("kind", list(RANGES))
@pytest.mark.parametrize("n,count,rank,k,o,order", [ADAPTERS[i] for i in (1, 3, 4, 7, 9, 10, 11, 12, 17, 22)])
def test_adapter_inner_product(gpu, n, count, rank, k, o, order, kind, dt):
    """The inner product, a sum in fp32, keeps fp32's range, and the second product takes it to 2^-15 of each value (bf16), 2^-22 of
    each and 2^-39 of the row's largest (fp16): its high half is cut to 8 (rounded to 11) bits, its low half rounded to as many, in fp16
    both of values whose largest is in [2^14, 2^15) and whose least step is 2^-24."""
    g = gen(n + rank)
    px, pa, pb, pw, py, ps = RANGES[kind]
    slots = slots_of(g, n, count, order)

    def drawn(factor, *shape):
        return (torch.randn(shape, generator=g, device=gpu) * factor).to(dt)

    x, w, a, b, y = drawn(px, n, k), drawn(pw, o, k), drawn(pa, count, rank, k), drawn(pb, count, o, rank), drawn(py, n, o)
    scale = (torch.rand(count, generator=g, device=gpu) + 0.5) * ps
    zero = torch.zeros((n, o), dtype=torch.float64, device=gpu)
    part = adapter64(zero, x, a, b, slots, scale, dt)[0]
    size = adapter64(zero, x.abs(), a.abs(), b.abs(), slots, scale, dt)[0]
    inner, most = zero.clone(), zero.clone()
    for s in range(count):
        r = (slots == s).nonzero().squeeze(1)
        h = (x[r].double() @ a[s].double().T * float(scale[s])).abs()
        inner[r] = h @ b[s].double().abs().T
        most[r] = h.amax(1, keepdim=True) * b[s].double().abs().sum(1)
    held = 2.0 ** -15 * inner if dt == torch.bfloat16 else 2.0 ** -22 * inner + 2.0 ** -39 * most
    t = torch.finfo(dt)
    for got, base, bs in ((sp.adapter_linear(x, w, a, b, slots, scale=scale), x.double() @ w.double().T, x.double().abs() @ w.double().abs().T),
                          (sp.adapter_add(y, x, a, b, slots, scale=scale), y.double(), y.double().abs())):
        want = base + part
        assert want.abs().max() < t.max / 2
        tol = (k + 2 * rank + 4) * 2.0 ** -23 * (bs + size) + 1.01 * held
        tol = tol + t.eps / 2 * (want.abs() + tol) + t.tiny * t.eps / 2
        assert ((got.double() - want).abs() <= tol).all(), float(((got.double() - want).abs() / tol).max())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,count,rank,k,o,order", [(1, 2, 256, 136, 72, "one"), (2, 2, 40, 520, 264, "mixed"), (5, 3, 8, 72, 136, "mixed"), (7, 3, 24, 136, 72, "mixed")]
                         + [ADAPTERS[i] for i in (7, 9, 11, 12, 17, 22)])
def test_adapter_workspaces(gpu, n, count, rank, k, o, order, dt):
    """The least workspace, in which the rows go in parts, ones between, and one that holds them all: the exact result each time, and
    nothing written behind it."""
    import ctypes

    g = gen(n + k + rank)
    slots = slots_of(g, n, count, order)
    x = ints(g, n, k, most=1, dt=dt) * (torch.rand((n, k), generator=g, device=gpu) < 20.0 / k).to(dt)
    w, a, b, y = ints(g, o, k, most=2, dt=dt), ints(g, count, rank, k, most=2, dt=dt), ints(g, count, o, rank, most=1, dt=dt), ints(g, n, o, most=20, dt=dt)
    part = adapter64(torch.zeros((n, o), dtype=torch.float64, device=gpu), x, a, b, slots, None, dt)[0]
    lib, least, code = sp.load_library(), ctypes.c_int64(), 2 if dt == torch.bfloat16 else 1

    def p(t):
        return ctypes.c_void_p(t.data_ptr())

    for depth, want in ((k, x.double() @ w.double().T + part), (0, y.double() + part)):
        assert lib.spc_adapter_workspace(n, rank, depth, o, ctypes.byref(least)) == 0
        for size in (least.value, least.value + 8, least.value + n * rank, least.value + 3 * n * rank):
            out, ws = torch.full_like(y, 7.0), torch.full((size + 256,), 255, dtype=torch.uint8, device=gpu)
            if depth:
                rc = lib.spc_adapter_linear(p(x), p(w), p(a), p(b), p(slots), None, None, code, 0, n, count, rank, k, o, p(out), p(ws), size)
            else:
                rc = lib.spc_adapter_add(p(y), p(x), p(a), p(b), p(slots), None, code, n, count, rank, k, o, p(out), p(ws), size)
            assert rc == 0, lib.spc_last_error()
            assert torch.equal(out, want.to(dt)) and (ws[size:] == 255).all()


# ---- sums in parts: a second kernel adds them from a workspace -----------------------------------------------------


def in_parts(product, n, groups, k, o):
    return sp._workspace_bytes("spc_group_linear_workspace", product, n, groups, k, o) > 0


def calls_in_parts(g, dt=torch.bfloat16):
    def v(*shape):
        return values(g, *shape, dt=dt)

    one, two, some, long, deep = ends_of([600]), ends_of([370, 0, 230]), ends_of([700, 0, 900]), ends_of([4100]), ends_of([3000, 0, 3300])
    assert in_parts(sp.GROUP_FORWARD, 600, 1, 4104, 40) and in_parts(sp.GROUP_FORWARD, 1600, 3, 4104, 40) and in_parts(sp.GROUP_DX, 600, 3, 136, 2056)
    assert in_parts(sp.GROUP_DW, 4100, 1, 72, 136) and in_parts(sp.GROUP_DW, 6300, 3, 72, 136) and in_parts(sp.GROUP_FORWARD, 600, 1, 4104, 136)
    x, w1, w3, b1 = v(1600, 4104), v(1, 40, 4104), v(3, 40, 4104), v(1, 40)
    dy, w, xl, dyl = v(600, 2056), v(3, 2056, 136), v(6300, 72), v(6300, 136)
    wa, a, b, slots = v(136, 4104), v(3, 16, 4104), v(3, 136, 16), slots_of(g, 600, 3, "mixed")
    return [lambda: sp.group_linear(x[:600], w1, one, bias=b1), lambda: sp.group_linear(x, w3, some), lambda: sp.group_linear_dx(dy, w, two),
            lambda: sp.group_linear_dw(dyl[:4100], xl[:4100], long, out_dtype=torch.float32, bias=True), lambda: sp.group_linear_dw(dyl, xl, deep),
            lambda: sp.adapter_linear(x[:600], wa, a, b, slots)]


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want)) if isinstance(got, tuple) else torch.equal(got, want)


def test_parts_same_bits_every_time(gpu):
    todo = calls_in_parts(gen(41))
    first = [c() for c in todo]
    for _ in range(3):
        junk = torch.full((1 << 25,), 255, dtype=torch.uint8, device=gpu)  # NaN in what the next workspaces may hold
        del junk
        assert all(same(c(), want) for c, want in zip(todo, first))


def captured(todo):
    """Each call in a graph of its own, and its result."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    try:
        for c in todo:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                sp.set_stream(torch.cuda.current_stream())
                outs.append(c())
            graphs.append(graph)
    finally:
        torch.cuda.synchronize()
        sp.set_stream(torch.cuda.current_stream())
    return graphs, outs


def test_parts_in_graphs(gpu):
    """Two graphs of each call, replayed in turn with the call itself between."""
    todo = calls_in_parts(gen(42))
    want = [c() for c in todo]
    graphs, outs = captured(todo + todo)
    for _ in range(4):
        for out in outs:
            for t in out if isinstance(out, tuple) else (out,):
                t.fill_(3.0)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(same(out, ref) for out, ref in zip(outs, want + want))
        assert all(same(c(), ref) for c, ref in zip(todo, want))


def test_parts_on_other_streams(gpu):
    todo = calls_in_parts(gen(43))
    want = [c() for c in todo]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    try:
        sp.set_stream(s)
        for _ in range(2):
            got = [c() for c in todo]
            torch.cuda.synchronize()
            assert all(same(a, b) for a, b in zip(got, want))
        with torch.cuda.stream(s):
            got = [c() for c in todo]
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(got, want))
    finally:
        torch.cuda.synchronize()
        sp.set_stream(torch.cuda.current_stream())


@pytest.mark.parametrize("dt", TYPES)
def test_parts_follow_ends(gpu, dt):
    """Captured calls in parts with other ends in the buffer at their replay, also ones outside the rows: the results of those; rows of no
    group stay."""
    g, n = gen(44), 1600
    x, w = ints(g, n, 4104, dt=dt, most=1), ints(g, 3, 40, 4104, dt=dt, most=1)
    dy, v = ints(g, 600, 2056, dt=dt, most=1), ints(g, 3, 2056, 136, dt=dt, most=1)
    xl, dyl = ints(g, 6300, 72, dt=dt, most=1), ints(g, 6300, 136, dt=dt, most=1)
    ends = [ends_of([t // 3] * 3) for t in (n, 600, 6300)]
    y, dx, dw = torch.zeros((n, 40), dtype=dt, device=gpu), torch.zeros((600, 136), dtype=dt, device=gpu), torch.zeros((3, 136, 72), device=gpu)
    todo = [lambda: sp.group_linear(x, w, ends[0], out=y), lambda: sp.group_linear_dx(dy, v, ends[1], out=dx), lambda: sp.group_linear_dw(dyl, xl, ends[2], out=dw)]
    graphs, _ = captured(todo)
    for now in ([1.0, 1.0, 1.0], [0, 0, 0.99], [0.03, 0.4, 0.5], [-0.5, 0.1, 9.0], [0, 0, 0], [-2.0, -1.0, -0.1], [0.4, 0.5, 1e9]):
        for e, t in zip(ends, (n, 600, 6300)):
            e.copy_(torch.tensor([min(int(f * t), 2 ** 31 - 1) for f in now], dtype=torch.int32))
        for run in ([graph.replay for graph in graphs], todo):
            for t, old in ((y, 5.0), (dx, 6.0), (dw, 7.0)):
                t.fill_(old)
            want = forward64(x, w, ends[0], None, y).to(dt), dx64(dy, v, ends[1], dx).to(dt), dw64(dyl, xl, ends[2])[0].float()
            for r in run:
                r()
            torch.cuda.synchronize()
            assert same((y, dx, dw), want)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n,rank", [(3, 8), (1, 32), (12, 40), (40, 256), (300, 72), (700, 16), (2600, 64)])
def test_adapter_infinities(gpu, n, rank, dt):
    """Infinities and NaN in x, a and b come out as the definition has them: infinities of the right sign, NaN where they meet a zero or each
    other, and finite values elsewhere."""
    g, k, o = gen(50 + n), 64, 200
    x, w, y = ints(g, n, k, dt=dt, most=1), ints(g, o, k, dt=dt, most=1), ints(g, n, o, dt=dt)
    a, b, slots = ints(g, 3, rank, k, dt=dt, most=1), ints(g, 3, o, rank, dt=dt, most=1), slots_of(g, n, 3, "mixed")
    slots[0] = 1
    x = x * (torch.rand((n, k), generator=g, device=gpu) < 0.3).to(dt)
    a[1, 3, 5], b[1, 7, 2], b[1, 9, :2] = float("inf"), float("-inf"), torch.tensor([float("inf"), float("nan")])
    b[2, 11, :2] = float("inf")
    x[n // 2, 4] = float("-inf")
    for got, base in ((sp.adapter_add(y, x, a, b, slots), y.double()), (sp.adapter_linear(x, w, a, b, slots), x.double() @ w.double().T)):
        want = adapter64(base, x, a, b, slots, None, dt)[0].to(dt)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def test_adapters_in_parts_of_many_rows(gpu):
    """So many inner products that room for all of them is not taken: the rows go in parts."""
    g, dt, n, rank = gen(60), torch.float16, 360011, 256
    x, w = ints(g, n, 16, dt=dt, most=1), ints(g, 24, 16, dt=dt, most=1)
    a, b, slots, y = ints(g, 3, rank, 16, dt=dt, most=1), ints(g, 3, 24, rank, dt=dt, most=1), slots_of(g, n, 3, "runs"), ints(g, n, 24, dt=dt)
    assert 3 * n * rank > 1 << 28
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    z = sp.adapter_add(y, x, a, b, slots)
    assert torch.cuda.max_memory_allocated() - before <= 2 * n * rank + z.nbytes + (1 << 20)
    v = sp.adapter_linear(x, w, a, b, slots)
    part = adapter64(torch.zeros((n, 24), dtype=torch.float64, device=gpu), x, a, b, slots, None, dt)[0]
    assert torch.equal(z, (y.double() + part).to(dt)) and torch.equal(v, (x.double() @ w.double().T + part).to(dt))
