"""Microscaled operators on the GPU against their definitions in 64 bits (mx_reference).

Quantisation is exact arithmetic (a power-of-two scale, one rounding), so codes and scales have to be equal. A norm's
fp32 result is off by at most TOL = 2^-15 of the magnitudes that enter it: up to 16384 / 256 = 64 additions in a lane, 8
across lanes and 4 across wavefronts for a sum, twice for a LayerNorm, at 2^-24 each, give 2^-16; the reciprocal root,
its three multiplications and the fused additions a few 2^-23 more. Its elements are then off by that and half an
element's step. Products: operands with few bits whose sums all fit in 24 are compared bit for bit; others by the
worst case of K additions of 2^-23 each, and the output's rounding of finfo.eps / 2. Of eight neighbouring e4m3 products,
which the matrix unit adds at once, it drops what is below 2^-13 of the largest: at most 7 * 2^-13 of it for each group (256 * 1
keeps 2^-5 * 1 beside it and loses 2^-6 * 1; e2m1 products all lie within 13 bits).
"""
import pytest
import torch

import mx_reference as R
import spconv_amd as sp

pytestmark = pytest.mark.gpu
TOL = 2.0 ** -15
F = {sp.MX_E4M3: "e4m3", sp.MX_E2M1: "e2m1"}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def features(n, k, dt, seed):
    g = gen(seed)
    spread = torch.exp(torch.randn(k, generator=g)) * torch.where(torch.rand(k, generator=g) < 0.05, 20.0, 1.0)
    return (torch.randn((n, k), generator=g) * spread).to(dt)


def ragged(q):
    """q's used scale bytes (int64)."""
    return q.scales[:, :q.shape[1] // 32].long()


def same(q, x, fmt):
    el, byte = R.quantize(x, fmt)
    assert torch.equal(ragged(q), byte)
    assert torch.equal(R.elements(q.codes, fmt), el)
    assert int(q.scales[:, q.shape[1] // 32:].sum()) == 0


@pytest.mark.parametrize("fmt", [sp.MX_E4M3, sp.MX_E2M1])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,k", [(1, 32), (3, 96), (1, 4096), (257, 512), (1000, 544), (33, 2080)])
def test_quantize(gpu, fmt, dt, n, k):
    x = features(n, k, dt, n + k).to(gpu)
    q = sp.mx_quantize(x, fmt)
    assert q.shape == (n, k) and q.fmt == fmt
    same(q, x, fmt)
    v = R.values(*R.quantize(x, fmt))
    for odt in (torch.float32, torch.bfloat16, torch.float16):
        assert torch.equal(sp.mx_dequantize(q, odt), v.to(odt))


@pytest.mark.parametrize("fmt", [sp.MX_E4M3, sp.MX_E2M1])
def test_quantize_borders(gpu, fmt):
    """Halves between elements, the border between two scales, the smallest and largest floats, signed zeros, blocks of zeros."""
    one = torch.linspace(0, 8, 1025, dtype=torch.float64)[:1024]
    rows = [one, -one, one * 2.0 ** -126, one * 2.0 ** -149, one * 2.0 ** 120, torch.zeros(1024, dtype=torch.float64)]
    tops = []
    for m in (255, 256, 447, 448, 449, 463, 464, 464.0001, 465, 511, 5.99, 6, 6.0001, 6.999999, 7, 7.5, 3.4e38, 1e-45):
        r = torch.zeros(32, dtype=torch.float64)
        r[:] = torch.linspace(-1, 1, 32, dtype=torch.float64) * m
        r[7] = m
        tops.append(r)
    rows.append(torch.cat(tops + [torch.zeros(1024 - 32 * len(tops), dtype=torch.float64)]))
    x = torch.stack(rows).float().to(gpu)
    q = sp.mx_quantize(x, fmt)
    same(q, x, fmt)
    assert torch.equal(sp.mx_dequantize(q, torch.float32), R.values(*R.quantize(x, fmt)).float())


@pytest.mark.parametrize("fmt", [sp.MX_E4M3, sp.MX_E2M1])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
def test_quantize_not_finite(gpu, fmt, dt):
    """A block with an infinity or NaN has scale 255, zero elements and reads as NaN; its neighbours are untouched."""
    x = features(5, 160, dt, 3)
    x[1, 40] = float("inf")
    x[2, 0] = float("-inf")
    x[3, 159] = float("nan")
    q = sp.mx_quantize(x.to(gpu), fmt)
    same(q, x.to(gpu), fmt)
    bad = torch.zeros((5, 5), dtype=torch.bool)
    bad[1, 1] = bad[2, 0] = bad[3, 4] = True
    v = sp.mx_dequantize(q, torch.float32).cpu().view(5, 5, 32)
    assert torch.equal(v.isnan().all(2), bad) and torch.equal(v.isnan().any(2), bad)
    assert int(q.codes.view(5, 5, -1)[bad.to(gpu)].sum()) == 0


def test_quantize_into_given_buffers(gpu):
    """Rows behind the given ones stay as they were; a view of later rows is a valid buffer."""
    x = features(11, 96, torch.float16, 1).to(gpu)
    codes = torch.full((16, 48), 9, dtype=torch.uint8, device=gpu)
    scales = torch.full((16, 16), 9, dtype=torch.uint8, device=gpu)
    q = sp.MxTensor(codes[2:13], scales[2:13], 96, sp.MX_E2M1)
    assert sp.mx_quantize(x, sp.MX_E2M1, out=q) is q
    same(q, x, sp.MX_E2M1)
    for t in (codes, scales):
        assert bool((t[:2] == 9).all()) and bool((t[13:] == 9).all())


def norm64(t, kind, gamma, beta, eps):
    """The norm of float64 rows, and what its fp32 computation may be off by."""
    mean = t.mean(1, keepdim=True) if kind == sp.NORM_LAYER else torch.zeros_like(t[:, :1])
    rstd = 1 / torch.sqrt((t - mean).square().mean(1, keepdim=True) + eps)
    g = 1.0 if gamma is None else gamma.double()
    y = (t - mean) * rstd * g
    off = TOL * (t.abs() + (t.abs().mean(1, keepdim=True) if kind == sp.NORM_LAYER else 0)) * rstd * (1.0 if gamma is None else g.abs())
    if beta is not None:
        y = y + beta.double()
        off = off + 2.0 ** -22 * beta.double().abs()
    return y, off


def near(q, y, off, fmt):
    """q holds y, computed within off and then quantised."""
    n, k = y.shape
    byte = ragged(q)
    top, slack = y.view(n, -1, 32).abs().amax(2), off.view(n, -1, 32).amax(2)
    assert bool((byte >= R.scale_bytes((top - slack).clamp(min=0), fmt)).all()) and bool((byte <= R.scale_bytes(top + slack, fmt)).all())
    s = R.scale_values(byte).repeat_interleave(32, 1)
    err = (R.values(R.elements(q.codes, fmt), byte) - y).abs()
    allowed = R.half_step(y.abs() + off, s, fmt) + off
    assert bool((err <= allowed).all()), float((err / allowed).max())


NORM_C = [32, 64, 96, 128, 160, 256, 352, 512, 544, 1024, 1056, 2048, 2080, 4096, 4128, 8192, 16384]


@pytest.mark.parametrize("C", NORM_C)
@pytest.mark.parametrize("kind", [sp.NORM_RMS, sp.NORM_LAYER])
def test_add_norm(gpu, C, kind):
    for n, dt, fmt, affine, residual in ((1, torch.bfloat16, sp.MX_E4M3, True, True), (37, torch.float16, sp.MX_E4M3, True, False),
                                         (130, torch.bfloat16, sp.MX_E2M1, False, True)):
        g = gen(C + n)
        x = features(n, C, dt, C + n)
        x[n // 2] = 0.25  # a constant row: no variance
        r = (torch.randn((n, C), generator=g) * 3 + 1).to(dt) if residual else None
        gamma = (torch.rand(C, generator=g) + 0.5).to(dt if n == 37 else torch.float32) if affine else None
        beta = torch.randn(C, generator=g).to(gamma.dtype) if affine and kind == sp.NORM_LAYER else None
        dev = [None if a is None else a.to(gpu) for a in (x, r, gamma, beta)]
        t, q = sp.add_norm_mx(*dev, eps=1e-5, kind=kind, fmt=fmt)
        if residual:
            want = (dev[0].double() + dev[1].double()).to(dt)
            assert torch.equal(t, want)
        else:
            assert t is dev[0] and torch.equal(t.cpu(), x)
        near(q, *norm64(t.double(), kind, dev[2], dev[3], 1e-5), fmt)
        assert int(q.scales[:, C // 32:].sum()) == 0


@pytest.mark.parametrize("C,n", [(64, 70001), (256, 40003), (1024, 9001), (4096, 5003)])
def test_add_norm_many_rows(gpu, C, n):
    """More rows than a launch's workgroups hold at once; the sum over the residual, then over x, gives the same bits."""
    x, r = features(n, C, torch.bfloat16, 1).to(gpu), features(n, C, torch.bfloat16, 2).to(gpu)
    t, q = sp.add_norm_mx(x, r)
    near(q, *norm64(t.double(), sp.NORM_RMS, None, None, 1e-6), sp.MX_E4M3)
    for over in (1, 0):
        a = [x.clone(), r.clone()]
        t2, q2 = sp.add_norm_mx(*a, sum=a[over])
        assert t2.data_ptr() == a[over].data_ptr() and torch.equal(t2, t)
        assert torch.equal(q2.codes, q.codes) and torch.equal(q2.scales, q.scales)


@pytest.mark.parametrize("C", [32, 96, 160, 544, 2080])
def test_add_norm_writes_its_rows_only(gpu, C):
    """Rows before and behind stay as they were; the sum alone (no residual) is a copy of x."""
    x = features(5, C, torch.float16, C).to(gpu)
    buf = sp.MxTensor.empty(9, C, sp.MX_E4M3, gpu)
    buf.codes.fill_(9)
    buf.scales.fill_(9)
    sums = torch.full((9, C), 9.0, dtype=torch.float16, device=gpu)
    q = sp.MxTensor(buf.codes[2:7], buf.scales[2:7], C, sp.MX_E4M3)
    t, got = sp.add_norm_mx(x, sum=sums[2:7], out=q)
    assert got is q and torch.equal(sums[2:7], x) and torch.equal(t, x)
    near(q, *norm64(x.double(), sp.NORM_RMS, None, None, 1e-6), sp.MX_E4M3)
    for b in (buf.codes, buf.scales, sums):
        assert bool((b[:2] == 9).all()) and bool((b[7:] == 9).all())


@pytest.mark.parametrize("C", [32, 96, 224, 416, 480, 832, 1984, 3936, 7872, 16320])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_layer_norm_of_constant_rows(gpu, C, dt):
    """Every value is the mean, so the norm is beta, whatever the row's size: the sums fit in 24 bits (11 of the value, at most 11 of the
    count of eights), and their quotient by C is the value itself."""
    v = torch.tensor([65504.0, -65504.0, 60000.0, 1000.5, -333.25, 2.0 ** -14, 0.0]).to(dt)
    x = v[:, None].expand(-1, C).contiguous().to(gpu)
    for beta in (None, torch.full((C,), -1.5, device=gpu)):
        _, q = sp.add_norm_mx(x, None, torch.full((C,), 2.0, device=gpu), beta, kind=sp.NORM_LAYER)
        assert torch.equal(sp.mx_dequantize(q, torch.float32), torch.full((len(v), C), 0.0 if beta is None else -1.5, device=gpu))


@pytest.mark.parametrize("C", [32, 512, 4096, 16384])
@pytest.mark.parametrize("kind", [sp.NORM_RMS, sp.NORM_LAYER])
def test_add_norm_of_the_largest_values(gpu, C, kind):
    """Up to the documented 2^57 the sum of squares stays below 2^128: 2^14 * (2^57 (1 - 2^-8))^2."""
    top = 2.0 ** 57 * (1 - 2.0 ** -8)
    x = torch.full((3, C), top)
    x[1, ::2] = -top
    x[2] = torch.linspace(-top, top, C)
    x = x.to(torch.bfloat16).to(gpu)
    t, q = sp.add_norm_mx(x, None, kind=kind)
    near(q, *norm64(x.double(), kind, None, None, 1e-6), sp.MX_E4M3)


def test_past_four_gigabytes(gpu):
    """Rows whose offsets pass 32 bits, in and out: the last ones are right."""
    n, k, o = 1100000, 64, 2080
    x = torch.full((n, 2048), 0.5, dtype=torch.bfloat16, device=gpu)  # 4.5 GB
    x[-3:] = features(3, 2048, torch.bfloat16, 1).to(gpu)
    t, q = sp.add_norm_mx(x, x, sum=x)
    assert bool((t[:-3] == 1).all())
    tail = sp.MxTensor(q.codes[-3:], q.scales[-3:], 2048, sp.MX_E4M3)
    near(tail, *norm64(t[-3:].double(), sp.NORM_RMS, None, None, 1e-6), sp.MX_E4M3)
    assert bool((q.codes[:-3] == q.codes[0]).all()) and bool((q.scales[:-3] == q.scales[0]).all())
    q = sp.mx_quantize(x, sp.MX_E2M1)
    want = sp.mx_quantize(x[-5:].contiguous(), sp.MX_E2M1)
    assert torch.equal(q.codes[-5:], want.codes) and torch.equal(q.scales[-5:], want.scales)
    assert torch.equal(sp.mx_dequantize(q)[-5:], sp.mx_dequantize(want))
    del x, t, q, tail
    x = mx(*small_ints(4, k, sp.MX_E2M1, 1, 0, 0), k, sp.MX_E2M1, gpu)
    big = sp.MxTensor(x.codes.repeat(n // 4, 1), x.scales.repeat(n // 4, 1), k, sp.MX_E2M1)
    w = mx(*small_ints(o, k, sp.MX_E2M1, 2, 0, 0), k, sp.MX_E2M1, gpu)
    y = sp.mx_linear(big, w)  # 4.6 GB
    want = (matrix(x) @ matrix(w).T).to(torch.bfloat16)
    assert bool((y.view(n // 4, 4, o) == want).all())


def test_add_norm_edges(gpu):
    """Zero rows, rows whose sum overflows fp16, infinities and NaN. A NaN, or infinities alone, make the row NaN; beside one
    infinity the formula gives t / sqrt(inf) = 0 for the finite values and NaN for it, so its block alone reads as NaN."""
    x = torch.ones((6, 128), dtype=torch.float16)
    x[1] = 0
    x[2] = 60000
    x[3, 5] = float("nan")
    x[4, 70] = float("-inf")
    r = x.clone()
    t, q = sp.add_norm_mx(x.to(gpu), r.to(gpu))
    v = sp.mx_dequantize(q, torch.float32).cpu()
    assert torch.equal(v[0], torch.ones(128)) and torch.equal(v[5], torch.ones(128)) and torch.equal(v[1], torch.zeros(128))
    assert bool(v[2:4].isnan().all())
    assert bool(v[4, 64:96].isnan().all()) and torch.equal(v[4, :64], torch.zeros(64)) and torch.equal(v[4, 96:], torch.zeros(32))


# ---- product ----------------------------------------------------------------------------------------------------


def small_ints(rows, k, fmt, seed, lo, hi):
    """Rows whose elements are integers in [lo, hi] (times 1/2 for e2m1 below 2) and whose scales are 1/2, 1 or 2."""
    g = gen(seed)
    if fmt == sp.MX_E4M3:
        el = torch.randint(lo, hi + 1, (rows, k), generator=g).float()
        codes = el.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        c = torch.randint(0, 16, (rows, k // 2, 2), generator=g, dtype=torch.uint8)
        codes = c[:, :, 0] | c[:, :, 1] << 4
    scales = torch.full((rows, (k + 511) // 512 * 16), 255, dtype=torch.uint8)  # the padding is not to be read
    scales[:, :k // 32] = torch.randint(126, 129, (rows, k // 32), generator=g, dtype=torch.uint8)
    return codes, scales


def mx(codes, scales, k, fmt, dev):
    return sp.MxTensor(codes.to(dev), scales.to(dev), k, fmt)


def matrix(q):
    return R.values(R.elements(q.codes, q.fmt), ragged(q))


SHAPES = [(1, 32, 32), (1, 4096, 96), (2, 64, 32), (5, 160, 288), (15, 512, 128), (16, 544, 4128), (17, 128, 64), (31, 96, 1056),
          (33, 1024, 256), (63, 288, 160), (65, 2080, 96), (77, 4096, 512), (127, 256, 256), (129, 480, 384), (255, 640, 288),
          (257, 1024, 1024), (300, 96, 32), (1803, 1024, 544), (2500, 128, 4096), (5000, 224, 3520)]


@pytest.mark.parametrize("n,k,o", SHAPES)
@pytest.mark.parametrize("fmt", [sp.MX_E4M3, sp.MX_E2M1])
def test_linear_bits(gpu, n, k, o, fmt):
    """Sums of few bits come out exactly, whatever their order: at most 8 * 6 * 4 K in units of 1/8 (e4m3: integers, halves,
    scales from 1/4) or 6 * 6 * 4 K in units of 1/16 (e2m1) stay below 2^24 units for K <= 4096."""
    x = mx(*small_ints(n, k, fmt, n + k, -8, 8), k, fmt, gpu)
    w = mx(*small_ints(o, k, sp.MX_E2M1, o + k, 0, 0), k, sp.MX_E2M1, gpu)
    want = matrix(x) @ matrix(w).T
    got = sp.mx_linear(x, w, out_dtype=torch.float32)
    assert torch.equal(got.double(), want)
    g = gen(o)
    bias = torch.randint(-64, 65, (o,), generator=g).to(torch.float16).to(gpu)
    res = torch.randint(-64, 65, (n, o), generator=g)
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        r = res.to(dt).to(gpu)
        full = want + bias.double() + r.double()
        buf = torch.full((n + 3, o), 7.0, dtype=dt, device=gpu)
        got = sp.mx_linear(x, w, bias, residual=r, out=buf[:n])
        assert torch.equal(got, full.float().to(dt)) and bool((buf[n:] == 7).all())
        got = sp.mx_linear(x, w, bias, residual=r, out=r)  # over the residual
        assert got is r and torch.equal(got, full.float().to(dt))


def tile_is(cus, n, o, fmt, want, **out):
    """The shape runs in this tile: checked on the part whose number of CUs the shapes below are chosen for."""
    if cus == 256:
        assert sp.mx_linear_tile(n, o, fmt, **out) == want


# (n, k, o), the tile (rows, channels) for e2m1, and of e4m3 for 16-bit results (else as e2m1)
FEW = [(24, 160, 16384, (32, 32), None), (60, 1184, 4096, (32, 32), None), (70, 1184, 4096, (48, 32), None),
       (113, 1184, 4096, (64, 32), None), (70, 1184, 8192, (80, 32), None), (90, 1184, 8192, (96, 32), (64, 128)),
       (128, 2080, 8192, (128, 32), (64, 128)), (101, 608, 6144, (128, 32), (64, 128)), (40, 160, 16384, (64, 128), (64, 128))]


@pytest.mark.parametrize("n,k,o,tile,tile16", FEW)
@pytest.mark.parametrize("fmt", [sp.MX_E4M3, sp.MX_E2M1])
def test_linear_bits_of_few_rows(gpu, n, k, o, tile, tile16, fmt):
    """test_linear_bits in every number of row tiles."""
    cus = torch.cuda.get_device_properties(gpu).multi_processor_count
    x = mx(*small_ints(n, k, fmt, n + k, -8, 8), k, fmt, gpu)
    w = mx(*small_ints(o, k, sp.MX_E2M1, o + k, 0, 0), k, sp.MX_E2M1, gpu)
    exact = (matrix(x) @ matrix(w).T).float()
    tile16 = tile16 if tile16 and fmt == sp.MX_E4M3 else tile
    for dt in (torch.float32, torch.bfloat16):
        tile_is(cus, n, o, fmt, tile if dt == torch.float32 else tile16, out_dtype=dt)
        buf = torch.full((n + 3, o), 7.0, dtype=dt, device=gpu)
        got = sp.mx_linear(x, w, out=buf[:n])
        assert torch.equal(got, exact.to(dt)) and bool((buf[n:] == 7).all())
    for ofmt in (sp.MX_E4M3, sp.MX_E2M1):
        tile_is(cus, n, o, fmt, tile, out_fmt=ofmt)
        got, want = sp.mx_linear(x, w, out_fmt=ofmt), sp.mx_quantize(exact, ofmt)
        assert torch.equal(got.scales, want.scales)
        assert torch.equal(sp.mx_dequantize(got, torch.float32), sp.mx_dequantize(want, torch.float32))


# 64, 128 and 256 channels' tiles with K of several times 512, in even and odd numbers of steps, and a remainder
DEEP = [(300, 1184, 1056, (64, 128)), (300, 2080, 1024, (64, 128)), (2500, 1184, 4096, (128, 128)), (2500, 2080, 4096, (128, 128)),
        (2450, 1632, 4128, (128, 128)), (5000, 1184, 3520, (128, 256)), (5000, 2080, 3520, (128, 256)), (5050, 1632, 3552, (128, 256))]


@pytest.mark.parametrize("n,k,o,tile", DEEP)
@pytest.mark.parametrize("fmt", [sp.MX_E4M3, sp.MX_E2M1])
def test_linear_bits_in_deep_tiles(gpu, n, k, o, tile, fmt):
    """test_linear_bits where every slot of a tile's pipeline is filled again and all four of a word's scales are used."""
    cus = torch.cuda.get_device_properties(gpu).multi_processor_count
    x = mx(*small_ints(n, k, fmt, n + k, -8, 8), k, fmt, gpu)
    w = mx(*small_ints(o, k, sp.MX_E2M1, o + k, 0, 0), k, sp.MX_E2M1, gpu)
    exact = matrix(x) @ matrix(w).T
    g = gen(o)
    bias = torch.randint(-64, 65, (o,), generator=g).float().to(gpu)
    res = torch.randint(-64, 65, (n, o), generator=g).to(gpu)
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        tile_is(cus, n, o, fmt, tile, out_dtype=dt)
        assert torch.equal(sp.mx_linear(x, w, out_dtype=dt), exact.float().to(dt))
        r = res.to(dt)
        assert torch.equal(sp.mx_linear(x, w, bias, residual=r, out=r), (exact + bias.double() + res.to(dt).double()).float().to(dt))
    for ofmt in (sp.MX_E4M3, sp.MX_E2M1):
        tile_is(cus, n, o, fmt, tile, out_fmt=ofmt)
        got, want = sp.mx_linear(x, w, bias, out_fmt=ofmt), sp.mx_quantize((exact + bias.double()).float(), ofmt)
        assert torch.equal(got.scales, want.scales)
        assert torch.equal(sp.mx_dequantize(got, torch.float32), sp.mx_dequantize(want, torch.float32))


def eights(X, W):
    """Sum over groups of 8 consecutive columns of the group's largest |x w|, [n,o]."""
    s = torch.zeros((X.shape[0], W.shape[0]), dtype=torch.float64, device=X.device)
    for c in range(0, X.shape[1], 8):
        s += (X[:, None, c:c + 8].abs() * W[None, :, c:c + 8].abs()).amax(2)
    return s


@pytest.mark.parametrize("n,k,o", [(1, 256, 256), (3, 4096, 128), (16, 1024, 96), (40, 96, 512), (200, 512, 1024), (1500, 352, 800)])
@pytest.mark.parametrize("fmt", [sp.MX_E4M3, sp.MX_E2M1])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_linear_of_values(gpu, n, k, o, fmt, dt):
    """x quantised by the call, SiLU, residual; values or microscaled rows out. The call's quantisation is mx_quantize's."""
    g = gen(n + k + o)
    x = features(n, k, dt, n + k).to(gpu)
    w = sp.mx_quantize((torch.randn((o, k), generator=g) / k ** 0.5).to(gpu), sp.MX_E2M1)
    bias = torch.randn(o, generator=g).to(gpu)
    q = sp.mx_quantize(x, fmt)
    X, W = matrix(q), matrix(w)
    acc = X @ W.T + bias.double()
    off = (2.0 ** -23 * (k + 2)) * (X.abs() @ W.abs().T + bias.double().abs())  # of the sum before the activation
    if fmt == sp.MX_E4M3:
        off = off + 7 * 2.0 ** -13 * eights(X, W)
    # silu(v): |silu'| <= 1.1; its exp and reciprocal are off by (|v| + 4) 2^-23 relative
    y = acc * torch.sigmoid(acc)
    yoff = 1.1 * off + (acc.abs() + 4) * 2.0 ** -23 * y.abs() + 1e-37
    res = torch.randn((n, o), generator=g).to(dt).to(gpu)
    for act, ref, roff in ((sp.ACT_NONE, acc, off), (sp.ACT_SILU, y, yoff)):
        for r in (None, res):
            got = sp.mx_linear(x, w, bias, residual=r, act=act, fmt=fmt)
            assert got.dtype == dt
            want = ref if r is None else ref + r.double()
            allowed = roff + 2.0 ** -22 * want.abs() + (torch.finfo(dt).eps / 2) * (want.abs() + roff) + torch.finfo(dt).tiny
            err = (got.double() - want).abs()
            assert bool((err <= allowed).all()), (act, float((err / allowed).max()))
            assert torch.equal(got, sp.mx_linear(q, w, bias, residual=r, act=act, out_dtype=dt))
        for ofmt in (sp.MX_E4M3, sp.MX_E2M1):
            got = sp.mx_linear(x, w, bias, act=act, fmt=fmt, out_fmt=ofmt)
            assert got.fmt == ofmt and int(got.scales[:, o // 32:].sum()) == 0
            near(got, ref, roff, ofmt)


@pytest.mark.parametrize("n,k,o", [(5, 160, 288), (77, 1024, 96), (300, 1024, 1024), (1803, 1024, 544), (2500, 128, 4096), (7001, 224, 2080)])
@pytest.mark.parametrize("fmt", [sp.MX_E4M3, sp.MX_E2M1])
def test_linear_microscaled_bits(gpu, n, k, o, fmt):
    """Of exact sums (test_linear_bits) the epilogue's quantisation is mx_quantize's, and rows behind the last stay."""
    x = mx(*small_ints(n, k, fmt, n + k, -8, 8), k, fmt, gpu)
    w = mx(*small_ints(o, k, sp.MX_E2M1, o + k, 0, 0), k, sp.MX_E2M1, gpu)
    bias = torch.randint(-64, 65, (o,), generator=gen(o)).float().to(gpu)
    exact = (matrix(x) @ matrix(w).T + bias.double()).float()
    for ofmt in (sp.MX_E4M3, sp.MX_E2M1):
        want = sp.mx_quantize(exact, ofmt)
        buf = sp.MxTensor.empty(n + 2, o, ofmt, gpu)
        buf.codes.fill_(9)
        buf.scales.fill_(9)
        out = sp.MxTensor(buf.codes[:n], buf.scales[:n], o, ofmt)
        assert sp.mx_linear(x, w, bias, out=out) is out
        # (zeros keep a sign that the sum of opposite terms need not share)
        assert torch.equal(out.scales, want.scales)
        assert torch.equal(sp.mx_dequantize(out, torch.float32), sp.mx_dequantize(want, torch.float32))
        assert bool((buf.codes[n:] == 9).all()) and bool((buf.scales[n:] == 9).all())


SMALL = torch.tensor([2.0 ** -9, 3 * 2.0 ** -9, 2.0 ** -6, 1.875 * 2.0 ** -6, 2.0 ** -3, 0.5, 1.125, 1.875, 2.25, 3.5, 3.75])
LARGE = torch.tensor([256.0, 288.0, 320.0, 416.0, 448.0])


def both_ends(n, k, o, cancel, seed, dev):
    """e4m3 rows (as values) and e2m1 weights with both ends of the elements in one group of eight neighbours: cancel: every block
    of 32 has a large element and its opposite beside it, under equal weights; else four blocks of a row have a single large one, or
    one from 4 up. All sums are multiples of 2^-10 below 2^14: exact in fp32, whatever their order."""
    g = gen(seed)
    pick = lambda t, *shape: t[torch.randint(0, len(t), shape, generator=g)]
    sign = lambda *shape: 1.0 - 2.0 * torch.randint(0, 2, shape, generator=g)
    x = pick(SMALL, n, k) * sign(n, k) * (torch.rand((n, k), generator=g) < 0.2)
    if cancel:
        at = torch.arange(0, k, 32) + 2 * torch.randint(0, 16, (n, k // 32), generator=g)
        v = pick(LARGE, n, k // 32) * sign(n, k // 32)
        x.scatter_(1, at, v).scatter_(1, at + 1, -v)
    else:
        at = 32 * torch.rand((n, k // 32), generator=g).argsort(1)[:, :4] + torch.randint(0, 32, (n, 4), generator=g)
        x.scatter_(1, at, pick(torch.cat((LARGE, torch.tensor([4.0, 4.5, 7.5]))), n, 4) * sign(n, 4))
    c = torch.randint(0, 16, (o, k // 2), generator=g, dtype=torch.uint8)
    c = c | c << 4 if cancel else c | torch.randint(0, 16, (o, k // 2), generator=g, dtype=torch.uint8) << 4
    one = lambda rows: torch.full((rows, (k + 511) // 512 * 16), 127, dtype=torch.uint8)
    w = mx(c, one(o), k, sp.MX_E2M1, dev)
    q = mx(x.to(torch.float8_e4m3fn).view(torch.uint8), one(n), k, sp.MX_E4M3, dev)
    X, W = matrix(q), matrix(w)
    assert torch.equal(X.cpu().float(), x) and float((X.abs() @ W.abs().T).max()) < (2 ** 19 if cancel else 2 ** 14)
    full = X @ W.T
    assert float(full.abs().max()) < 2 ** 14
    return x.to(dev), q, w, full


@pytest.mark.parametrize("n,o", [(1, 32), (5, 96), (16, 64), (30, 64), (70, 4096), (100, 4096), (70, 8192), (90, 8192), (128, 8192),
                                 (300, 1024), (2500, 4096), (5000, 3520)])
@pytest.mark.parametrize("cancel", [False, True])
def test_linear_both_ends_of_e4m3(gpu, n, o, cancel):
    """Nothing of a small element is lost beside a large one: fp32 and microscaled results, and 16-bit ones of up to 32 rows."""
    x, q, w, full = both_ends(n, 640, o, cancel, n + o, gpu)
    exact = full.float()
    assert torch.equal(sp.mx_linear(q, w, out_dtype=torch.float32), exact)
    for ofmt in (sp.MX_E4M3, sp.MX_E2M1):
        got, want = sp.mx_linear(q, w, out_fmt=ofmt), sp.mx_quantize(exact, ofmt)
        assert torch.equal(got.scales, want.scales)
        assert torch.equal(sp.mx_dequantize(got, torch.float32), sp.mx_dequantize(want, torch.float32))
    if n <= 32:
        for dt in (torch.float16, torch.bfloat16):
            assert torch.equal(sp.mx_linear(q, w, out_dtype=dt), exact.to(dt))
    if cancel and n <= 16:  # as values: each block's largest element makes its scale 1
        for dt in (torch.float32, torch.float16, torch.bfloat16):
            assert torch.equal(sp.mx_linear(x.to(dt), w, out_dtype=dt), exact.to(dt))
            assert torch.equal(sp.mx_linear(x.to(dt), w, out_dtype=torch.float32), exact)


@pytest.mark.parametrize("n,o", [(300, 96), (2500, 4096), (7001, 2080)])
@pytest.mark.parametrize("fmt", [sp.MX_E4M3, sp.MX_E2M1])
def test_linear_not_finite_in_tiles(gpu, n, o, fmt):
    """A row with a NaN block and a channel with one are NaN throughout in each size of tile; the rest is as without them."""
    x = mx(*small_ints(n, 160, fmt, n, -8, 8), 160, fmt, gpu)
    w = mx(*small_ints(o, 160, sp.MX_E2M1, o, 0, 0), 160, sp.MX_E2M1, gpu)
    for kw in ({"out_dtype": torch.float32}, {"out_dtype": torch.float16}):
        x.scales[n - 2, 3] = w.scales[33, 4] = 127
        want = sp.mx_linear(x, w, **kw)
        want[n - 2], want[:, 33] = float("nan"), float("nan")
        x.scales[n - 2, 3] = w.scales[33, 4] = 255
        assert torch.equal(sp.mx_linear(x, w, **kw).nan_to_num(1e4), want.nan_to_num(1e4))
    got = sp.mx_dequantize(sp.mx_linear(x, w, out_fmt=sp.MX_E4M3), torch.float32).isnan()
    blocks = torch.zeros((n, o), dtype=torch.bool, device=gpu)
    blocks[n - 2] = True
    blocks[:, 32:64] = True  # a block with a NaN reads as NaN
    assert torch.equal(got, blocks)


def test_linear_not_finite(gpu):
    """A row with an infinity or NaN is NaN throughout; a weight row whose block is NaN is a NaN channel; nothing else is."""
    x = features(70, 256, torch.bfloat16, 5)
    x[3, 100] = float("inf")
    x[66, 0] = float("nan")
    w = sp.mx_quantize(features(96, 256, torch.float32, 6).to(gpu), sp.MX_E2M1)
    w.scales[50, 7] = 255
    for rows in (70, 4):  # both forms of the product
        for fmt in (sp.MX_E4M3, sp.MX_E2M1):
            y = sp.mx_linear(x[:rows].contiguous().to(gpu), w, fmt=fmt, out_dtype=torch.float32).cpu()
            bad = torch.zeros((rows, 96), dtype=torch.bool)
            bad[3] = True
            bad[:, 50] = True
            if rows > 66:
                bad[66] = True
            assert torch.equal(y.isnan(), bad)


def test_linear_scales_at_their_ends(gpu):
    """Scale bytes 0 and 254 are 2^-127 and 2^127: their product with the other operand's 2^127 and 2^-127 is 1."""
    k = 128
    one = torch.full((20, k), 0x38, dtype=torch.uint8)  # e4m3 1.0
    two = torch.full((32, k // 2), 0x44, dtype=torch.uint8)  # e2m1 2.0
    for bx, bw in ((0, 254), (254, 0), (127, 127)):
        sx, sw = torch.full((20, 16), bx, dtype=torch.uint8), torch.full((32, 16), bw, dtype=torch.uint8)
        y = sp.mx_linear(mx(one, sx, k, sp.MX_E4M3, gpu), mx(two, sw, k, sp.MX_E2M1, gpu), out_dtype=torch.float32)
        assert torch.equal(y, torch.full((20, 32), 2.0 * k, device=gpu)), (bx, bw)


def test_empty(gpu):
    w = sp.mx_quantize(torch.ones((64, 32), device=gpu), sp.MX_E2M1)
    x = torch.empty((0, 32), dtype=torch.bfloat16, device=gpu)
    assert sp.mx_quantize(x, sp.MX_E4M3).shape == (0, 32)
    assert sp.mx_dequantize(sp.mx_quantize(x, sp.MX_E4M3)).shape == (0, 32)
    assert sp.mx_linear(x, w).shape == (0, 64) and sp.mx_linear(x, w, out_fmt=sp.MX_E4M3).shape == (0, 64)
    t, q = sp.add_norm_mx(x, x)
    assert t.shape == (0, 32) and q.shape == (0, 32)
    w1 = sp.mx_quantize(torch.ones((128, 32), device=gpu), sp.MX_E2M1)
    w2 = sp.mx_quantize(torch.ones((32, 128), device=gpu), sp.MX_E2M1)
    assert sp.convnext_mlp_mx(x, x, None, None, w1, None, w2, None).shape == (0, 32)


# ---- the operators together ----------------------------------------------------------------------------------------


def tail(n, c, dt, seed, dev, pdt=torch.float32):
    g = gen(seed)
    h, x = (features(n, c, dt, seed) + 1).to(dt), torch.randn((n, c), generator=g).to(dt)
    gamma, beta = (torch.rand(c, generator=g) + 0.5).to(pdt), (torch.randn(c, generator=g) * 0.2).to(pdt)
    w1 = sp.mx_quantize((torch.randn((4 * c, c), generator=g) / c ** 0.5).to(dev), sp.MX_E2M1)
    w2 = sp.mx_quantize((torch.randn((c, 4 * c), generator=g) / (4 * c) ** 0.5).to(dev), sp.MX_E2M1)
    b1, b2 = (torch.randn(4 * c, generator=g) * 0.1).to(pdt), (torch.randn(c, generator=g) * 0.1).to(pdt)
    return h.to(dev), x.to(dev), gamma.to(dev), beta.to(dev), w1, b1.to(dev), w2, b2.to(dev)


@pytest.mark.parametrize("c,n", [(32, 1), (96, 77), (256, 1), (256, 4099), (512, 300), (544, 1000), (1024, 1803), (256, 140001)])
@pytest.mark.parametrize("fmt", [sp.MX_E4M3, sp.MX_E2M1])
def test_tail(gpu, c, n, fmt):
    """The tail is its parts: norm, product with SiLU into microscaled rows, product with the residual, also with many rows
    in parts, over h and over x; and without the parameters."""
    dt = torch.float16 if c % 64 else torch.bfloat16
    a = tail(n, c, dt, c + n, gpu, torch.float32 if n > 1 else dt)
    h, x, gamma, beta, w1, b1, w2, b2 = a
    _, q = sp.add_norm_mx(h, None, gamma, beta, kind=sp.NORM_LAYER, fmt=fmt)
    want = sp.mx_linear(sp.mx_linear(q, w1, b1, act=sp.ACT_SILU, out_fmt=fmt), w2, b2, residual=x, out_dtype=dt)
    y = sp.convnext_mlp_mx(*a, fmt=fmt)
    assert y.dtype == dt and bool(torch.isfinite(y).all()) and torch.equal(y, want)
    for over in (0, 1):
        b = [t.clone() if isinstance(t, torch.Tensor) else t for t in a]
        assert torch.equal(sp.convnext_mlp_mx(*b, fmt=fmt, out=b[over]), want)
    bare = sp.convnext_mlp_mx(h, x, None, None, w1, None, w2, None, fmt=fmt)
    ones, zeros = torch.ones(c, device=gpu), torch.zeros(4 * c, device=gpu)
    assert torch.equal(bare, sp.convnext_mlp_mx(h, x, ones, zeros[:c].contiguous(), w1, zeros, w2, zeros[:c].contiguous(), fmt=fmt))


@pytest.mark.parametrize("c,n", [(128, 129), (128, 4099), (128, 70001), (256, 6145), (256, 58321)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_tail_in_one_kernel(gpu, c, n, dt):
    """Where the tail is one kernel (it asks for no workspace) its bits are its parts'."""
    assert sp._workspace_bytes("spc_convnext_mlp_mx_workspace", n, c, sp.MX_E4M3) == 0
    h, x, gamma, beta, w1, b1, w2, b2 = a = tail(n, c, dt, c + n, gpu, torch.float32 if n % 2 else dt)
    _, q = sp.add_norm_mx(h, None, gamma, beta, kind=sp.NORM_LAYER)
    want = sp.mx_linear(sp.mx_linear(q, w1, b1, act=sp.ACT_SILU, out_fmt=sp.MX_E4M3), w2, b2, residual=x, out_dtype=dt)
    assert torch.equal(sp.convnext_mlp_mx(*a), want)
    for over in (0, 1):
        b = [t.clone() if isinstance(t, torch.Tensor) else t for t in a]
        assert torch.equal(sp.convnext_mlp_mx(*b, out=b[over]), want)
    bare = sp.convnext_mlp_mx(h, x, None, None, w1, None, w2, None)
    _, q = sp.add_norm_mx(h, None, kind=sp.NORM_LAYER)
    hid = sp.mx_linear(q, w1, act=sp.ACT_SILU, out_fmt=sp.MX_E4M3)
    assert torch.equal(bare, sp.mx_linear(hid, w2, residual=x, out_dtype=dt))


@pytest.mark.parametrize("c", [128, 256])
def test_tail_in_one_kernel_sums_both_ends(gpu, c):
    """The first product beside large elements that cancel: gamma = 0 leaves beta, rows of both ends of e4m3, to be multiplied."""
    x, q, w1, full = both_ends(1, c, 4 * c, True, c, gpu)
    n = 200 if c == 128 else 8200
    assert sp._workspace_bytes("spc_convnext_mlp_mx_workspace", n, c, sp.MX_E4M3) == 0
    h, res = features(n, c, torch.bfloat16, 1).to(gpu), torch.zeros((n, c), dtype=torch.bfloat16, device=gpu)
    w2 = sp.mx_quantize((torch.randn((c, 4 * c), generator=gen(c)) / c).to(gpu), sp.MX_E2M1)
    got = sp.convnext_mlp_mx(h, res, torch.zeros(c, device=gpu), x[0].contiguous(), w1, None, w2, None)
    y = full.expand(n, -1)
    y = y * torch.sigmoid(y)
    rows = sp.MxTensor(q.codes.repeat(n, 1), q.scales.repeat(n, 1), c, sp.MX_E4M3)
    hid = sp.mx_linear(rows, w1, act=sp.ACT_SILU, out_fmt=sp.MX_E4M3)
    near(hid, y, (full.abs() + 4) * 2.0 ** -23 * y.abs() + 1e-37, sp.MX_E4M3)  # exact sums: what is left is the SiLU's own error
    assert torch.equal(got, sp.mx_linear(hid, w2, residual=res, out_dtype=torch.bfloat16))


@pytest.mark.parametrize("c,n,fmt", [(512, 140001, sp.MX_E4M3), (256, 300007, sp.MX_E2M1), (1024, 40003, sp.MX_E4M3)])
def test_tail_in_unequal_parts(gpu, c, n, fmt):
    """A tail whose hidden units pass the parts' limit, so that its workspace is for some of the rows: every row as in calls of few
    rows each, also over h and over x."""
    whole = n * sp._workspace_bytes("spc_convnext_mlp_mx_workspace", 512, c, fmt) // 512
    assert 0 < sp._workspace_bytes("spc_convnext_mlp_mx_workspace", n, c, fmt) < 0.6 * whole
    a = tail(n, c, torch.bfloat16, c, gpu)
    want = torch.empty_like(a[0])
    step = 20011
    for i in range(0, n, step):
        want[i:i + step] = sp.convnext_mlp_mx(a[0][i:i + step], a[1][i:i + step], *a[2:], fmt=fmt)
    assert torch.equal(sp.convnext_mlp_mx(*a, fmt=fmt), want)
    for over in (0, 1):
        b = [t.clone() if k == over else t for k, t in enumerate(a)]
        assert torch.equal(sp.convnext_mlp_mx(*b, fmt=fmt, out=b[over]), want)


@pytest.mark.parametrize("c,n", [(128, 131), (256, 129), (256, 65 * 7 + 1), (512, 140)])
def test_tail_writes_its_rows_only(gpu, c, n):
    a = tail(n, c, torch.bfloat16, c, gpu)
    buf = torch.full((n + 8, c), 7.0, dtype=torch.bfloat16, device=gpu)
    y = sp.convnext_mlp_mx(*a, out=buf[4:n + 4])
    assert torch.equal(y, sp.convnext_mlp_mx(*a)) and bool((buf[:4] == 7).all()) and bool((buf[n + 4:] == 7).all())


def test_tail_in_one_kernel_edges(gpu):
    """At 256 channels: rows before and behind stay, rows that are not finite stay alone (at 128 the tests around this one)."""
    n, c = 8193 + 64 * 3, 256
    assert sp._workspace_bytes("spc_convnext_mlp_mx_workspace", n, c, sp.MX_E4M3) == 0
    a = list(tail(n, c, torch.float16, c, gpu))
    want = sp.convnext_mlp_mx(*a)
    a[0], a[1] = a[0].clone(), a[1].clone()
    a[0][5, 3], a[0][n - 1, c - 1], a[1][9, 0] = float("nan"), float("inf"), float("inf")
    buf = torch.full((n + 8, c), 7.0, dtype=torch.float16, device=gpu)
    y = sp.convnext_mlp_mx(*a, out=buf[4:n + 4])
    assert bool((buf[:4] == 7).all()) and bool((buf[n + 4:] == 7).all())
    assert bool(y[5].isnan().all()) and bool(y[n - 1].isnan().all()) and float(y[9, 0]) == float("inf")
    want[5], want[n - 1], want[9, 0] = float("nan"), float("nan"), float("inf")
    assert torch.equal(y.nan_to_num(5.0), want.nan_to_num(5.0))


@pytest.mark.parametrize("c,n", [(128, 200), (256, 300), (512, 300)])
def test_tail_not_finite(gpu, c, n):
    """A row of h with an infinity or NaN gives a NaN row, an infinite x passes through, no other row changes."""
    a = list(tail(n, c, torch.float16, c, gpu))
    want = sp.convnext_mlp_mx(*a)
    a[0], a[1] = a[0].clone(), a[1].clone()
    a[0][5, 3] = float("nan")
    a[0][70, c - 1] = float("inf")
    a[1][9, 0] = float("inf")
    y = sp.convnext_mlp_mx(*a)
    assert bool(y[5].isnan().all()) and bool(y[70].isnan().all()) and float(y[9, 0]) == float("inf")
    same = torch.ones((n, c), dtype=torch.bool, device=gpu)
    same[5] = same[70] = False
    same[9, 0] = False
    assert torch.equal(y[same], want[same])


def test_block(gpu):
    """A ConvNeXt block as a decoder runs it: conv on a kernel map, then the tail with 4-bit weights, beside the tail in
    16 bits. The difference is what quantising costs: e2m1 weights are off by 11%, e4m3 activations by 2.7% (2-norm), so
    each product by about 12% of its size, and the MLP's part of y by about twice that."""
    from spconv_amd import workloads as W
    c = 64
    coords = torch.from_numpy(W.shell_coords(W.CONFIGS["c1"])).to(gpu)
    cache, n = sp.build_neighbors(coords), coords.shape[0]
    g = gen(9)
    x = torch.randn((n, c), generator=g).to(torch.float16).to(gpu)
    cw = (torch.randn((c, 27, c), generator=g) / (14 * c) ** 0.5).to(torch.float16).to(gpu)
    h = sp.subm_conv_fused(x, cw, None, cache)
    w1 = (torch.randn((4 * c, c), generator=g) / c ** 0.5).to(torch.float16).to(gpu)
    w2 = (torch.randn((c, 4 * c), generator=g) / (4 * c) ** 0.5).to(torch.float16).to(gpu)
    full = sp.convnext_mlp(h, x, None, None, w1, None, w2, None)
    mx_y = sp.convnext_mlp_mx(h, x, None, None, sp.mx_quantize(w1), None, sp.mx_quantize(w2), None)
    part = (full.double() - x.double()).norm()
    assert float((mx_y.double() - full.double()).norm() / part) < 0.3
    assert float((mx_y.double() - full.double()).norm() / part) > 0.02  # the weights do have 4 bits


def test_graph_replays(gpu):
    """Two captured calls (each with its own workspace, taken at capture), replayed in turn with eager work between, on a stream
    of their own, give the eager results on every replay."""
    a, b = tail(700, 256, torch.bfloat16, 1, gpu), tail(9, 256, torch.bfloat16, 2, gpu)
    x = features(40, 512, torch.float16, 3).to(gpu)
    w = sp.mx_quantize(features(96, 512, torch.float32, 4).to(gpu), sp.MX_E2M1)
    want = [sp.convnext_mlp_mx(*a), sp.convnext_mlp_mx(*b), sp.mx_linear(x, w)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    try:
        for call in (lambda: sp.convnext_mlp_mx(*a), lambda: sp.convnext_mlp_mx(*b), lambda: sp.mx_linear(x, w)):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                sp.set_stream(torch.cuda.current_stream())
                outs.append(call())
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
        assert torch.equal(sp.convnext_mlp_mx(*a), want[0])


def test_captured_call_without_a_workspace(gpu):
    """The C entries' own workspace is not for a graph: refused before anything is recorded, and the capture goes on."""
    lib, P = sp.load_library(), lambda t: t.data_ptr()
    x = features(40, 64, torch.float16, 3).to(gpu)
    w = sp.mx_quantize(features(32, 64, torch.float32, 4).to(gpu), sp.MX_E2M1)
    y = torch.empty((40, 32), dtype=torch.float16, device=gpu)

    def call():
        return lib.spc_mx_linear(P(x), None, sp.F16, sp.MX_E4M3, P(w.codes), P(w.scales), None, 0, None, 0, 40, 64, 32, sp.F16, P(y),
                                 None, None, 0)

    assert call() == 0
    want = y.clone()
    assert torch.equal(want, sp.mx_linear(x, w))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph, stream=s):
            sp.set_stream(torch.cuda.current_stream())
            y.fill_(2.0)
            rc = call()
    finally:
        torch.cuda.synchronize()
        sp.set_stream(torch.cuda.current_stream())
    assert rc == -1 and "workspace" in lib.spc_last_error().decode()
    graph.replay()
    torch.cuda.synchronize()
    assert bool((y == 2).all()) and call() == 0 and torch.equal(y, want)


def test_other_stream(gpu):
    """Calls on a stream that the library was given, ordered after work on it."""
    x = features(300, 256, torch.bfloat16, 3).to(gpu)
    w = sp.mx_quantize(features(128, 256, torch.float32, 4).to(gpu), sp.MX_E2M1)
    want = sp.mx_linear(x * 2, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    try:
        with torch.cuda.stream(s):
            sp.set_stream(s)
            got = sp.mx_linear(x * 2, w)
        s.synchronize()
    finally:
        sp.set_stream(torch.cuda.current_stream())
    assert torch.equal(got, want)


def test_library_on_another_stream_than_torch(gpu):
    """Workspaces follow the library's stream, not torch's: work on torch's own meanwhile does not reach them."""
    x = features(4000, 1024, torch.bfloat16, 3).to(gpu)
    w = sp.mx_quantize(features(1024, 1024, torch.float32, 4).to(gpu), sp.MX_E2M1)
    want = sp.mx_linear(x, w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    outs, junk = [], []
    try:
        sp.set_stream(s)
        for _ in range(8):
            outs.append(sp.mx_linear(x, w, out=torch.empty_like(want)))
            junk.append(torch.full((4000, 1056), 255, dtype=torch.uint8, device=gpu))  # on torch's stream
        s.synchronize()
    finally:
        sp.set_stream(torch.cuda.current_stream())
    for got in outs:
        assert torch.equal(got, want)


def test_stream_set_through_the_c_entry(gpu):
    """As above where the stream was set behind the binding's back: workspaces still follow it."""
    lib = sp.load_library()
    x = features(4000, 1024, torch.bfloat16, 3).to(gpu)
    w = sp.mx_quantize(features(1024, 1024, torch.float32, 4).to(gpu), sp.MX_E2M1)
    want = sp.mx_linear(x, w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    outs, junk = [torch.empty_like(want) for _ in range(8)], []
    try:
        assert lib.spc_set_stream(s.cuda_stream) == 0
        assert sp._library_stream() == s.cuda_stream
        for out in outs:
            sp.mx_linear(x, w, out=out)
            junk.append(torch.full((4000, 1056), 255, dtype=torch.uint8, device=gpu))  # on torch's stream
        s.synchronize()
    finally:
        sp.set_stream(torch.cuda.current_stream())
    for got in outs:
        assert torch.equal(got, want)


def test_refusals(gpu):
    """Calls that the binding or the library refuses before anything runs."""
    x = features(8, 64, torch.bfloat16, 1).to(gpu)
    w = sp.mx_quantize(features(32, 64, torch.float32, 1).to(gpu), sp.MX_E2M1)
    big = torch.zeros((16, 64), dtype=torch.bfloat16, device=gpu)
    for call in (lambda: sp.mx_quantize(x[:, :48].contiguous()), lambda: sp.mx_quantize(x.t()), lambda: sp.mx_quantize(x, 3),
                 lambda: sp.mx_linear(x, sp.mx_quantize(x, sp.MX_E4M3)), lambda: sp.mx_linear(x[:, :32].contiguous(), w),
                 lambda: sp.mx_linear(x, sp.mx_quantize(x[:5].contiguous(), sp.MX_E2M1)),
                 lambda: sp.mx_linear(x, w, residual=x), lambda: sp.mx_linear(x, w, act=2), lambda: sp.mx_linear(x.cpu(), w),
                 lambda: sp.mx_linear(x, w, torch.zeros(31, device=gpu)),
                 lambda: sp.mx_linear(x, w, out_fmt=sp.MX_E4M3, residual=torch.zeros((8, 32), device=gpu)),
                 lambda: sp.add_norm_mx(big[:8], big[4:12], sum=big[1:9]), lambda: sp.add_norm_mx(x, x.float()),
                 lambda: sp.add_norm_mx(x.float()), lambda: sp.add_norm_mx(x, kind=2),
                 lambda: sp.add_norm_mx(torch.zeros((2, 16416), dtype=torch.float16, device=gpu))):
        with pytest.raises((ValueError, RuntimeError)):
            call()
    n64 = sp.mx_quantize(torch.ones((64, 64), device=gpu), sp.MX_E2M1)
    sq = features(64, 64, torch.bfloat16, 2).to(gpu)
    with pytest.raises(RuntimeError, match="overlap"):
        sp.mx_linear(sq, n64, out=sq)
