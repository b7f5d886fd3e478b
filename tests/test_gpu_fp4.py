"""Microscaled 4-bit matrices on the device against 64-bit numpy: quantisation and its inverse bit
for bit, products to the bound of their fp32 accumulation, top-k exactly."""
import numpy as np
import pytest

import _fp4_ref as ref

pytestmark = pytest.mark.gpu

FMTS = ["nvfp4", "mxfp4"]
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # half a step, relative


def _dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _parts(rng, rows, cols, fmt, spread=4):
    """Random codes and scales: every code, scales over a few binades, some zero blocks."""
    nb = -(-cols // ref.BLOCK[fmt])
    codes = rng.integers(0, 16, (rows, cols)).astype(np.uint8)
    if fmt == "mxfp4":
        scales = rng.integers(127 - spread, 127 + spread + 1, (rows, nb)).astype(np.uint8)
    else:
        scales = rng.integers(8 * (7 - spread), 8 * (7 + spread) + 1, (rows, nb)).astype(np.uint8)
        scales[rng.random((rows, nb)) < 0.05] = 0
    return codes, scales


def _matrix(codes, scales, cols, fmt, g=None):
    import rfx_b200
    return rfx_b200.Fp4Matrix.from_parts(_dev(ref.pack(codes)), _dev(scales), g, cols=cols, format=fmt)


def _same(got, want):
    got, want = np.asarray(got), np.asarray(want)
    assert got.shape == want.shape
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    bad = np.argwhere((got != want) & ~nan)
    assert len(bad) == 0, (len(bad), bad[:4].tolist(), got[tuple(bad[0])], want[tuple(bad[0])])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 15), (5, 16), (2, 17), (128, 64), (129, 33), (300, 50), (40, 256),
                                       (70, 257), (20, 1000), (257, 511), (5, 4097)])
def test_quantize_matches_the_definition(fmt, rows, cols):
    import torch
    import rfx_b200
    rng = np.random.default_rng(rows * 7919 + cols)
    x = (rng.normal(size=(rows, cols)) * np.exp(rng.normal(size=(rows, 1)))).astype(np.float32)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        t = torch.from_numpy(x).cuda().to(dt)
        m = rfx_b200.fp4_quantize(t, format=fmt)
        codes, scales, g = ref.quantize(t.double().cpu().numpy(), fmt)
        c, s, gs = m.parts()
        assert np.array_equal(s.cpu().numpy(), scales)
        _same(ref.values(ref.unpack(c.cpu().numpy(), cols), scales, g, fmt), ref.values(codes, scales, g, fmt))
        if fmt == "nvfp4":
            assert float(gs) == g
        want = ref.values(codes, scales, g, fmt)
        for odt in (torch.float32, torch.bfloat16):  # both hold the values exactly
            _same(m.dequantize(odt).double().cpu().numpy(), want)
        _same(m.dequantize(torch.float16).cpu().numpy(), want.astype(np.float32).astype(np.float16))


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_borders(fmt):
    """Values on, just below and just above every border between two codes and two scales."""
    import torch
    import rfx_b200
    rng = np.random.default_rng(2)
    mids = (ref.E2M1[1:] + ref.E2M1[:-1]) / 2
    rows = []
    for scale in list(ref.E4M3[1::5]) + [2.0 ** -20, 3.0, 1e-3]:
        for amax in (6.0, 4.5, 5.3125, 6.1875, 3.0):
            v = np.concatenate([mids, ref.E2M1, [5.9]])
            base = np.float32(v * scale)
            up, dn = np.nextafter(base, np.float32(np.inf)), np.nextafter(base, np.float32(-np.inf))
            for b in (base, up, dn):
                r = np.zeros(32, np.float32)
                r[:16] = b * np.where(rng.random(16) < 0.5, -1, 1)
                r[16:] = b
                r[0] = r[16] = np.float32(amax * scale)
                rows.append(r)
    # a block maximum on the borders between two scales, and beside them
    edge = (ref.E4M3[1:] + ref.E4M3[:-1]) / 2 * 6
    for b in (np.float32(edge), np.nextafter(np.float32(edge), np.float32(1e9)), np.nextafter(np.float32(edge), np.float32(0))):
        for v in b:
            r = np.zeros(32, np.float32)
            r[5] = r[21] = v
            rows.append(r)
    rows.append(np.full(32, 2688.0, np.float32))  # g = 1
    x = np.stack(rows)
    m = rfx_b200.fp4_quantize(torch.from_numpy(x).cuda(), format=fmt)
    codes, scales, g = ref.quantize(x, fmt)
    assert np.array_equal(m.parts()[1].cpu().numpy(), scales)
    _same(m.dequantize().double().cpu().numpy(), ref.values(codes, scales, g, fmt))


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_extremes(fmt):
    """Zeros, denormals, the largest floats, infinities and NaN, strided and unaligned rows."""
    import torch
    import rfx_b200
    big = np.float32(3.0e38)
    x = np.zeros((9, 70), np.float32)
    x[1, :] = 1e-45
    x[2, 3] = big
    x[3, ::2] = -1e-38
    x[4, 7] = np.inf
    x[5, 40] = np.nan
    x[6, :] = np.linspace(-1, 1, 70)
    x[7, :] = -0.0
    x[8, 69] = -np.inf
    for rowset in (range(9), [0, 1, 3], [0], [4, 5], [6, 7]):
        y = x[list(rowset)]
        buf = torch.zeros((len(y), 77), device="cuda")
        buf[:, 3:73] = torch.from_numpy(y)
        m = rfx_b200.fp4_quantize(buf[:, 3:73], format=fmt)
        codes, scales, g = ref.quantize(y, fmt)
        assert np.array_equal(m.parts()[1].cpu().numpy(), scales), rowset
        with np.errstate(over="ignore"):
            want = ref.values(codes, scales, g, fmt).astype(np.float32)
        _same(m.dequantize().cpu().numpy(), want)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (130, 31), (128, 128), (77, 300), (300, 640)])
def test_parts_round_trip(fmt, rows, cols):
    import torch
    rng = np.random.default_rng(rows + cols)
    codes, scales = _parts(rng, rows, cols, fmt)
    g = None if fmt == "mxfp4" else 0.375
    m = _matrix(codes, scales, cols, fmt, g)
    c, s, gs = m.parts()
    assert np.array_equal(ref.unpack(c.cpu().numpy(), cols), codes) and np.array_equal(s.cpu().numpy(), scales)
    want = ref.values(codes, scales, 1.0 if g is None else g, fmt)
    _same(m.dequantize().double().cpu().numpy(), want.astype(np.float32))
    out = torch.full((rows, cols + 5), -7.0, device="cuda")
    m.dequantize(out=out[:, 2:2 + cols])
    _same(out[:, 2:2 + cols].cpu().numpy(), want.astype(np.float32))
    assert (out[:, :2] == -7).all() and (out[:, 2 + cols:] == -7).all()
    if gs is not None:
        assert float(gs) == g


@pytest.mark.parametrize("fmt", FMTS)
def test_widest_matrix(fmt):
    """One row of the most columns, and its product with itself."""
    import torch
    import rfx_b200
    from rfx_b200 import fp4
    x = torch.zeros(1, fp4.MAX_COLS, device="cuda", dtype=torch.bfloat16)
    x[0, -5:] = torch.tensor([1.0, -2.0, 3.0, 4.0, 6.0])
    x[0, 7] = 6.0
    m = rfx_b200.fp4_quantize(x, format=fmt)
    assert torch.equal(m.dequantize(torch.bfloat16), x)
    assert float(rfx_b200.fp4_product(m, m)[0, 0]) == 1 + 4 + 9 + 16 + 36 + 36
    c, s, g = m.parts()
    again = rfx_b200.Fp4Matrix.from_parts(c, s, g, cols=fp4.MAX_COLS, format=fmt)
    assert torch.equal(again.dequantize(torch.bfloat16), x)
    rfx_b200.fp4_status()
    with pytest.raises(ValueError, match="at most"):
        rfx_b200.fp4_quantize(torch.zeros(1, 1, device="cuda").expand(1, fp4.MAX_COLS + 1).contiguous(), format=fmt)


def _product_check(rng, fmt, m, n, k, dtype="float32", spread=4):
    import torch
    import rfx_b200
    ca, sa = _parts(rng, m, k, fmt, spread)
    cb, sb = _parts(rng, n, k, fmt, spread)
    va, vb = ref.values(ca, sa, 1.0, fmt), ref.values(cb, sb, 1.0, fmt)
    a, b = _matrix(ca, sa, k, fmt), _matrix(cb, sb, k, fmt)
    buf = torch.full((m, n + 3), -7.0, device="cuda", dtype=getattr(torch, dtype))
    out = rfx_b200.fp4_product(a, b, out=buf[:, :n])
    rfx_b200.fp4_status()
    got = out.double().cpu().numpy()
    want, size = va @ vb.T, np.abs(va) @ np.abs(vb).T
    # products are exact; k fp32 additions, each off by at most a unit of the last place (2^-23)
    # of a partial sum, none of which exceeds `size`; then one rounding to the output type
    tol = k * 2.0 ** -23 * size
    tol = tol + HALF[dtype] * (np.abs(want) + tol) + (2.0 ** -25 if dtype == "float16" else 0)
    bad = np.argwhere(~(np.abs(got - want) <= tol))
    assert len(bad) == 0, (len(bad), bad[:3].tolist(), got[tuple(bad[0])], want[tuple(bad[0])], tol[tuple(bad[0])])
    assert (buf[:, n:] == -7).all()
    print(f"worst error / size: {np.max(np.abs(got - want) / np.maximum(size, 1e-300)):.3g}")


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", [(16, 128, 64), (1, 1, 1), (128, 128, 64), (256, 256, 64), (1, 300, 17), (17, 129, 128),
                                   (129, 130, 192), (100, 257, 256), (33, 200, 320), (300, 500, 1000), (257, 640, 65),
                                   (513, 3000, 64), (70, 1000, 4100), (8, 1000, 64), (9, 1025, 64),
                                   (17, 5000, 64), (32, 700, 200), (33, 40, 64), (5, 200000, 64), (3, 30000, 256),
                                   (1, 100, 2048), (16, 4000, 4096), (64, 1000, 3000), (33, 129, 9000), (7, 8192, 2100)])
def test_product(fmt, m, n, k):
    _product_check(np.random.default_rng(m + 1000 * n + k), fmt, m, n, k)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_product_half_outputs(fmt, dtype):
    rng = np.random.default_rng(5)
    for m, n, k in ((1, 100, 64), (65, 260, 50), (300, 301, 300)):
        _product_check(rng, fmt, m, n, k, dtype, spread=1)


@pytest.mark.parametrize("m,k", [(4, 64), (4, 4096), (40, 200), (300, 300)])
def test_product_of_scales_outside_fp32(m, k):
    """Matrix scales whose product overflows or vanishes, where the results need not."""
    import torch
    import rfx_b200
    rng = np.random.default_rng(m + k)
    n = 200
    x = rng.integers(1, 7, (m, k)).astype(np.float32)
    y = rng.integers(1, 7, (n, k)).astype(np.float32)
    x[1], y[3] = 0, 0
    x[2, : k // 2], y[4, k // 2:] = 0, 0  # halves of which nothing meets: x[2] . y[4] = 0
    def product(e, f):
        mats, vals = [], []
        for t, s in ((x, e), (y, f)):
            t = t * np.float32(2.0 ** s)
            mats.append(rfx_b200.fp4_quantize(torch.from_numpy(t).cuda()))
            vals.append(ref.values(*ref.quantize(t, "nvfp4"), "nvfp4"))
        got = rfx_b200.fp4_product(*mats).double().cpu().numpy()
        rfx_b200.fp4_status()
        return got, vals[0] @ vals[1].T
    got, want = product(120, 110)  # every nonzero result is beyond fp32
    assert np.array_equal(got, np.where(want > 0, np.inf, 0.0)) and (want == 0).sum() >= n + m
    for e, f in ((-20, -118), (-118, -20), (100, -90)):
        got, want = product(e, f)
        # k additions of exact terms, all positive, off by at most 2^-23 each; one rounding, to a
        # multiple of 2^-149 where the result has few bits left
        assert (np.abs(got - want) <= (k * 2.0 ** -23 + 2.0 ** -24) * want + 2.0 ** -150).all()
        assert (want > 0).sum() > 0.9 * (m - 1) * (n - 1)


@pytest.mark.parametrize("m,k", [(4, 64), (4, 4096), (40, 200), (300, 300)])
@pytest.mark.parametrize("fmt", FMTS)
def test_product_of_nan_rows(fmt, m, k):
    """A block that is not finite makes its row's products NaN and no others."""
    import torch
    import rfx_b200
    rng = np.random.default_rng(m + k)
    x, y = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((150, k)).astype(np.float32)
    x[2, k - 1], y[7, 0], y[130, 20] = np.nan, np.inf, -np.inf
    got = rfx_b200.fp4_product(*(rfx_b200.fp4_quantize(torch.from_numpy(t).cuda(), format=fmt) for t in (x, y)))
    rfx_b200.fp4_status()
    want = np.zeros((m, 150), bool)
    want[2], want[:, [7, 130]] = True, True
    assert np.array_equal(np.isnan(got.cpu().numpy()), want)


def _topk_check(a, b, va, vb, k, fmt, self_offset=None):
    import rfx_b200
    idx, val = rfx_b200.fp4_topk(a, b, k, self_offset=self_offset)
    rfx_b200.fp4_status()
    wi, wv = ref.topk(va, vb, k, self_offset, fmt)
    idx, val = idx.cpu().numpy(), val.cpu().numpy()
    bad = np.argwhere(idx != wi)
    assert len(bad) == 0, (len(bad), bad[:4].tolist(), idx[tuple(bad[0])], wi[tuple(bad[0])])
    assert np.array_equal(val, wv)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k,top", [(1, 1, 1, 1), (5, 40, 64, 7), (128, 128, 64, 50), (130, 700, 37, 50), (3, 5000, 64, 64),
                                       (300, 2000, 200, 10), (64, 3001, 256, 33), (1, 20000, 96, 50)])
def test_topk(fmt, m, n, k, top):
    rng = np.random.default_rng(m * 31 + n + k)
    ca, sa = _parts(rng, m, k, fmt)
    cb, sb = _parts(rng, n, k, fmt)
    _topk_check(_matrix(ca, sa, k, fmt), _matrix(cb, sb, k, fmt), ref.values(ca, sa, 1.0, fmt),
                ref.values(cb, sb, 1.0, fmt), top, fmt)


@pytest.mark.parametrize("fmt", FMTS)
def test_topk_ties_and_self(fmt):
    """Duplicated rows (equal values rank by index), zero rows, negative products, self left out."""
    rng = np.random.default_rng(8)
    n, k = 3000, 40
    c, s = _parts(rng, n, k, fmt, spread=1)
    c[rng.integers(0, n, 800)] = c[5]
    s[:] = s[0]
    c[100:140] = 0
    v = ref.values(c, s, 1.0, fmt)
    m = _matrix(c, s, k, fmt)
    for top in (1, 50, 64):
        _topk_check(m, m, v, v, top, fmt, self_offset=0)
    sub = m.rows(256, 700)
    _topk_check(sub, m, v[256:700], v, 20, fmt, self_offset=256)
    few = m.rows(0, 30)
    _topk_check(few, few, v[:30], v[:30], 50, fmt, self_offset=0)  # fewer neighbours than k
    one = m.rows(0, 1)
    _topk_check(one, one, v[:1], v[:1], 3, fmt, self_offset=0)     # none at all


@pytest.mark.parametrize("fmt", FMTS)
def test_topk_all_rows_equal(fmt):
    """Every product equal: the lowest indices win, however much passes the filter."""
    rng = np.random.default_rng(4)
    c, s = _parts(rng, 1, 64, fmt, spread=1)
    c, s = np.repeat(c, 2500, 0), np.repeat(s, 2500, 0)
    v = ref.values(c, s, 1.0, fmt)
    m = _matrix(c, s, 64, fmt)
    _topk_check(m.rows(0, 140), m, v[:140], v, 50, fmt)


@pytest.mark.parametrize("fmt", FMTS)
def test_topk_extreme_scales_and_nan(fmt):
    """Rows whose scale is NaN are nobody's neighbours; the largest and smallest scales."""
    rng = np.random.default_rng(9)
    n, k = 900, 64
    c, s = _parts(rng, n, k, fmt)
    s[rng.integers(0, n, 30), 0] = 255 if fmt == "mxfp4" else 127
    if fmt == "mxfp4":
        s[200:230] = rng.integers(0, 12, (30, s.shape[1]))
        s[300:310] = rng.integers(180, 200, (10, s.shape[1]))
    else:
        s[200:230] = rng.integers(0, 4, (30, s.shape[1]))
        s[300:310] = 126
    with np.errstate(all="ignore"):
        v = ref.values(c, s, 1.0, fmt)
        m = _matrix(c, s, k, fmt)
        _topk_check(m, m, v, v, 20, fmt, self_offset=0)


@pytest.mark.parametrize("fmt", FMTS)
def test_estimator_in_4_bits(fmt):
    """quant_mode: the factors are the float factors quantised; product and top-k follow them; the
    operators together on the same factors give the same answers."""
    import rfx_b200
    from _helpers import synth
    X, y = synth("multiclass", 700, 10, 5)
    kw = dict(nsample=700, ntree=30, mdim=10, mtry=3, compute_proximity=True, compute_importance=False,
              use_qlora=True, rank=24, show_progress=False)
    est = rfx_b200.RandomForestClassifier(quant_mode=fmt, **kw)
    est.fit(X, y)
    A, B, r = est.get_lowrank_factors()
    assert r == 24 and A.shape == (700, 24) and np.array_equal(A, B)
    with pytest.raises(RuntimeError, match="held as"):
        est.get_lowrank_quantized()
    P = est.get_lowrank_product()
    tol = 24 * 2.0 ** -23 * (np.abs(A) @ np.abs(A).T) + 2.0 ** -24 * np.abs(A @ A.T)
    assert (np.abs(P - A @ A.T) <= tol).all()
    assert np.array_equal(est.get_lowrank_product(301, 450), P[301:450])
    wi, wv = ref.topk(A, A, 12, 0, fmt)
    idx, val = est.get_lowrank_topk(12)
    assert np.array_equal(idx, wi) and np.array_equal(val, wv)
    idx, val = est.get_lowrank_topk(12, 333, 601)
    assert np.array_equal(idx, wi[333:601]) and np.array_equal(val, wv[333:601])
    # int8 factors of the same fit approximate the same floats: 4 bits within their own step
    e8 = rfx_b200.RandomForestClassifier(quant_mode="int8", **kw)
    e8.fit(X, y)
    A8, _, _ = e8.get_lowrank_factors()
    m = rfx_b200.fp4_quantize(_dev(A.astype(np.float32)), format=fmt)
    # quantising the quantised values keeps them (their scales divide them exactly)
    _same(m.dequantize().double().cpu().numpy(), A)
    _same(rfx_b200.fp4_product(m, m).cpu().numpy(), P)
    ti, tv = rfx_b200.fp4_topk(m, m, 12, self_offset=0)
    assert np.array_equal(ti.cpu().numpy(), wi) and np.array_equal(tv.cpu().numpy(), wv)
    step = np.abs(A8).max(1, keepdims=True) / 127 / 2
    # a code is off by at most 1 in units of its block's scale (between 4 and 6), the scale is at
    # most largest / 3 (mxfp4) or (1 + 2^-4) largest / 6 (nvfp4)
    bs = ref.BLOCK[fmt]
    for c in range(0, 24, bs):
        big = np.abs(A8[:, c:c + bs]).max(1, keepdims=True) + step
        assert (np.abs(A[:, c:c + bs] - A8[:, c:c + bs]) <= big / 3 + step).all()


@pytest.mark.parametrize("fmt,m,n,k,top", [("nvfp4", 320, 40000, 64, 50), ("mxfp4", 300, 140000, 40, 64), ("nvfp4", 310, 3000, 130, 64),
                                           ("mxfp4", 2, 1200000, 20, 50)])
def test_topk_many_rows(fmt, m, n, k, top):
    """The forms the selection takes by rows of a and keys of a row (units of one key, of eight, of
    several vectors), with duplicated rows; a sample of the queries is checked."""
    import rfx_b200
    rng = np.random.default_rng(n)
    ca, sa = _parts(rng, m, k, fmt, spread=2)
    cb, sb = _parts(rng, n, k, fmt, spread=2)
    src = rng.integers(0, n, 3000)
    dst = rng.integers(0, n, 3000)
    cb[dst], sb[dst] = cb[src], sb[src]
    a, b = _matrix(ca, sa, k, fmt), _matrix(cb, sb, k, fmt)
    idx, val = rfx_b200.fp4_topk(a, b, top)
    rfx_b200.fp4_status()
    pick = np.unique(np.concatenate([[0, m - 1], rng.integers(0, m, 12)]))
    wi, wv = ref.topk(ref.values(ca[pick], sa[pick], 1.0, fmt), ref.values(cb, sb, 1.0, fmt), top, None, fmt)
    assert np.array_equal(idx.cpu().numpy()[pick], wi)
    assert np.array_equal(val.cpu().numpy()[pick], wv)


def test_topk_masses_of_ties():
    """Few distinct rows, each thousands of times: more columns reach the bar than the selection has
    room for at once, in each of its forms."""
    import rfx_b200
    rng = np.random.default_rng(12)
    for m, n in ((3, 50000), (300, 40000), (300, 20000)):
        c, s = _parts(rng, 7, 64, "nvfp4", spread=1)
        which = rng.integers(0, 7, n)
        cb, sb = c[which], s[which]
        a, b = _matrix(cb[:m], sb[:m], 64, "nvfp4"), _matrix(cb, sb, 64, "nvfp4")
        idx, val = rfx_b200.fp4_topk(a, b, 33, self_offset=0)
        rfx_b200.fp4_status()
        pick = np.array([0, 1, m - 1])
        vb = ref.values(cb, sb, 1.0, "nvfp4")
        for i in pick:
            wi, wv = ref.topk(vb[i:i + 1], vb, 33, int(i), "nvfp4")
            assert np.array_equal(idx[i].cpu().numpy(), wi[0]) and np.array_equal(val[i].cpu().numpy(), wv[0])


@pytest.mark.parametrize("fmt,n,k,top,kind", [
    ("nvfp4", 10, 64, 20, "plain"), ("mxfp4", 1, 20, 1, "plain"), ("nvfp4", 3700, 64, 64, "plain"), ("mxfp4", 3700, 50, 10, "self"),
    ("nvfp4", 3700, 64, 33, "ties"), ("mxfp4", 3700, 64, 64, "ties"), ("nvfp4", 32700, 256, 50, "self"),
    ("mxfp4", 30000, 200, 64, "extreme"), ("nvfp4", 5000, 130, 1, "extreme"), ("mxfp4", 3700, 64, 50, "equal")])
def test_topk_a_warp_a_row(fmt, n, k, top, kind):
    """Thousands of rows against few keys; a sample of the queries is checked."""
    import rfx_b200
    m = 3700
    rng = np.random.default_rng(n + k + top)
    cb, sb = _parts(rng, n, k, fmt, spread=2)
    if kind in ("ties", "equal"):
        which = rng.integers(0, 5 if kind == "ties" else 1, n)
        cb, sb = cb[which], sb[which]
    if kind == "extreme":
        sb[rng.integers(0, n, n // 50), 0] = 255 if fmt == "mxfp4" else 127
        sb[50:90] = rng.integers(0, 8, (40, sb.shape[1]))
        sb[100:110] = rng.integers(180, 200, (10, sb.shape[1])) if fmt == "mxfp4" else 126
    same = kind != "plain" and n >= m
    ca, sa = (cb[:m], sb[:m]) if same else _parts(rng, m, k, fmt, spread=2)
    a, b = _matrix(ca, sa, k, fmt), _matrix(cb, sb, k, fmt)
    idx, val = rfx_b200.fp4_topk(a, b, top, self_offset=0 if same else None)
    rfx_b200.fp4_status()
    idx, val = idx.cpu().numpy(), val.cpu().numpy()
    pick = np.unique(np.concatenate([[0, m - 1], np.arange(48, 56), np.arange(99, 103), rng.integers(0, m, 12)]))
    vb = ref.values(cb, sb, 1.0, fmt)
    with np.errstate(all="ignore"):
        for i in pick:
            wi, wv = ref.topk(ref.values(ca[i:i + 1], sa[i:i + 1], 1.0, fmt), vb, top, int(i) if same else None, fmt)
            assert np.array_equal(idx[i], wi[0]) and np.array_equal(val[i], wv[0]), i


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n", [(2, 33), (3, 1000), (400, 1500), (3800, 700), (5, 2047), (2, 2070), (4, 40)])
def test_topk_fewer_chunks_than_neighbours(fmt, m, n):
    """So few rows that 32 times k reach them: the chunks' maxima bound nothing."""
    import rfx_b200
    rng = np.random.default_rng(m + n)
    cb, sb = _parts(rng, n, 72, fmt, spread=2)
    cb[n // 2: n // 2 + 20] = cb[0]
    sb[n // 2: n // 2 + 20] = sb[0]
    sb[7, 0] = 255 if fmt == "mxfp4" else 127
    which = rng.integers(0, n, m)
    which[0] = 0
    ca, sa = cb[which], sb[which]
    a, b = _matrix(ca, sa, 72, fmt), _matrix(cb, sb, 72, fmt)
    same = min(m, n)  # these are rows of b, themselves left out
    pick = np.unique(np.concatenate([[0, same - 1], rng.integers(0, same, 10)]))
    vb = ref.values(cb, sb, 1.0, fmt)
    for top in (64, 33):
        for got, at, va in ((rfx_b200.fp4_topk(a, b, top), None, ref.values(ca, sa, 1.0, fmt)),
                            (rfx_b200.fp4_topk(b.rows(0, same), b, top, self_offset=0), 0, vb)):
            rfx_b200.fp4_status()
            idx, val = (t.cpu().numpy() for t in got)
            for i in pick:
                wi, wv = ref.topk(va[i:i + 1], vb, top, None if at is None else int(i), fmt)
                assert np.array_equal(idx[i], wi[0]) and np.array_equal(val[i], wv[0]), (top, at, i)
