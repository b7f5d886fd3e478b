"""The 4-bit operators as programs use them: together, on streams, captured into graphs, on views and
strided tensors, at the sizes that hold nothing, refused where they cannot run."""
import numpy as np
import pytest

import _fp4_ref as ref

pytestmark = pytest.mark.gpu


def _rows(rng, n, k):
    x = rng.normal(size=(n, k)).astype(np.float32) / np.sqrt(np.arange(1, k + 1, dtype=np.float32))
    x[rng.integers(0, n, n // 20)] = x[rng.integers(0, n, n // 20)]
    return x


def _answers(x, y, fmt, top):
    """(values of x, of y, product, indices, top values) from the definition."""
    vx, vy = (ref.values(*ref.quantize(t, fmt), fmt) for t in (x, y))
    return vx, vy, vx @ vy.T, *ref.topk(vx, vy, top, None, fmt)


def _check(got, want, k):
    vx, vy, p, idx, val = want
    assert np.array_equal(got[0].double().cpu().numpy(), vx)
    tol = k * 2.0 ** -23 * (np.abs(vx) @ np.abs(vy).T)
    tol = tol + 2.0 ** -24 * (np.abs(p) + tol)  # fp32 additions, one rounding
    assert (np.abs(got[1].double().cpu().numpy() - p) <= tol).all()
    assert np.array_equal(got[2].cpu().numpy(), idx) and np.array_equal(got[3].cpu().numpy(), val)


def _run(x, b, fmt, top):
    """New rows against stored ones: quantised, compared, their neighbours found."""
    import rfx_b200
    a = rfx_b200.fp4_quantize(x, format=fmt)
    return (a.dequantize(), rfx_b200.fp4_product(a, b), *rfx_b200.fp4_topk(a, b, top))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_together_on_streams(fmt):
    """Two streams at once, each with its own queries against the same stored rows."""
    import torch
    import rfx_b200
    rng = np.random.default_rng(3)
    y = _rows(rng, 3000, 48)
    qs = [_rows(rng, m, 48) for m in (5, 200)]
    b = rfx_b200.fp4_quantize(torch.from_numpy(y).cuda(), format=fmt)
    ts = [torch.from_numpy(q).cuda() for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _run(ts[i], b, fmt, 20)
    torch.cuda.synchronize()
    for g, q in zip(got, qs):
        _check(g, _answers(q, y, fmt, 20), 48)
    rfx_b200.fp4_status()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k", [(3, 2500, 64), (300, 2000, 64), (40, 900, 130), (16, 700, 256)])
def test_captured_and_replayed(fmt, m, n, k):
    """Two graphs of the same calls on different inputs, replayed in turn with new inputs."""
    import torch
    import rfx_b200
    rng = np.random.default_rng(m + n + k)
    y = _rows(rng, n, k)
    b = rfx_b200.fp4_quantize(torch.from_numpy(y).cuda(), format=fmt)
    xs = [torch.zeros(m, k, device="cuda") for _ in range(2)]
    _run(xs[0], b, fmt, 12)  # every kernel has run before
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_run(x, b, fmt, 12))
        graphs.append(g)
    for _ in range(2):
        data = [_rows(rng, m, k) for _ in range(2)]
        for x, d in zip(xs, data):
            x.copy_(torch.from_numpy(d))
        for i in (1, 0, 1):
            graphs[i].replay()
        torch.cuda.synchronize()
        for o, d in zip(outs, data):
            _check(o, _answers(d, y, fmt, 12), k)


def test_long_axis_captured():
    """The cluster form of the product, captured."""
    import torch
    import rfx_b200
    rng = np.random.default_rng(6)
    x, y = rng.normal(size=(9, 4200)).astype(np.float32), rng.normal(size=(300, 4200)).astype(np.float32)
    a, b = (rfx_b200.fp4_quantize(torch.from_numpy(t).cuda()) for t in (x, y))
    eager = rfx_b200.fp4_product(a, b)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = rfx_b200.fp4_product(a, b)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)  # the same sums every time


def test_views_and_strides():
    import torch
    import rfx_b200
    rng = np.random.default_rng(4)
    x = _rows(rng, 700, 61)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for pad, off in ((3, 0), (3, 1), (19, 3), (67, 8)):
            buf = torch.full((700, 61 + pad), float("nan"), device="cuda", dtype=dtype)
            view = buf[:, off:off + 61] if off + 61 <= 61 + pad else buf[:, :61]
            view.copy_(torch.from_numpy(x))
            a = rfx_b200.fp4_quantize(view)
            b = rfx_b200.fp4_quantize(view.contiguous())
            assert all(torch.equal(s, t) for s, t in zip(a.parts(), b.parts()))
        every_third = torch.from_numpy(x).cuda().to(dtype)[::3]
        a = rfx_b200.fp4_quantize(every_third)
        b = rfx_b200.fp4_quantize(every_third.contiguous())
        assert torch.equal(a.dequantize(), b.dequantize())
        for width in (61, 64, 70):
            for start in (0, 1, 4):
                out = torch.full((700, width + 4), -3.0, device="cuda", dtype=dtype)
                a2 = rfx_b200.fp4_quantize(torch.from_numpy(x).cuda())
                a2.dequantize(out=out[:, start:start + 61])
                assert torch.equal(out[:, start:start + 61], a2.dequantize(dtype))
                assert (out[:, :start] == -3).all() and (out[:, start + 61:] == -3).all()
    m = rfx_b200.fp4_quantize(torch.from_numpy(x).cuda())
    sub = m.rows(256, 600)
    assert torch.equal(sub.dequantize(), m.dequantize()[256:600])
    assert torch.equal(rfx_b200.fp4_product(sub, m), rfx_b200.fp4_product(m, m)[256:600])
    assert torch.equal(rfx_b200.fp4_product(m.rows(512, 520), m.rows(128, 400)), rfx_b200.fp4_product(m, m)[512:520, 128:400])


def test_nothing_in_them():
    import torch
    import rfx_b200
    e = torch.empty(0, 20, device="cuda")
    x = torch.randn(7, 20, device="cuda")
    for fmt in ("nvfp4", "mxfp4"):
        none, some = rfx_b200.fp4_quantize(e, format=fmt), rfx_b200.fp4_quantize(x, format=fmt)
        assert none.dequantize().shape == (0, 20) and none.parts()[0].shape == (0, 10)
        if fmt == "nvfp4":
            assert float(none.parts()[2]) == 1.0
        assert rfx_b200.fp4_product(none, some).shape == (0, 7) and rfx_b200.fp4_product(some, none).shape == (7, 0)
        idx, val = rfx_b200.fp4_topk(none, some, 4)
        assert idx.shape == (0, 4) and val.shape == (0, 4)
        idx, val = rfx_b200.fp4_topk(some, none, 4)
        assert (idx == -1).all() and torch.isneginf(val).all()
        p = some.parts()
        assert rfx_b200.Fp4Matrix.from_parts(p[0][:0], p[1][:0], p[2], cols=20, format=fmt).shape == (0, 20)
    zero = rfx_b200.fp4_quantize(torch.zeros(40, 33, device="cuda"))
    idx, val = rfx_b200.fp4_topk(zero, zero, 3, self_offset=0)  # all products equal: the lowest others
    want = np.array([[j for j in range(5) if j != i][:3] for i in range(40)])
    assert np.array_equal(idx.cpu().numpy(), want) and (val == 0).all()


def test_nan_rows_are_quick_and_alone():
    import torch
    import rfx_b200
    x = torch.randn(400, 64, device="cuda")
    x[5, 3] = float("nan")
    x[9, 60] = float("inf")
    m = rfx_b200.fp4_quantize(x)
    idx, val = rfx_b200.fp4_topk(m, m, 5, self_offset=0)
    assert (idx[5] == -1).all() and torch.isneginf(val[9]).all()
    assert not ((idx == 5) | (idx == 9)).any()
    keep = torch.ones(400, dtype=torch.bool)
    keep[[5, 9]] = False
    p = rfx_b200.fp4_product(m, m)
    assert torch.isnan(p[5]).all() and torch.isnan(p[:, 9]).all()
    assert not torch.isnan(p[keep][:, keep]).any()


def test_refusals_on_device():
    import torch
    import rfx_b200
    x = torch.randn(6, 40, device="cuda")
    with pytest.raises(TypeError, match="dtype"):
        rfx_b200.fp4_quantize(x.double())
    for bad in (x.t(), x[:, ::2], x[0], x[:1].expand(5, 40), torch.empty(3, 0, device="cuda")):
        with pytest.raises(ValueError):
            rfx_b200.fp4_quantize(bad)
    a, b, c = rfx_b200.fp4_quantize(x), rfx_b200.fp4_quantize(x, format="mxfp4"), rfx_b200.fp4_quantize(x[:, :39])
    for other in (b, c):
        with pytest.raises(ValueError, match="share"):
            rfx_b200.fp4_product(a, other)
        with pytest.raises(ValueError, match="share"):
            rfx_b200.fp4_topk(a, other, 2)
    for k in (0, 65, -1):
        with pytest.raises(ValueError, match="k must"):
            rfx_b200.fp4_topk(a, a, k)
    for off in (-1, 1):
        with pytest.raises(ValueError, match="self_offset"):
            rfx_b200.fp4_topk(a, a, 2, self_offset=off)
    wide = rfx_b200.fp4_quantize(torch.randn(3, 257, device="cuda"))
    with pytest.raises(ValueError, match="256"):
        rfx_b200.fp4_topk(wide, wide, 2)
    out = torch.empty(6, 6, device="cuda")
    for bad in (out.t()[:, :5], out.double(), out[:5], out.cpu(), out.expand(6, 6)[:, ::2], torch.empty(6, 1, device="cuda").expand(6, 6)):
        with pytest.raises(ValueError, match="out must"):
            rfx_b200.fp4_product(a, a, dtype=torch.float32, out=bad)
    with pytest.raises(ValueError, match="gradient"):
        rfx_b200.fp4_product(a, a, out=out.clone().requires_grad_())
    with pytest.raises(TypeError, match="dtype"):
        rfx_b200.fp4_product(a, a, dtype=torch.float64)
    with pytest.raises(ValueError, match="multiple of 128"):
        a.rows(1, 3)
    with pytest.raises(ValueError, match="not in"):
        a.rows(0, 7)
    p, s, g = a.parts()
    for args, kw in (((p[:, 1:], s, g), {}), ((p, s[:3], g), {}), ((p, s, -1.0), {}), ((p, s, float("inf")), {}),
                     ((p, s, g.double()), {}), ((p, s[:, :2], 2.0), {"format": "mxfp4"})):
        with pytest.raises(ValueError):
            rfx_b200.Fp4Matrix.from_parts(*args, cols=40, **kw)
    with pytest.raises(rfx_b200.RfxError, match="RFX_ERR_STATE"):
        ctx = rfx_b200.Context(0)
        ctx.lowrank_pack4("nvfp4")


def test_determinism():
    import torch
    import rfx_b200
    x = torch.randn(900, 100, device="cuda")
    m = rfx_b200.fp4_quantize(x)
    first = (m.dequantize(), rfx_b200.fp4_product(m, m), *rfx_b200.fp4_topk(m, m, 30, self_offset=0))
    for _ in range(3):
        n = rfx_b200.fp4_quantize(x)
        again = (n.dequantize(), rfx_b200.fp4_product(n, n), *rfx_b200.fp4_topk(n, n, 30, self_offset=0))
        assert all(torch.equal(s, t) for s, t in zip(first, again))


@pytest.mark.skipif("__import__('torch').cuda.device_count() < 2")
def test_another_device():
    import torch
    import rfx_b200
    x = torch.randn(300, 64, device="cuda:1")
    with torch.cuda.device(0):
        m = rfx_b200.fp4_quantize(x)
        got = (m.dequantize(), rfx_b200.fp4_product(m, m), *rfx_b200.fp4_topk(m, m, 9))
        assert torch.cuda.current_device() == 0 and all(t.device == x.device for t in got)
    rfx_b200.fp4_status(1)
    y = rfx_b200.fp4_quantize(x.to("cuda:0"))
    assert torch.equal(got[1].cpu(), rfx_b200.fp4_product(y, y).cpu())
