"""The 4-bit operators at the ends of what they accept: matrix scales, roundings, memory on other
streams, row blocks, the routes of the selection."""
import numpy as np
import pytest

import _fp4_ref as ref

pytestmark = pytest.mark.gpu


def _dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _random(rng, rows, cols, fmt, spread=2):
    """Random codes and scale bytes, scales within 2^spread of 1."""
    nb = -(-cols // ref.BLOCK[fmt])
    codes = rng.integers(0, 16, (rows, cols)).astype(np.uint8)
    mid, unit = (127, 1) if fmt == "mxfp4" else (56, 8)
    return codes, rng.integers(mid - spread * unit, mid + spread * unit + 1, (rows, nb)).astype(np.uint8)


def _matrix(codes, scales, cols, fmt, g=None):
    import rfx_b200
    return rfx_b200.Fp4Matrix.from_parts(_dev(ref.pack(codes)), _dev(scales), g, cols=cols, format=fmt)


@pytest.mark.parametrize("g", [-1.0, -0.0, 0.0, float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("m", [3, 300, 4000])
def test_matrix_scale_that_is_not_positive(m, g):
    """A scale on the device cannot be refused without waiting for it: it makes every value NaN, on
    either side, and NaN rows are nobody's neighbours."""
    import torch
    import rfx_b200
    rng = np.random.default_rng(m)
    k = 40
    a = _matrix(*_random(rng, m, k, "nvfp4"), k, "nvfp4")
    c, s = _random(rng, 4500, k, "nvfp4")
    good = _matrix(c, s, k, "nvfp4", 0.5)
    bad = _matrix(c, s, k, "nvfp4", torch.tensor([g], device="cuda"))
    assert torch.isnan(bad.dequantize()).all() and torch.isnan(bad.dequantize(torch.float16)).all()
    assert torch.isnan(bad.parts()[2]).all()
    for x, y in ((a, bad), (bad.rows(0, m), good)):
        assert torch.isnan(rfx_b200.fp4_product(x, y)).all()
        idx, val = rfx_b200.fp4_topk(x, y, 7)
        assert (idx == -1).all() and torch.isneginf(val).all()
    idx, _ = rfx_b200.fp4_topk(a, good, 7)
    assert (idx >= 0).all()
    rfx_b200.fp4_status()


def _round(v, bits, emin):
    """v (64 bits) to the nearest number of `bits` significant bits, ties to even, with the
    exponent of the smallest normal number emin."""
    e = np.maximum(np.frexp(v)[1] - 1, emin)
    q = np.ldexp(1.0, e - bits + 1)
    return np.rint(v / q) * q


@pytest.mark.parametrize("dtype,bits,emin", [("bfloat16", 8, -126), ("float16", 11, -14), ("float32", 24, -126)])
def test_dequantize_rounds_once(dtype, bits, emin):
    """Matrix scales that are no powers of two, chosen so that code x scale x matrix scale lies next to
    the middle of two numbers of the type: rounding to fp32 on the way would land on it."""
    import torch
    codes = np.tile(np.arange(16, dtype=np.uint8), (126, 1))
    scales = np.arange(1, 127, dtype=np.uint8)[:, None]
    x = ref.values(codes, scales, 1.0, "nvfp4")  # at most 6 significant bits
    twice = 0
    for lo in (1.0, 2.0 ** (emin + 1), 2.0 ** (emin - 3)):
        # middles of neighbours near lo, one in three above: no multiples of 3
        q = 2.0 ** (max(np.frexp(lo)[1] - 1, emin) - bits + 1)
        for i in (0, 1, 2, 4, 5, 9):
            for base in (3.0, 0.1015625):  # values among x
                g = np.float32((lo + (i + 0.5) * q) / base)
                if not 2.0 ** -126 <= g < 2.0 ** 100:
                    continue
                v = x * np.float64(g)  # 30 bits: exact
                want = _round(v, bits, emin)
                with np.errstate(over="ignore"):
                    want = np.where(np.abs(want) > float(torch.finfo(getattr(torch, dtype)).max), np.copysign(np.inf, want), want)
                    twice += int((_round(_round(v, 24, -126), bits, emin) != _round(v, bits, emin)).sum())
                got = _matrix(codes, scales, 16, "nvfp4", float(g)).dequantize(getattr(torch, dtype))
                got = got.double().cpu().numpy()
                bad = np.argwhere(got != want)
                assert len(bad) == 0, (lo, i, base, len(bad), got[tuple(bad[0])], want[tuple(bad[0])], v[tuple(bad[0])])
    assert dtype == "float32" or twice > 0  # a second rounding would have been seen


def test_product_rows_in_several_blocks():
    """get_lowrank_product over more rows than one block holds: the scratch stays within 256 MB (128
    rows, where those take more), whatever the first row, and the rows are the same."""
    import torch
    import rfx_b200
    from _helpers import synth
    n = 300000  # a block of 256 MB: 223 rows
    X, y = synth("class", n, 6, 3)
    est = rfx_b200.RandomForestClassifier(nsample=n, ntree=2, mdim=6, mtry=2, compute_proximity=True, compute_importance=False,
                                          use_qlora=True, quant_mode="nvfp4", rank=8, show_progress=False)
    est.fit(X, y)
    A = est.get_lowrank_factors()[0]
    rfx_b200.empty_cache()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    P = est.get_lowrank_product(100, 400)
    used = before - torch.cuda.mem_get_info()[0]
    assert P.shape == (300, n)
    for r0, r1 in ((100, 101), (127, 129), (255, 390)):
        assert np.array_equal(est.get_lowrank_product(r0, r1), P[r0 - 100:r1 - 100])
    for r0 in range(100, 400, 50):
        a = A[r0:r0 + 50]
        want = a @ A.T
        # 8 fp32 additions of exact terms, one rounding
        tol = 8 * 2.0 ** -23 * (np.abs(a) @ np.abs(A).T) + 2.0 ** -24 * np.abs(want)
        assert (np.abs(P[r0 - 100:r0 - 50] - want) <= tol).all()
    assert used <= (256 + 8) << 20, used


def test_memory_used_on_another_stream():
    """A matrix made on one stream, used on another and dropped: after record_stream its memory is not
    given out again before the other stream is done."""
    import torch
    import rfx_b200
    made, used = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(made):
        x = torch.randn(3000, 64, device="cuda")
        m = rfx_b200.fp4_quantize(x)
        want = m.dequantize()
        torch.full((1,), 255, dtype=torch.uint8, device="cuda")  # loading a kernel waits for the device
    used.wait_stream(made)
    torch.cuda.synchronize()
    where, size = m._keep.data_ptr(), m._keep.numel()
    with torch.cuda.stream(used):
        torch.cuda._sleep(200_000_000)  # about a tenth of a second
        view = m.rows(0, 3000)
        got = view.dequantize()
        view.record_stream(used)
    del m, view
    with torch.cuda.stream(made):
        new = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(3)]
    assert not used.query()  # the other stream was still at work
    assert where not in [t.data_ptr() for t in new]
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_errors_reach_their_own_callers():
    """The device's status word belongs to the calls without a context: an error in it is neither
    raised nor erased by an estimator's calls, and rfx_fp4_status reports it once."""
    import ctypes as C
    import torch
    import rfx_b200
    from rfx_b200.shard import _DeviceInts
    from _helpers import synth
    X, y = synth("class", 500, 6, 3)
    est = rfx_b200.RandomForestClassifier(nsample=500, ntree=4, mdim=6, mtry=2, compute_proximity=True, compute_importance=False,
                                          use_qlora=True, quant_mode="mxfp4", rank=8, show_progress=False)
    est.fit(X, y)
    first = (*est.get_lowrank_topk(5), est.get_lowrank_product(3, 9))
    at = C.c_void_p()
    assert rfx_b200.load_library().rfx_fp4_status_word(C.byref(at)) == 0
    word = torch.as_tensor(_DeviceInts(at.value, 1), device="cuda")
    rfx_b200.fp4_status()
    assert int(word) == 0
    word.fill_(5)  # as a kernel on another stream would
    torch.cuda.synchronize()
    again = (*est.get_lowrank_topk(5), est.get_lowrank_product(3, 9))
    assert all(np.array_equal(s, t) for s, t in zip(first, again))
    assert int(word) == 5
    with pytest.raises(rfx_b200.RfxError, match="code 5"):
        rfx_b200.fp4_status()
    rfx_b200.fp4_status()
    assert int(word) == 0


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_values_at_the_ends_of_the_range(fmt):
    """Next to the largest float the nearest code can stand for 2^128 or more, and nvfp4's smallest
    values have more bits than bf16 has there: each type gets the value, rounded once."""
    import torch
    import rfx_b200
    f = np.finfo(np.float32)
    tops = [2.8e38, 2.92e38, 2.93e38, 3.5 * 2.0 ** 126, 3.0e38, 2016 * 2.0 ** 117, 3.36e38, float(f.max)]
    for top in tops:
        x = np.zeros((3, 64), np.float32)
        x[0, ::3], x[1, 40:] = np.float32(top), -np.float32(top) * np.float32(0.87)
        x[2] = 1.0
        codes, scales, g = ref.quantize(x, fmt)
        v = ref.values(codes, scales, g, fmt)
        m = rfx_b200.fp4_quantize(torch.from_numpy(x).cuda(), format=fmt)
        assert np.array_equal(m.parts()[1].cpu().numpy(), scales)
        for dtype in (torch.float32, torch.bfloat16):
            got = m.dequantize(dtype).double().cpu().numpy()
            want = np.where(np.abs(v) >= 2.0 ** 128, np.copysign(np.inf, v), v)
            assert np.array_equal(got, want), (top, dtype)
            assert np.isfinite(got[np.abs(x) < 2.9e38]).all()
    rng = np.random.default_rng(5)
    for top in (2.0 ** -117, 2.0 ** -120, 2.0 ** -126, 2.0 ** -130):
        x = (rng.uniform(-top, top, (40, 64)) * 2.0 ** -rng.integers(0, 16, (40, 1)).astype(np.float64)).astype(np.float32)
        codes, scales, g = ref.quantize(x, fmt)
        v = ref.values(codes, scales, g, fmt)
        m = rfx_b200.fp4_quantize(torch.from_numpy(x).cuda(), format=fmt)
        assert np.array_equal(m.dequantize().double().cpu().numpy(), v)
        half = m.dequantize(torch.bfloat16).double().cpu().numpy()
        assert np.array_equal(half, _round(v, 8, -126))
        held = np.abs(v) >= 2.0 ** -128 if fmt == "nvfp4" else np.ones_like(v, bool)
        assert np.array_equal(half[held], v[held])


def test_matrix_scale_numbers_that_fp32_cannot_hold():
    """A number is checked as it is kept: one that rounds to 0 or infinity in fp32 is refused."""
    rng = np.random.default_rng(1)
    c, s = _random(rng, 3, 40, "nvfp4")
    top = float(np.finfo(np.float32).max)  # 2^128 (1 - 2^-24); from 2^128 (1 - 2^-25) on numbers round to infinity
    for g in (1e39, 1e-50, 2.0 ** -151, 2.0 ** 128 * (1 - 2.0 ** -25), -1e-50, 0.0, float("nan")):
        with pytest.raises(ValueError, match="positive and finite"):
            _matrix(c, s, 40, "nvfp4", g)
    # (1 - 2^-24) (1 + 2^-25) = 1 - 2^-25 - 2^-49: below that border, so it rounds to the largest number
    for g, kept in ((2.0 ** -149, 2.0 ** -149), (top, top), (top * (1 + 2.0 ** -25), top)):
        assert float(_matrix(c, s, 40, "nvfp4", g).parts()[2]) == kept


def test_matrix_scale_of_a_negated_view():
    """A lazily negated tensor (the imaginary part of a conjugate is one) counts by its value."""
    import torch
    rng = np.random.default_rng(2)
    c, s = _random(rng, 5, 40, "nvfp4")
    g = torch.tensor([1 - 0.375j], device="cuda").conj().imag
    assert g.is_neg() and float(g) == 0.375
    m = _matrix(c, s, 40, "nvfp4", g)
    assert float(m.parts()[2]) == 0.375
    assert np.array_equal(m.dequantize().double().cpu().numpy(), ref.values(c, s, 0.375, "nvfp4"))
