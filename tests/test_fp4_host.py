"""CPU-only checks of the 4-bit matrices' boundary: refusals of the C ABI and of the Python calls
(all before any device work), the layout that the Python side computes, quant_mode."""
import ctypes as C

import numpy as np
import pytest

import _fp4_ref as ref
import rfx_b200
from rfx_b200 import _abi as A
from rfx_b200 import fp4

ERR_ARG, ERR_UNSUPPORTED = -1, -4


def _matrix(format=1, rows=4, cols=64, codes=1024, scales=2048, scale=4096, bounds=8192):
    """A matrix of made-up device addresses: nothing here may reach them."""
    return A.Fp4Struct(format, rows, cols, codes, scales, scale, bounds)


def _fails(rc, text, code=ERR_ARG):
    assert rc == code, rc
    assert text in A.load_library().rfx_last_error().decode(), A.load_library().rfx_last_error()


def test_sizes():
    L = A.load_library()
    lay = A.Fp4Layout()
    for f, name in ((0, "mxfp4"), (1, "nvfp4")):
        for rows in (0, 1, 128, 129, 5000):
            for cols in (1, 16, 63, 64, 65, 128, 129, 256, 257, 4095):
                assert L.rfx_fp4_sizes(f, rows, cols, C.byref(lay)) == 0
                padded, tiles = (cols + 63) // 64 * 64, (rows + 127) // 128
                assert lay.pitch == padded // 2 and lay.codes == rows * lay.pitch
                assert lay.tile_bytes == 512 * (padded // 64 if name == "nvfp4" else (padded + 127) // 128)
                assert lay.scales == tiles * lay.tile_bytes and lay.scale == 8
                assert lay.bounds == (4 * tiles if padded <= 256 else 0)
    _fails(L.rfx_fp4_sizes(2, 1, 1, C.byref(lay)), "format")
    _fails(L.rfx_fp4_sizes(0, -1, 1, C.byref(lay)), "rows")
    _fails(L.rfx_fp4_sizes(0, 1, 0, C.byref(lay)), "cols")
    _fails(L.rfx_fp4_sizes(0, 1, 1 << 25, C.byref(lay)), "cols")
    _fails(L.rfx_fp4_sizes(0, 1, 1, None), "null")


def test_largest_shapes():
    """Rows and columns beyond a 32-bit count or a launch's grid are refused, not cut short."""
    L = A.load_library()
    lay = A.Fp4Layout()
    assert L.rfx_fp4_sizes(1, fp4.MAX_ROWS, fp4.MAX_COLS, C.byref(lay)) == 0
    assert lay.codes == fp4.MAX_ROWS * (fp4.MAX_COLS // 2)
    _fails(L.rfx_fp4_sizes(1, fp4.MAX_ROWS + 1, 1, C.byref(lay)), "rows")
    _fails(L.rfx_fp4_sizes(1, 1, fp4.MAX_COLS + 1, C.byref(lay)), "cols")
    for rows, cols in ((fp4.MAX_ROWS + 1, 1), (2 ** 32 + 3, 64), (1, fp4.MAX_COLS + 1), (1, 0)):
        with pytest.raises(ValueError, match="at most"):
            fp4._check_shape(rows, cols)


def test_abi_refusals():
    L = A.load_library()
    at = C.addressof
    m, other, wide, mx = _matrix(), _matrix(cols=63), _matrix(cols=300), _matrix(format=0)
    _fails(L.rfx_fp4_quantize(64, 0, 64, None, None), "null matrix")
    _fails(L.rfx_fp4_quantize(64, 3, 64, at(m), None), "dtype")
    _fails(L.rfx_fp4_quantize(64, 0, 63, at(m), None), "row_stride")
    _fails(L.rfx_fp4_quantize(None, 0, 64, at(m), None), "x is null")
    _fails(L.rfx_fp4_quantize(66, 0, 64, at(m), None), "unaligned")
    for bad in (_matrix(codes=8), _matrix(scales=0), _matrix(scale=4), _matrix(bounds=0), _matrix(format=5), _matrix(cols=0)):
        assert L.rfx_fp4_quantize(64, 0, 64, at(bad), None) == ERR_ARG
    _fails(L.rfx_fp4_dequantize(at(m), 0, 5, 64, 0, 64, None), "row range")
    _fails(L.rfx_fp4_dequantize(at(m), 3, 2, 64, 0, 64, None), "row range")
    _fails(L.rfx_fp4_dequantize(at(m), 0, 4, 64, 0, 63, None), "ld")
    _fails(L.rfx_fp4_dequantize(at(m), 0, 4, None, 0, 64, None), "out is null")
    _fails(L.rfx_fp4_pack(None, 64, None, at(m), None), "null codes")
    _fails(L.rfx_fp4_unpack(at(m), None, 64, None), "null output")
    _fails(L.rfx_fp4_product(at(m), at(other), 64, 0, 64, None), "share")
    _fails(L.rfx_fp4_product(at(m), at(mx), 64, 0, 64, None), "share")
    _fails(L.rfx_fp4_product(at(m), at(m), 64, 9, 64, None), "dtype")
    _fails(L.rfx_fp4_product(at(m), at(m), 64, 0, 3, None), "ld")
    need = C.c_longlong()
    _fails(L.rfx_fp4_topk_workspace(at(m), at(m), 0, C.byref(need)), "k must be")
    _fails(L.rfx_fp4_topk_workspace(at(m), at(m), 65, C.byref(need)), "k must be")
    _fails(L.rfx_fp4_topk_workspace(at(wide), at(wide), 5, C.byref(need)), "256 columns", ERR_UNSUPPORTED)
    _fails(L.rfx_fp4_topk(at(m), at(m), 5, 1, 64, 64, None, 0, None), "self must be")
    _fails(L.rfx_fp4_topk(at(m), at(m), 5, -2, 64, 64, None, 0, None), "self must be")
    _fails(L.rfx_fp4_topk(at(m), at(m), 5, -1, None, 64, None, 0, None), "null or unaligned output")
    _fails(L.rfx_lowrank_pack4(None, 1), "null context")
    _fails(L.rfx_lowrank4_topk(None, 1, 0, 1, None, None), "null context")


def test_python_refusals():
    import torch
    x = torch.zeros(3, 4)
    with pytest.raises(TypeError, match="CUDA"):
        rfx_b200.fp4_quantize(x)
    with pytest.raises(TypeError, match="CUDA"):
        rfx_b200.fp4_quantize(np.zeros((3, 4), np.float32))
    with pytest.raises(ValueError, match="format"):
        rfx_b200.fp4_quantize(x, format="nf4")
    with pytest.raises(TypeError):
        rfx_b200.Fp4Matrix()
    with pytest.raises(TypeError, match="uint8"):
        rfx_b200.Fp4Matrix.from_parts(x, x, cols=4)
    with pytest.raises(ValueError, match="format"):
        rfx_b200.Fp4Matrix.from_parts(x, x, cols=4, format="int8")
    with pytest.raises(ValueError, match="cols"):
        rfx_b200.Fp4Matrix.from_parts(x, x, cols=0)
    for f in (rfx_b200.fp4_product, lambda a, b: rfx_b200.fp4_topk(a, b, 3)):
        with pytest.raises(TypeError, match="Fp4Matrix"):
            f(x, x)


def test_quant_mode():
    ok = dict(compute_proximity=True, use_qlora=True, rank=8)
    for mode in ("int8", "nvfp4", "mxfp4", "NVFP4"):
        e = rfx_b200.RandomForestClassifier(quant_mode=mode, **ok)
        assert e._lowrank4() == (None if mode == "int8" else mode.lower())
    with pytest.raises(NotImplementedError, match="nvfp4"):
        rfx_b200.RandomForestClassifier(quant_mode="nf4", **ok)
    with pytest.raises(NotImplementedError, match="rank"):
        rfx_b200.RandomForestClassifier(quant_mode="nvfp4", compute_proximity=True, use_qlora=True, rank=65)
    assert fp4.FORMATS is A.FP4_FORMATS


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_reference_quantiser(fmt):
    """The checker itself: every value within half a step of its code's neighbours, scales minimal."""
    rng = np.random.default_rng(1)
    x = rng.normal(size=(50, 70)).astype(np.float32) * np.exp(rng.normal(size=(50, 1)))
    codes, scales, g = ref.quantize(x, fmt)
    v = ref.values(codes, scales, g, fmt)
    assert np.array_equal(ref.unpack(ref.pack(codes), 70), codes)
    bs = ref.BLOCK[fmt]
    for b in range(scales.shape[1]):
        s = ref.values(np.full((50, 1), 2, np.uint8), scales[:, b:b + 1], g, fmt)  # the scale: code 2 is 1
        blk, vb = x[:, b * bs:(b + 1) * bs], v[:, b * bs:(b + 1) * bs]
        amax = np.abs(blk).max(1, keepdims=True)
        if fmt == "mxfp4":
            assert (amax <= 6 * s).all() and (amax > 3 * s).all()
        else:
            assert (np.abs(amax / 6 - s) <= s / 16).all()
        step = np.where(np.abs(vb) >= 4 * s, 2, np.where(np.abs(vb) >= 2 * s, 1, 0.5)) * s
        assert (np.abs(blk - vb) <= step / 2 + 1e-12).all()
