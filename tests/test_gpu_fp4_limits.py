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
