"""CPU-only checks of what the 4-bit matrices' Python layer does around its calls."""
import pytest

from rfx_b200 import fp4


def test_written_outputs_are_seen_by_autograd():
    """An ``out`` tensor that a graph has saved is known to have changed, as after any in-place call."""
    import torch
    fp4._load()
    cpu = torch.device("cpu")
    w, buf = torch.ones(3, 4, requires_grad=True), torch.ones(3, 4)
    y = (w * buf).sum()
    assert fp4._out(buf, (3, 4), torch.float32, cpu) is buf
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()
    before = buf._version
    with torch.inference_mode():
        fp4._out(buf, (3, 4), torch.float32, cpu)
        made_here = torch.ones(3, 4)
        assert fp4._out(made_here, (3, 4), torch.float32, cpu) is made_here
    assert buf._version > before
    with pytest.raises(ValueError, match="out must"):
        fp4._out(buf, (4, 3), torch.float32, cpu)


@pytest.mark.parametrize("mode,told", [("nvfp4", True), ("mxfp4", True), ("int8", False)])
def test_saving_tells_what_the_file_cannot_say(mode, told, monkeypatch, tmp_path):
    """The model file's only 4-bit code is nf4's: a 4-bit quant_mode is written as that, with a warning."""
    import warnings
    import rfx_b200
    from rfx_b200 import model_io
    written = []
    monkeypatch.setattr(model_io, "from_estimator", lambda est: {"of": est})
    monkeypatch.setattr(model_io, "write", lambda path, m: written.append((path, m["of"])))
    est = rfx_b200.RandomForestClassifier(quant_mode=mode, compute_proximity=True, use_qlora=True, rank=8)
    est._fitted = True
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        est.save(tmp_path / "m.rfx")
    assert [w for w in seen if "nf4" in str(w.message) and mode in str(w.message)] if told else not seen
    assert written == [(str(tmp_path / "m.rfx"), est)]
    plain = rfx_b200.RandomForestClassifier(quant_mode=mode)  # no low-rank factors: nothing is lost
    plain._fitted = True
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        plain.save(tmp_path / "m.rfx")


def test_views_take_any_whole_numbers():
    """Bounds from numpy or torch make the view that plain ones make; others are refused."""
    import numpy as np
    import torch
    from rfx_b200 import _abi as A
    fp4._load()
    m = object.__new__(fp4.Fp4Matrix)  # of made-up addresses: nothing here reads them
    m.format, m.shape, m.device = "nvfp4", (400, 64), torch.device("cpu")
    m._pitch, m._tile_bytes, m._keep = 32, 512, torch.zeros(4)
    m._set(A.Fp4Struct(1, 400, 64, 1 << 20, 2 << 20, 3 << 20, 4 << 20))
    want = m.rows(128, 300)
    for begin, end in ((np.int64(128), np.int32(300)), (torch.tensor(128), torch.tensor(300))):
        got = m.rows(begin, end)
        assert got.shape == want.shape == (172, 64)
        assert all(getattr(got._c, f) == getattr(want._c, f) for f, _ in A.Fp4Struct._fields_)
    for begin, end in ((128.0, 300), (0, 300.5), ("0", 300)):
        with pytest.raises(TypeError, match="integer"):
            m.rows(begin, end)
    for begin, end in ((np.int64(128), np.int64(401)), (np.int64(-128), 5), (np.int64(64), 100)):
        with pytest.raises(ValueError):
            m.rows(begin, end)
