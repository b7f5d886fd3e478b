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
