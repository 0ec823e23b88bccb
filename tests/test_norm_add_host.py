"""CPU tests of the residual norms' eps: it has no default, and None is none."""
import pytest


@pytest.mark.parametrize("name", ["rms_norm_add", "rms_norm_add_w8a8_quantize"])
def test_eps(mcv, name):
    import torch
    x, g = torch.zeros(3, 32, dtype=torch.float16), torch.zeros(32, dtype=torch.float16)
    with pytest.raises(mcv.McvError, match=f"^{name}: eps must be a number"):
        getattr(mcv, name)(x, x, g, None)
    with pytest.raises(TypeError):
        getattr(mcv, name)(x, x, g, "small")
    with pytest.raises(mcv.McvError, match="tensors must be on a GPU"):
        getattr(mcv, name)(x, x, g, 1e-6)
