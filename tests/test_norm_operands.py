"""What the norm's wrapper refuses before any launch: no GPU is needed."""
import pytest
import torch


def norm(**k):
    from vic_b200 import kernels
    a = dict(hidden=torch.zeros(3, 64), delta=None, weight_f16=torch.ones(64, dtype=torch.float16), eps=1e-6, x_out=torch.zeros(3, 64, dtype=torch.bfloat16))
    a.update(k)
    kernels.residual_rms_norm(**a)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.int16])
def test_norm_weights_of_other_types(dtype):
    with pytest.raises(ValueError, match="norm weights"):
        norm(weight_f16=torch.ones(64, dtype=dtype))
