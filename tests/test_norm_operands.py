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


z = torch.zeros


@pytest.mark.parametrize("name,bad", [
    # fewer rows or columns than the hidden state has: the launch would write or read behind them
    ("x_out", z(2, 64)), ("x_out", z(3, 60)), ("x_out", z(64)), ("x_out", z(64, 3).t()), ("x_out", z(1, 64).expand(3, 64)),
    ("x_out", z(3, 64, dtype=torch.float64)),
    ("delta", z(2, 64)), ("delta", z(3, 32)), ("delta", z(64)), ("delta", z(64, 3).t()), ("delta", z(3, 64, dtype=torch.float64)),
    ("delta2", z(2, 64)), ("delta2", z(3, 64, dtype=torch.bfloat16)), ("delta2", z(64, 3).t()),
    ("weight_f16", z(63, dtype=torch.float16)), ("weight_f16", z(128, dtype=torch.float16)[::2]),
    # (rows of 16-bit values would be written as floats, beyond the tensor)
    ("hidden", z(3, 64, dtype=torch.bfloat16)), ("hidden", z(3, 64, dtype=torch.float16)), ("hidden", z(64, 3).t()), ("hidden", z(64))])
def test_norm_operands_that_do_not_fit_the_hidden_state(name, bad):
    with pytest.raises(ValueError, match="hidden|norm weights"):
        norm(**{name: bad})


@pytest.mark.parametrize("change", [
    {"x_out": z(4, 64)}, {"x_out": z(3, 72, dtype=torch.float16)}, {"delta": z(5, 64, dtype=torch.bfloat16)}, {"delta": z(1, 64).expand(3, 64)},
    {"delta2": z(3, 80)}, {"weight_f16": z(80, dtype=torch.float16)}, {"weight_f16": None},
    {"hidden": z(1, 64), "x_out": z(64), "delta": z(64), "delta2": z(64)}, {"hidden": z(3, 128)[:, 64:]}])
def test_larger_buffers_and_single_rows_pass_the_comparison(change):
    """What is refused here is the device: every operand lies on the CPU."""
    with pytest.raises(ValueError, match="device tensor"):
        norm(**change)


@pytest.mark.gpu
def test_a_hidden_state_on_another_device_than_the_current_one(cuda_dev, monkeypatch):
    from vic_b200 import kernels
    a = {n: torch.zeros(3, 64, device=cuda_dev) for n in ("hidden", "x_out")}
    norm(**a, weight_f16=None)
    monkeypatch.setattr(kernels, "_current_device", lambda: 1)
    with pytest.raises(ValueError, match="current device"):
        norm(**a, weight_f16=None)
