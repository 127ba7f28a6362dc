"""The norm before a sublayer with weights of either 16-bit type, against its formula in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,T", [(1024, 3), (7168, 1), (200, 2), (9000, 2), (1026, 1)])
@pytest.mark.parametrize("weights", [torch.float16, torch.bfloat16])
def test_norm_weights_of_both_16_bit_types(cuda_dev, H, T, weights):
    """fp32 out: the sum of squares takes at most 9 + 16 additions in a row in any of the forms, the rest some five roundings; 64 2^-24 covers them."""
    from vic_b200 import kernels
    g = torch.Generator(device=cuda_dev).manual_seed(H + T)
    h = 2 * torch.randn(T, H, generator=g, device=cuda_dev)
    delta = (0.3 * torch.randn(T, H, generator=g, device=cuda_dev)).to(torch.bfloat16)
    w = (1 + 0.1 * torch.randn(H, generator=g, device=cuda_dev)).to(weights)
    w[5], w[H - 2] = -0.75, 0.0
    if weights is torch.bfloat16:
        w[6], w[7] = 2.0 ** -40, 2.0 ** 20                # beyond what fp16 holds
    want_h = h + delta.float()
    for center in (False, True):
        x, hid = torch.zeros(T, H, device=cuda_dev), h.clone()
        kernels.residual_rms_norm(hid, delta, w, 1e-6, x, center=center)
        assert torch.equal(hid, want_h)
        d = want_h.double()
        off = d.mean(1, keepdim=True) if center else 0.0
        want = (d - off) / ((d - off).square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
        slack = 2.0 ** -20 * w.double().abs() if center else 0.0        # (of the mean: values of magnitude 2 to 8 added up in fp32)
        assert bool(((x.double() - want).abs() <= 64 * 2.0 ** -24 * want.abs() + slack).all())


def test_a_decode_layer_with_norms_of_its_own_type(cuda_dev):
    from tests.test_gpu_decode_layer import layer_of
    layer, cache, g = layer_of(cuda_dev, 3, 12)
    layer.attention_norm, layer.moe_norm = layer.attention_norm.to(torch.bfloat16), layer.moe_norm.to(torch.bfloat16)
    cache.begin_step([2, 1, 2])
    h = torch.randn(6, 1024, generator=g, device=cuda_dev)
    before = h.double()
    layer.forward(h, cache)
    att = layer.attention
    x = before / (before.square().mean(1, keepdim=True) + 1e-6).sqrt() * layer.attention_norm.double()
    kv = x @ att.w_kv.double().T          # (x is rounded to bf16 before the product, and so is the product)
    bound = 2.0 ** -8 * (x.abs() @ att.w_kv.double().abs().T) + 2.0 ** -8 * kv.abs() + 1e-5
    assert bool(((att.kv_in[:6].double() - kv).abs() <= bound).all())
    mid = before + att.out[:6].double()
    x = mid / (mid.square().mean(1, keepdim=True) + 1e-6).sqrt() * layer.moe_norm.double()
    assert bool(((layer.x[:6].double() - x).abs() <= 2.0 ** -8 * x.abs() + 1e-5).all())
