"""The router's selection bias through a decode layer: it moves which experts are chosen, not their weights."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sequences,new", [(1, [1]), (3, [4, 2, 4]), (3, [1, 1, 1])])
def test_a_selection_bias_reaches_the_router(cuda_dev, oracle, sequences, new):
    from tests.test_gpu_decode_layer import layer_of
    from vic_b200.attention import DecodeLayer
    plain, cache, g = layer_of(cuda_dev, sequences, 1 if sequences == 1 else 12)
    model = plain.moe.model
    sh = model.shape
    bias = torch.tensor([0.0, 5.0, 0.0, 0.3, -5.0, 0.0], device=cuda_dev)
    layer = DecodeLayer(plain.attention, plain.moe, 0, plain.attention_norm, plain.moe_norm, selection_bias=bias)
    cache.begin_step(new)
    T = cache.step_rows
    start = torch.randn(T, sh.hidden, generator=g, device=cuda_dev)
    h = start.clone()
    layer.forward(h, cache)
    moe = layer.moe
    ids = (moe.ids[None] if sequences == 1 else moe.ids)[:T, :sh.top_k].cpu().numpy().view(np.uint16)
    ws = (moe.weights[None] if sequences == 1 else moe.weights)[:T, :sh.top_k].cpu().numpy()
    x, moved = layer.x[:T].float().cpu().numpy(), 0
    for t in range(T):
        oi, ow, _ = oracle.router(x[t], model.router_w[0].cpu().numpy(), sh.top_k, sh.scoring, sh.scaling_factor, sh.normalize, bias.cpu().numpy(),
                                  oracle.ORDER_SEQUENTIAL)
        assert np.array_equal(ids[t], oi) and np.allclose(ws[t], ow, rtol=1e-5), t
        assert oi[0] == 1 and 4 not in oi
        ui, _, _ = oracle.router(x[t], model.router_w[0].cpu().numpy(), sh.top_k, sh.scoring, sh.scaling_factor, sh.normalize)
        moved += sorted(ui.tolist()) != sorted(oi.tolist())
    assert moved
    mid = start + layer.attention.out[:T].float()
    if sequences == 1:
        own = moe.forward_layer(0, layer.x[0], bias=bias)[None]
    else:
        own = moe.forward(0, layer.x[:T], bias=bias)
    torch.testing.assert_close(h, mid + own, rtol=1e-6, atol=1e-5)
    assert int(moe.status) == 0
