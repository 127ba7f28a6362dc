"""Steps of the latent cache behind captured graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_captured_step_of_more_rows_leaves_the_live_rows_as_they_are(cuda_dev):
    from tests.test_gpu_decode_layer import layer_of
    layer, cache, g = layer_of(cuda_dev, 3, 12)
    h = torch.randn(12, 1024, generator=g, device=cuda_dev)
    cache.begin_step([4, 4, 4])
    layer.forward(h, cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward(h, cache)
    cache.begin_step([1, 1, 1])
    before = cache.rows.clone()
    new = cache.slots[:3].clone()
    h.copy_(torch.randn(12, 1024, generator=g, device=cuda_dev))
    graph.replay()
    changed = (cache.rows[0].view(-1, 576) != before[0].view(-1, 576)).any(1).nonzero()[:, 0]
    assert sorted(changed.tolist()) == sorted(new.tolist())
