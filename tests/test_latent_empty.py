"""Calls without tokens launch nothing, whatever their addresses: an empty tensor's is null.  No GPU is needed but where marked."""
import pytest
import torch

from tests.test_latent_refusals import append, attention, query, value


def test_launchers_with_null_rows():
    assert append(n_tokens=0, kv=0, positions=0, slots=0) == 0
    assert query(n_tokens=0, q=0, positions=0, out=0) == 0
    assert value(n_tokens=0, o=0, out=0) == 0
    assert attention(q_len=0, q=0, out=0) == 0
    assert attention(batch=0, q=0, table=0, lens=0, out=0) == 0
    # what is no row of a token is looked at as before
    assert append(n_tokens=0, kv_dtype=7, kv=0, positions=0, slots=0) == -1
    assert query(n_tokens=0, nope=24, q=0, positions=0, out=0) == -1
    assert attention(q_len=0, q=0, out=0, workspace_bytes=8) == -8


def test_a_layer_of_a_step_without_tokens(monkeypatch):
    from tests.test_decode_layer_refusals import Grouped, Single, parts
    for moe in (Grouped(128), Single()):
        layer, cache, launched = parts(monkeypatch, moe, 24, 12)
        h = torch.ones(0, 64)
        assert layer.forward(h, cache) is h                  # before the first step, too
        cache.begin_step([1, 0, 0])
        cache.begin_step([0, 0, 0])
        assert layer.forward(h, cache) is h and layer.attention.forward(torch.ones(0, 64, dtype=torch.bfloat16), cache, 0).shape == (0, 64)
        with pytest.raises(ValueError, match="rows"):
            layer.forward(torch.ones(1, 64), cache)
        assert launched == []


@pytest.mark.gpu
def test_wrappers_with_empty_tensors(cuda_dev):
    from vic_b200 import kernels as K
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=cuda_dev)  # noqa: E731
    i32, f = torch.int32, torch.ones(32, dtype=torch.float64, device=cuda_dev)
    cache, status = z(2, 8, 576), z(1, dtype=i32)
    ws = torch.empty(K.latent_attention_workspace_bytes(), dtype=torch.uint8, device=cuda_dev)
    K.latent_append(z(4, 576)[:0], z(512), 1e-6, z(4, dtype=i32)[:0], z(0, dtype=torch.int64), f, cache, status=status)
    K.latent_query(z(0, 4, 192), z(4, 128, 512), z(0, dtype=i32), f, z(0, 4, 576), status=status)
    K.latent_value(z(0, 4, 512), z(4, 128, 512), z(0, 4, 128), status=status)
    K.latent_attention(z(0, 4, 576), cache, z(2, 3, dtype=i32), z(2, dtype=i32), 0.1, z(0, 4, 512), z(0, 4, dtype=torch.float32), workspace=ws, status=status)
    K.latent_attention(z(0, 4, 576), cache, z(0, 3, dtype=i32), z(0, dtype=i32), 0.1, z(0, 4, 512), workspace=ws, status=status)
    assert int(status) == 0 and not bool(cache.any())
