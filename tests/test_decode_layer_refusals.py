"""What DecodeLayer refuses, before its first launch and before anything has changed: no GPU is needed."""
import pytest
import torch


class Model:
    def __init__(self, hidden=64, n_layers=1):
        self.shape, self.n_layers = type("Shape", (), {"hidden": hidden, "num_experts": 6}), n_layers
        self.router_w = torch.zeros(n_layers, 6, hidden)


class Grouped:
    """Stands for a GroupedDecoder: DecodeLayer tells the two kinds of decoders apart by max_tokens."""
    def __init__(self, max_tokens, model=None):
        self.max_tokens, self.model = max_tokens, model or Model()

    def forward(self, *a, **k):
        raise AssertionError("reached")


class Single:
    model = Model()

    def forward_layer(self, *a, **k):
        raise AssertionError("reached")


def parts(monkeypatch, moe, cache_tokens, layer_tokens, sequences=3):
    """A layer on the CPU whose launches are recorded instead of made."""
    from vic_b200 import attention, kernels
    from vic_b200.core_types import LatentShape
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    cache = attention.LatentCache(1, 60, 8, sequences, 20, torch.bfloat16, "cpu", cache_tokens)
    sh = LatentShape("small", 64, 2, 16, 16, 10000.0, 1e-6)
    att = attention.LatentAttention(sh, z(2 * 80, 64), z(576, 64), z(512), z(2, 32, 512), z(64, 32), max_tokens=layer_tokens,
                                    workspace=torch.zeros(16, dtype=torch.uint8))
    launched = []
    for name in ("residual_rms_norm", "latent_append", "latent_query", "latent_attention", "latent_value"):
        monkeypatch.setattr(kernels, name, lambda *a, name=name, **k: launched.append(name))
    return attention.DecodeLayer(att, moe, 0, z(64), z(64)), cache, launched


@pytest.mark.parametrize("moe,cache_tokens,layer_tokens,new,rows", [
    (Grouped(128), 24, 12, [5, 5, 5], 15),       # more rows than the attention's buffers: self.x would be cut and written behind its end
    (Grouped(128), 24, 12, [1, 1, 1], 4),        # not the step's rows
    (Grouped(128), 24, 12, [1, 1, 1], 2),
    (Grouped(4), 24, 12, [2, 2, 2], 6),          # more rows than the grouped decoder takes
    (Single(), 24, 12, [1, 1, 1], 3),            # several rows for the decoder of one
])
def test_rows_that_do_not_fit(monkeypatch, moe, cache_tokens, layer_tokens, new, rows):
    layer, cache, launched = parts(monkeypatch, moe, cache_tokens, layer_tokens)
    cache.begin_step(new)
    with pytest.raises(ValueError, match="row"):
        layer.forward(torch.ones(rows, 64), cache)
    assert launched == []


@pytest.mark.parametrize("h", [torch.ones(3, 64, dtype=torch.bfloat16), torch.ones(3, 32), torch.ones(64), torch.ones(64, 3).t(), torch.ones(1, 64).expand(3, 64)])
def test_hidden_states_of_another_type_or_layout(monkeypatch, h):
    layer, cache, launched = parts(monkeypatch, Grouped(128), 24, 12)
    cache.begin_step([1, 1, 1])
    with pytest.raises(ValueError, match="h:"):
        layer.forward(h, cache)
    assert launched == []


def test_norms_that_do_not_fit_are_refused_when_the_layer_is_made(monkeypatch):
    from vic_b200.attention import DecodeLayer
    layer, _, _ = parts(monkeypatch, Grouped(128), 24, 12)
    good = torch.ones(64, dtype=torch.bfloat16)
    for bad in (good.float(), good[:32], good.view(1, 64), torch.ones(128, dtype=torch.float16)[::2]):
        for norms in ((bad, good), (good, bad)):
            with pytest.raises(ValueError, match="norm"):
                DecodeLayer(layer.attention, layer.moe, 0, *norms)


def test_decoders_that_do_not_fit_are_refused_when_the_layer_is_made(monkeypatch):
    """(Rows of another width would be read and written behind their ends; a missing layer was found after the attention had run.)"""
    from vic_b200.attention import DecodeLayer
    layer, cache, launched = parts(monkeypatch, Grouped(128), 24, 12)
    norm = torch.ones(64, dtype=torch.bfloat16)
    for moe, number in ((Grouped(128, Model(hidden=128)), 0), (Grouped(128, Model(n_layers=2)), 2), (Grouped(128), -2)):
        with pytest.raises(ValueError, match="moe"):
            DecodeLayer(layer.attention, moe, number, norm, norm)
    second = DecodeLayer(layer.attention, Grouped(128, Model(n_layers=2)), 1, norm, norm)
    cache.begin_step([1, 1, 1])
    with pytest.raises(ValueError, match="cache"):           # (the cache has one layer)
        second.forward(torch.ones(3, 64), cache)
    assert launched == []


def test_frequencies_of_another_form_are_refused_when_the_layer_is_made():
    from vic_b200.attention import LatentAttention
    from vic_b200.core_types import LatentShape
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    sh = LatentShape("small", 64, 2, 16, 16, 10000.0, 1e-6)
    make = lambda f: LatentAttention(sh, z(160, 64), z(576, 64), z(512), z(2, 32, 512), z(64, 32), inv_freq=f)  # noqa: E731
    for bad in (torch.ones(32), torch.ones(64, dtype=torch.float64), torch.ones(64, dtype=torch.float64)[::2], torch.ones(1, 32, dtype=torch.float64)):
        with pytest.raises(ValueError, match="inv_freq"):
            make(bad)
    good = torch.rand(32, dtype=torch.float64)
    assert make(good).inv_freq is good and make(None).inv_freq[1].item() == pytest.approx(10000.0 ** (-1 / 32), rel=1e-15)


def test_selection_biases_of_another_form_are_refused_when_the_layer_is_made(monkeypatch):
    from vic_b200.attention import DecodeLayer
    layer, _, _ = parts(monkeypatch, Grouped(128), 24, 12)
    norm = torch.ones(64, dtype=torch.bfloat16)
    for bad in (torch.zeros(5), torch.zeros(6, dtype=torch.bfloat16), torch.zeros(12)[::2], torch.zeros(1, 6)):
        with pytest.raises(ValueError, match="selection_bias"):
            DecodeLayer(layer.attention, layer.moe, 0, norm, norm, selection_bias=bad)
    assert DecodeLayer(layer.attention, layer.moe, 0, norm, norm, selection_bias=torch.zeros(6)).selection_bias is not None


def test_queries_of_low_rank_that_do_not_fit_are_refused_when_the_layer_is_made():
    from vic_b200.attention import LatentAttention
    from vic_b200.core_types import LatentShape
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    sh = LatentShape("small", 64, 2, 16, 16, 10000.0, 1e-6)
    make = lambda w_q, **k: LatentAttention(sh, w_q, z(576, 64), z(512), z(2, 32, 512), z(64, 32), **k)  # noqa: E731
    make(z(160, 24), q_down=z(24, 64), q_norm=z(24))
    for w_q, k in ((z(160, 24), {}), (z(160, 64), dict(q_down=z(24, 64), q_norm=z(24))), (z(160, 24), dict(q_down=z(24, 64))), (z(160, 64), dict(q_norm=z(64))),
                   (z(160, 24), dict(q_down=z(24, 32), q_norm=z(24))), (z(160, 24), dict(q_down=z(24, 64).half(), q_norm=z(24))),
                   (z(160, 24), dict(q_down=z(24, 64), q_norm=z(23))), (z(160, 24), dict(q_down=z(24, 64), q_norm=z(24).float())),
                   (z(160, 24), dict(q_down=z(24, 64), q_norm=z(24).to("meta"))), (z(160, 24), dict(q_down=z(24, 64).to("meta"), q_norm=z(24)))):
        with pytest.raises(ValueError):
            make(w_q, **k)


def test_a_decoder_on_another_device_is_refused_when_the_layer_is_made(monkeypatch):
    from vic_b200.attention import DecodeLayer
    layer, _, _ = parts(monkeypatch, Grouped(128), 24, 12)
    norm = torch.ones(64, dtype=torch.bfloat16)
    elsewhere = Model()
    elsewhere.router_w = torch.zeros(1, 6, 64, device="meta")
    with pytest.raises(ValueError, match="moe"):
        DecodeLayer(layer.attention, Grouped(128, elsewhere), 0, norm, norm)
    for norms in ((norm.to("meta"), norm), (norm, norm.to("meta"))):
        with pytest.raises(ValueError, match="norm"):
            DecodeLayer(layer.attention, layer.moe, 0, *norms)
