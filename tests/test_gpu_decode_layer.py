"""A decode layer with latent attention before the MoE sublayer: steps of one and of several sequences, prompt chunks and single tokens."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def layer_of(dev, sequences, max_tokens, dtype=torch.bfloat16):
    from vic_b200.attention import DecodeLayer, LatentAttention, LatentCache
    from vic_b200.core_types import SCORING_SIGMOID, LatentShape, MoeShape
    from vic_b200.grouped import GroupedDecoder
    from vic_b200.moe import MoeDecoder
    from vic_b200.synth import build_synthetic_moe
    model = build_synthetic_moe(MoeShape("small", 1024, 2048, 6, 3, 1, SCORING_SIGMOID, 2.5, True), 1, dev, seed=3, slot_seed=4)
    sh = LatentShape("small", 1024, 16, 128, 64, 10000.0, 1e-6)
    g = torch.Generator(device=dev).manual_seed(5)
    rnd = lambda *s: (torch.randn(*s, generator=g, device=dev) * s[-1] ** -0.5).to(dtype)  # noqa: E731
    att = LatentAttention(sh, rnd(16 * 192, 1024), rnd(576, 1024), torch.ones(512, dtype=dtype, device=dev), rnd(16, 192, 512), rnd(1024, 16 * 64), max_tokens)
    cache = LatentCache(1, 40, 16, sequences, 8, dtype, dev, max_tokens)
    norms = (1 + 0.1 * torch.randn(2, 1024, generator=g, device=dev)).to(torch.float16)
    moe = MoeDecoder(model) if max_tokens == 1 else GroupedDecoder(model, max_tokens=max_tokens)
    return DecodeLayer(att, moe, 0, norms[0], norms[1]), cache, g


def attention64(att, cache, T, q_len):
    """The sublayer from its projections' outputs (library products) in 64 bits, with the bound of what the step rounds:
    q and o to the 16-bit type (u each) and every weight of the softmax (u), the scores' error through exp (2 ds)."""
    sh, u = att.shape, torch.finfo(att.w_q.dtype).eps / 2
    q_in = att.q_in[:T].double().view(T, sh.heads, sh.nope + 64)
    pos = cache.positions[:T].double()
    a = pos[:, None, None] * att.inv_freq
    x, y = q_in[..., sh.nope::2], q_in[..., sh.nope + 1::2]
    rot = torch.stack((x * a.cos() - y * a.sin(), y * a.cos() + x * a.sin()), -1).flatten(-2)
    lat = torch.einsum("thn,hnc->thc", q_in[..., :sh.nope], att.kv_b[:, :sh.nope].double())
    q = torch.cat((lat, rot), -1)
    out, bound = torch.zeros(T, sh.heads, sh.value, dtype=torch.float64, device=q.device), torch.zeros(T, sh.heads, sh.value, dtype=torch.float64, device=q.device)
    w = att.kv_b[:, sh.nope:].double()
    for b, n in enumerate(cache.lens.tolist()):
        ids = cache.table[b, :-(-n // cache.page_size)].long()
        keys = cache.rows[0][ids].reshape(-1, 576)[:n].double()
        for j in range(q_len):
            seen = n - q_len + j + 1
            if seen <= 0:
                continue
            t = b * q_len + j
            s = q[t] @ keys[:seen].T * sh.scale
            ds = (q[t].abs() @ keys[:seen].abs().T * sh.scale).amax(1) * (u + 640 * 2.0 ** -23) + 2.0 ** -20
            p = torch.softmax(s, 1)
            o, mag = p @ keys[:seen, :512], p @ keys[:seen, :512].abs()
            err = (2 * ds + 2 * u + 2.0 ** -12)[:, None] * mag
            out[t] = torch.einsum("hc,hvc->hv", o, w)
            bound[t] = torch.einsum("hc,hvc->hv", err, w.abs()) + u * out[t].abs() + 512 * 2.0 ** -23 * torch.einsum("hc,hvc->hv", mag, w.abs())
    return out, bound


def expected_rows(att, cache, T):
    """The cache rows of the step's tokens from the key-value projection."""
    kv, u = att.kv_in[:T].double(), torch.finfo(att.w_q.dtype).eps / 2
    lat = kv[:, :512] / (kv[:, :512].square().mean(1, keepdim=True) + att.shape.eps).sqrt() * att.kv_norm.double()
    a = cache.positions[:T].double()[:, None] * att.inv_freq
    x, y = kv[:, 512::2], kv[:, 513::2]
    rot = torch.stack((x * a.cos() - y * a.sin(), y * a.cos() + x * a.sin()), -1).flatten(-2)
    want = torch.cat((lat, rot), 1)
    return want, u * want.abs() + 2.0 ** -19 * kv.abs().amax(1, keepdim=True)


@pytest.mark.parametrize("steps", [[[7, 3, 0], [1, 1, 1], [1, 0, 1], [4, 4, 4], [1, 1, 1]], [[40, 40, 40], [1, 1, 1], [2, 2, 2]]])
def test_steps_of_a_batch(cuda_dev, steps):
    layer, cache, g = layer_of(cuda_dev, 3, 120)
    att = layer.attention
    for new in steps:
        q_len = max(new)
        T = 3 * q_len
        cache.begin_step(new)
        h = torch.randn(T, 1024, generator=g, device=cuda_dev)
        before = h.clone()
        out = layer.forward(h, cache)
        assert out.data_ptr() == h.data_ptr()
        want, bound = attention64(att, cache, T, q_len)
        assert bool(((att.v[:T].double() - want).abs() <= bound).all())
        rows, tol = expected_rows(att, cache, T)
        live = cache.slots[:T] >= 0
        got = cache.rows[0].view(-1, 576)[cache.slots[:T][live]].double()
        assert bool(((got - rows[live]).abs() <= tol[live]).all())
        # the layer: h + attention + moe(norm(h + attention)), the second norm's rows still in layer.x
        mid = before + att.out[:T].float()
        moe = layer.moe.forward(0, layer.x[:T]).clone()
        torch.testing.assert_close(h, mid + moe, rtol=1e-6, atol=1e-5)
        x = mid / (mid.square().mean(1, keepdim=True) + 1e-6).sqrt() * layer.moe_norm.float()
        assert bool(((layer.x[:T].float() - x).abs() <= 2.0 ** -8 * x.abs() + 1e-5).all())
    assert int(att.status) == 0 and int(layer.moe.status) == 0


def test_single_tokens_in_a_captured_graph(cuda_dev):
    """One request: the step captured once and replayed token by token gives what the eager steps give, bit for bit."""
    layer, cache, g = layer_of(cuda_dev, 1, 1)
    other, cache2, _ = layer_of(cuda_dev, 1, 1)
    h, tokens = torch.zeros(1, 1024, device=cuda_dev), torch.randn(20, 1024, generator=g, device=cuda_dev)
    side = torch.cuda.Stream()
    cache.begin_step([1])
    h.copy_(tokens[:1])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.forward(h, cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    got = [h.clone()]
    with torch.cuda.graph(graph):
        layer.forward(h, cache)
    for t in range(1, 20):
        cache.begin_step([1])
        h.copy_(tokens[t:t + 1])
        graph.replay()
        got.append(h.clone())
    for t in range(20):
        cache2.begin_step([1])
        e = tokens[t:t + 1].clone()
        other.forward(e, cache2)
        assert torch.equal(e, got[t]), t
    assert int(layer.attention.status) == 0 and cache.host_lens == [20]


def test_rows_that_do_not_fit_the_step_are_refused(cuda_dev):
    layer, cache, _ = layer_of(cuda_dev, 3, 12)
    cache.begin_step([1, 1, 1])
    for n in (2, 4, 15):
        with pytest.raises(ValueError):
            layer.attention.forward(torch.zeros(n, 1024, dtype=torch.bfloat16, device=cuda_dev), cache, 0)
