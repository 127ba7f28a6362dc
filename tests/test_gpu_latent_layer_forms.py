"""The forms of a latent-attention layer: scaled positions, the order of the rotation, the softmax's factor."""
import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu


def layer(dev, shape, dtype=torch.bfloat16, max_tokens=24, seed=5, **more):
    from vic_b200.attention import LatentAttention, LatentCache
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: (torch.randn(*s, generator=g, device=dev) * s[-1] ** -0.5).to(dtype)  # noqa: E731
    H = shape.heads
    att = LatentAttention(shape, rnd(H * (shape.nope + 64), more.pop("q_width", shape.hidden)), rnd(576, shape.hidden), (1 + 0.1 * rnd(512)).to(dtype),
                          rnd(H, shape.nope + shape.value, 512), rnd(shape.hidden, H * shape.value), max_tokens, **more)
    return att, LatentCache(1, 40, 16, 3, 8, dtype, dev, max_tokens), g


def shape_of(**more):
    from vic_b200.core_types import LatentShape
    return dataclasses.replace(LatentShape("small", 256, 8, 64, 32, 10000.0, 1e-6), **more)


@pytest.mark.parametrize("pairs,rope_scale,softmax_scale,slowed", [(True, 1.0, None, False), (False, 1.25, 0.11, True), (True, 0.5, 0.2, True), (False, 1.0, None, False)])
def test_rotation_and_scale_are_the_layers(cuda_dev, pairs, rope_scale, softmax_scale, slowed):
    """Rows of the cache, queries and weighted latents from the projections' outputs, in 64 bits, with the shape's rotation and factor."""
    from tests.test_gpu_latent import assert_rounded, attention64, rotate64, u
    sh = shape_of(pairs=pairs, rope_scale=rope_scale, softmax_scale=softmax_scale)
    freq = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64, device=cuda_dev) / 64)
    if slowed:       # positions stretched over a longer context: the slow half of the frequencies divided
        freq[16:] /= 8
    att, cache, g = layer(cuda_dev, sh, inv_freq=freq if slowed else None)
    scale = 128 ** -0.5 if softmax_scale is None else softmax_scale
    assert sh.scale == scale
    for new in ([5, 8, 2], [1, 1, 1]):
        cache.begin_step(new)
        T = cache.step_rows
        x = torch.randn(T, 256, generator=g, device=cuda_dev).to(torch.bfloat16)
        att.forward(x, cache, 0)
        pos, live = cache.positions[:T], cache.slots[:T] >= 0
        q_in = att.q_in[:T].view(T, 8, 128)
        magnitude = 16 * 2.0 ** -24 * 2 * max(rope_scale, 1.0)
        assert_rounded(att.q[:T, :, 512:], rotate64(q_in[..., 64:], pos, freq, pairs, rope_scale), magnitude * q_in[..., 64:].double().abs().amax(-1, keepdim=True))
        rows = cache.rows[0].view(-1, 576)[cache.slots[:T][live]]
        kv = att.kv_in[:T][live]
        assert_rounded(rows[:, 512:], rotate64(kv[:, 512:], pos[live], freq, pairs, rope_scale), magnitude * kv[:, 512:].double().abs().amax(1, keepdim=True))
        want, _, mag, err = attention64(att.q[:T], cache.rows[0], cache.table, cache.lens, scale)
        ds = 576 * 2.0 ** -23 * err + 2.0 ** -20
        assert_rounded(att.o[:T], want, (2 * ds + u(torch.bfloat16) + 64 * 2.0 ** -24).unsqueeze(-1) * mag)
    assert int(att.status) == 0


@pytest.mark.parametrize("rank,norm_dtype", [(96, torch.bfloat16), (1536, torch.float16)])
def test_queries_of_low_rank(cuda_dev, rank, norm_dtype):
    """norm(x q_down^T) w_q^T: each product within its operands' and its own rounding (2^-8 of the magnitudes' sum covers any order of additions)."""
    from tests.test_gpu_latent import assert_rounded, attention64, u
    g = torch.Generator(device=cuda_dev).manual_seed(9)
    down = (torch.randn(rank, 256, generator=g, device=cuda_dev) / 16).to(torch.bfloat16)
    norm = (1 + 0.2 * torch.randn(rank, generator=g, device=cuda_dev)).to(norm_dtype)
    att, cache, g = layer(cuda_dev, shape_of(), q_width=rank, q_down=down, q_norm=norm)
    for new in ([5, 8, 2], [1, 1, 1]):
        cache.begin_step(new)
        T = cache.step_rows
        x = torch.randn(T, 256, generator=g, device=cuda_dev).to(torch.bfloat16)
        att.forward(x, cache, 0)
        low = x.double() @ down.double().T
        assert bool(((att.q_low32[:T].double() - low).abs() <= 2.0 ** -8 * (x.double().abs() @ down.double().abs().T)).all())
        low = att.q_low32[:T].double()
        low = low / (low.square().mean(1, keepdim=True) + 1e-6).sqrt() * norm.double()
        assert_rounded(att.q_low[:T], low, 64 * 2.0 ** -24 * low.abs())
        a, b = att.q_low[:T].double(), att.w_q.double()
        assert bool(((att.q_in[:T].double() - a @ b.T).abs() <= 2.0 ** -8 * (a.abs() @ b.abs().T)).all())
        want, _, mag, err = attention64(att.q[:T], cache.rows[0], cache.table, cache.lens, 128 ** -0.5)
        assert_rounded(att.o[:T], want, (2 * (576 * 2.0 ** -23 * err + 2.0 ** -20) + u(torch.bfloat16) + 64 * 2.0 ** -24).unsqueeze(-1) * mag)
    assert int(att.status) == 0
