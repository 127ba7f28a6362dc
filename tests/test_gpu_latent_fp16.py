"""fp16 weights of the softmax: a key far above the others must not cost these their share of the result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ROW, RANK = 576, 512


def test_many_weak_keys_beside_a_dominating_one(cuda_dev):
    """One key whose score is 2^S above all others, with values of 0, and N keys of the same weight 2^-S with values of 1, in one CTA's
    piece: o = W / (1 + W) with W = N 2^-S.  The weights are fp16 in a scale in which the row's largest stands at 2^7 or above, so that one is
    off by at most half a step of 2^-24 there, 2^-32 of the largest, or by 2^-11 of itself; then the sum in fp32, N 2^-24 of W, and the result's rounding."""
    from vic_b200 import kernels
    sms = torch.cuda.get_device_properties(cuda_dev).multi_processor_count
    page, pages = 64, 891
    n = page * pages - 24
    cache = torch.zeros(pages, page, ROW, dtype=torch.float16, device=cuda_dev)
    cache[..., :RANK] = 1.0
    cache[0, 0, :RANK] = 0.0
    cache[0, 0, RANK] = 1.0
    table = torch.arange(pages, dtype=torch.int32, device=cuda_dev).expand(sms, pages).contiguous()      # (one cache row set for all sequences)
    lens = torch.full((sms,), n, dtype=torch.int32, device=cuda_dev)
    gap = 14.0 + torch.arange(sms, device=cuda_dev) % 16 + torch.tensor([26.0, 40.0, 5.0], device=cuda_dev).repeat(sms)[:sms] / 64
    q = torch.zeros(sms, 1, ROW, dtype=torch.float16, device=cuda_dev)
    q[:, 0, RANK] = gap.half()
    assert bool((q[:, 0, RANK].float() == gap).all())
    scale = math.log(2.0)
    out, lse = torch.empty(sms, 1, RANK, dtype=torch.float16, device=cuda_dev), torch.empty(sms, 1, device=cuda_dev)
    ws = torch.empty(kernels.latent_attention_workspace_bytes(), dtype=torch.uint8, device=cuda_dev)
    kernels.latent_attention(q, cache, table, lens, scale, out, lse, workspace=ws)
    W = (n - 1) * torch.exp2(-gap.double())
    want = W / (1 + W)
    tol = (n * 2.0 ** -32 + (n * 2.0 ** -24 + 2.0 ** -11 + 2.0 ** -18) * W) / (1 + W) + 2.0 ** -11 * want + 2.0 ** -25
    off = (out[:, 0].double() - want[:, None]).abs()
    assert bool((off <= tol[:, None]).all()), (off / tol[:, None]).amax(1)
    wlse = math.log(2.0) * gap.double() + torch.log1p(W)
    # The sum of the weights: eight threads share a row, each adds its keys in pairs, and one of them holds the dominating key's weight
    # from the start: n / 16 additions, each off by at most half a step of that sum, 2^-24 of it.
    assert bool(((lse[:, 0].double() - wlse).abs() <= n / 16 * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * wlse).all())


def test_scores_that_grow_and_fall_in_fp16(cuda_dev):
    from tests.test_gpu_latent import check_attention, gen, paged
    n, dt = 1500, torch.float16
    cache, table, lens = paged(cuda_dev, [n, n, n, 20000], 64, dt, 6)
    q = torch.randn(4, 64, ROW, generator=gen(cuda_dev, 7), device=cuda_dev).to(dt)
    ramp = torch.linspace(0.0, 1.0, n, device=cuda_dev)
    for b, r in enumerate((ramp, ramp.flip(0), torch.zeros_like(ramp))):
        k = torch.arange(n, device=cuda_dev)
        cache[table[b].long()[k // 64], k % 64] = (q[b, :, :].float().mean(0) * 300.0 * r[:, None]).to(dt)
    check_attention(q, cache, table, lens, 0.3)
