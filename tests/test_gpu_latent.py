"""Latent attention on the GPU against its formulas in 64 bits.

Tolerances: with u = eps/2 of the 16-bit type (bf16 2^-8 / 2 ... = torch.finfo.eps / 2), a result that is rounded once is off
by at most u |y|; a sum of n products accumulated in fp32 adds at most n 2^-23 times the sum of the magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

RANK, ROPE, ROW = 512, 64, 576
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def u(dtype):
    return torch.finfo(dtype).eps / 2


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def inv_freq(dev, theta=50000.0):
    return theta ** (-torch.arange(0, ROPE, 2, dtype=torch.float64, device=dev) / ROPE)


def rotate64(x, positions, freq, pairs, scale=1.0):
    """x [T, ..., 64] in 64 bits."""
    a = positions.double()[:, None] * freq
    a = a.reshape(a.shape[0], *(1,) * (x.dim() - 2), ROPE // 2)
    c, s, x = a.cos() * scale, a.sin() * scale, x.double()
    p, q = (x[..., 0::2], x[..., 1::2]) if pairs else (x[..., :32], x[..., 32:])
    r = (p * c - q * s, q * c + p * s)
    return torch.stack(r, -1).flatten(-2) if pairs else torch.cat(r, -1)


def assert_rounded(got, want, more=0.0):
    """One rounding of `want` (a relative u, and half a step of the subnormals) plus `more` (absolute, a tensor or number)."""
    tiny = torch.finfo(got.dtype).smallest_normal * u(got.dtype)
    off = (got.double() - want).abs()
    allowed = want.abs() * u(got.dtype) + tiny + more
    assert bool((off <= allowed).all()), f"largest excess {(off / allowed).max().item():.3g} of the tolerance"


# ── append ───────────────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("tokens,kv,cache_dt,page,pairs,normed,pad", [
    (1, "bf16", "bf16", 64, True, True, 0), (29, "fp16", "fp16", 16, False, True, 0), (5, "fp32", "bf16", 8, True, True, 0),
    (130, "fp32", "fp16", 24, False, False, 64), (257, "bf16", "fp16", 128, True, True, 8), (3, "fp16", "bf16", 1, True, True, 0)])
def test_append_matches_the_formula_and_touches_nothing_else(cuda_dev, tokens, kv, cache_dt, page, pairs, normed, pad):
    from vic_b200 import kernels
    g = gen(cuda_dev, tokens)
    pages = -(-tokens // page) + 2
    x = torch.randn(tokens, ROW + 16, generator=g, device=cuda_dev).to(DT[kv])[:, 8:8 + ROW]
    store = torch.randn(pages, page, ROW + pad, generator=g, device=cuda_dev).to(DT[cache_dt])
    cache, before = store[..., :ROW], store.clone()
    w = (1 + 0.2 * torch.randn(RANK, generator=g, device=cuda_dev)).to(DT[cache_dt]) if normed else None
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device=cuda_dev, dtype=torch.int32)
    slots = torch.randperm(pages * page, generator=g, device=cuda_dev)[:tokens].contiguous()
    if tokens > 4:
        slots[2] = -1
        slots[4] = -(1 << 40)
    f, status = inv_freq(cuda_dev), torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    kernels.latent_append(x, w, 1e-6, pos, slots, f, cache, pairs=pairs, rope_scale=1.25, status=status)
    lat = x[:, :RANK].double()
    if normed:
        lat = lat / (lat.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
    want = torch.cat((lat, rotate64(x[:, RANK:], pos, f, pairs, 1.25)), 1)
    keep = slots >= 0
    at = slots[keep]
    rows = cache[at // page, at % page]
    # fp32 arithmetic: a few roundings of 2^-24 each relative to the two products of a rotation or to the value
    assert_rounded(rows, want[keep], 16 * 2.0 ** -24 * (want[keep].abs() + 2.5 * x[keep].double().abs().amax(1, keepdim=True)))
    assert int(status) == 0
    untouched = torch.ones(pages, page, dtype=torch.bool, device=cuda_dev)
    untouched[at // page, at % page] = False
    assert torch.equal(store[untouched], before[untouched]) and torch.equal(store[..., ROW:], before[..., ROW:])


def test_append_slot_beyond_the_cache_sets_the_status_and_is_skipped(cuda_dev):
    from vic_b200 import kernels
    cache = torch.zeros(2, 8, ROW, dtype=torch.bfloat16, device=cuda_dev)
    x = torch.ones(3, ROW, dtype=torch.bfloat16, device=cuda_dev)
    pos = torch.zeros(3, dtype=torch.int32, device=cuda_dev)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    slots = torch.tensor([16, 3, 1 << 45], device=cuda_dev)
    kernels.latent_append(x, None, 0.0, pos, slots, inv_freq(cuda_dev), cache, status=status)
    assert int(status) == 1
    assert torch.equal(cache.view(-1, ROW)[3], x[1]) and int((cache != 0).any(-1).sum()) == 1


def test_append_and_attention_past_32_bit_offsets(cuda_dev):
    """A cache of more than 2^31 elements: slots and pages at its end."""
    from vic_b200 import kernels
    pages, page = 4000000 // 64, 64
    cache = torch.empty(pages, page, ROW, dtype=torch.bfloat16, device=cuda_dev)
    assert cache.numel() > 1 << 31
    n = 100
    x = torch.randn(n, ROW, generator=gen(cuda_dev, 1), device=cuda_dev).to(torch.bfloat16)
    table = torch.tensor([[pages - 1, pages - 7]], dtype=torch.int32, device=cuda_dev)
    at = torch.arange(n, device=cuda_dev)
    slots = table[0].long()[at // page] * page + at % page
    pos = torch.zeros(n, dtype=torch.int32, device=cuda_dev)
    kernels.latent_append(x, None, 0.0, pos, slots, inv_freq(cuda_dev), cache)
    assert torch.equal(cache[pages - 1], x[:64]) and torch.equal(cache[pages - 7, :36], x[64:])
    q = torch.randn(1, 16, ROW, generator=gen(cuda_dev, 2), device=cuda_dev).to(torch.bfloat16)
    check_attention(q, cache, table, torch.tensor([n], dtype=torch.int32, device=cuda_dev), 0.07)


# ── per-head products ────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("tokens,heads,nope,dt,pairs", [
    (1, 64, 128, "bf16", True), (1, 1, 16, "fp16", False), (7, 3, 80, "fp16", True), (16, 16, 192, "bf16", False), (17, 5, 48, "bf16", True),
    (47, 64, 128, "fp16", True), (65, 128, 256, "bf16", False), (200, 9, 112, "fp16", False)])
def test_query_matches_the_formula(cuda_dev, tokens, heads, nope, dt, pairs):
    from vic_b200 import kernels
    g, dt = gen(cuda_dev, tokens + heads), DT[dt]
    q = torch.randn(tokens, heads, nope + ROPE + 8, generator=g, device=cuda_dev).to(dt)[..., :nope + ROPE]
    w = (torch.randn(heads, nope + 32, RANK, generator=g, device=cuda_dev) * nope ** -0.5).to(dt)[:, :nope]
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device=cuda_dev, dtype=torch.int32)
    f = inv_freq(cuda_dev)
    store = torch.full((heads + 1, tokens + 1, ROW + 8), 7.0, dtype=dt, device=cuda_dev)
    out = store.transpose(0, 1)[:tokens, :heads, :ROW]          # heads outermost
    kernels.latent_query(q, w, pos, f, out, pairs=pairs, rope_scale=0.75)
    a, b = q[..., :nope].double().transpose(0, 1), w.double()
    lat, mag = torch.bmm(a, b).transpose(0, 1), torch.bmm(a.abs(), b.abs()).transpose(0, 1)
    assert_rounded(out[..., :RANK], lat, nope * 2.0 ** -23 * mag)
    rot = rotate64(q[..., nope:], pos, f, pairs, 0.75)
    assert_rounded(out[..., RANK:], rot, 16 * 2.0 ** -24 * 2 * q[..., nope:].double().abs().amax(-1, keepdim=True))
    store[:heads, :tokens, :ROW] = 7.0
    assert bool((store == 7.0).all())


@pytest.mark.parametrize("tokens,heads,value,dt", [
    (1, 64, 128, "bf16"), (1, 1, 16, "fp16"), (7, 3, 80, "fp16"), (16, 16, 256, "bf16"), (17, 5, 48, "bf16"), (128, 64, 128, "fp16"),
    (65, 128, 112, "bf16"), (300, 9, 128, "fp16")])
def test_value_matches_the_formula(cuda_dev, tokens, heads, value, dt):
    from vic_b200 import kernels
    g, dt = gen(cuda_dev, tokens + heads), DT[dt]
    o = torch.randn(tokens, heads, RANK + 8, generator=g, device=cuda_dev).to(dt)[..., :RANK]
    w = (torch.randn(heads, value + 64, RANK, generator=g, device=cuda_dev) * RANK ** -0.5).to(dt)[:, 64:]
    store = torch.full((tokens + 1, heads + 1, value + 8), 7.0, dtype=dt, device=cuda_dev)
    out = store[:tokens, :heads, :value]
    kernels.latent_value(o, w, out)
    a, b = o.double().transpose(0, 1), w.double().transpose(1, 2)
    want, mag = torch.bmm(a, b).transpose(0, 1), torch.bmm(a.abs(), b.abs()).transpose(0, 1)
    assert_rounded(out, want, RANK * 2.0 ** -23 * mag)
    store[:tokens, :heads, :value] = 7.0
    assert bool((store == 7.0).all())


def test_products_do_not_read_values_outside_their_operands(cuda_dev):
    """NaN in every place that belongs to no operand: behind the rows, between the heads, behind the last token."""
    from vic_b200 import kernels
    T, H, n, dt = 21, 3, 80, torch.bfloat16
    big = torch.full((T + 3, H + 2, n + ROPE + 16), math.nan, dtype=dt, device=cuda_dev)
    wide = torch.full((H + 2, n + 8, RANK), math.nan, dtype=dt, device=cuda_dev)
    q, w = big[:T, :H, :n + ROPE], wide[:H, :n]
    q.fill_(0.5)
    w.fill_(0.25)
    pos, f = torch.zeros(T, dtype=torch.int32, device=cuda_dev), inv_freq(cuda_dev)
    out = torch.empty(T, H, ROW, dtype=dt, device=cuda_dev)
    kernels.latent_query(q, w, pos, f, out)
    assert bool((out[..., :RANK] == 10.0).all()) and bool((out[..., RANK:] == 0.5).all())
    ob = torch.full((T + 3, H + 2, RANK + 16), math.nan, dtype=dt, device=cuda_dev)
    o = ob[:T, :H, :RANK]
    o.fill_(0.5)
    out = torch.empty(T, H, n, dtype=dt, device=cuda_dev)
    kernels.latent_value(o, w, out)
    assert bool((out == 64.0).all())


# ── attention ────────────────────────────────────────────────────────────────────────────────

def attention64(q, cache, table, lens, scale):
    """out [T, H, 512], lse [T, H] and the largest |score| bound of every row, in 64 bits.  Keys whose page is out of range are left out."""
    T, H, _ = q.shape
    B = lens.numel()
    Q, page, pages = T // B, cache.shape[1], cache.shape[0]
    out = torch.zeros(T, H, RANK, dtype=torch.float64, device=q.device)
    mag = torch.zeros(T, H, RANK, dtype=torch.float64, device=q.device)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device=q.device)
    err = torch.zeros(T, H, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lens.tolist()):
        n_pages = min(-(-max(n, 0) // page), table.shape[1])
        ids = table[b, :n_pages].long()
        good = (ids >= 0) & (ids < pages)
        keys = cache[torch.where(good, ids, 0)].reshape(-1, ROW)[:max(n, 0)].double()
        good = good.repeat_interleave(page)[:max(n, 0)]
        for j in range(Q):
            seen = min(max(n - Q + j + 1, 0), keys.shape[0])
            k = keys[:seen][good[:seen]]
            if k.shape[0] == 0:
                continue
            t = b * Q + j
            s = q[t].double() @ k.T * scale
            err[t] = (q[t].double().abs() @ k.abs().T * abs(scale)).amax(1)
            lse[t] = torch.logsumexp(s, 1)
            p = torch.softmax(s, 1)
            out[t] = p @ k[:, :RANK]
            mag[t] = p @ k[:, :RANK].abs()
    return out, lse, mag, err


def check_attention(q, cache, table, lens, scale, out=None, lse=None, status=0, workspace=None):
    """A score is off by at most 576 2^-23 of its magnitudes' sum (fp32 accumulation) and exp by a few 2^-22 more; a weight is rounded once to the
    16-bit type before its product with the value, and so is the result: |o - o'| <= (2 (ds + 2^-20) + u + (keys) 2^-23) sum p |c| + u |o|."""
    from vic_b200 import kernels
    T, H, _ = q.shape
    dev = q.device
    out = torch.full((T, H, RANK), 9.0, dtype=q.dtype, device=dev) if out is None else out
    lse = torch.full((T, H), 9.0, device=dev) if lse is None else lse
    workspace = torch.empty(kernels.latent_attention_workspace_bytes(), dtype=torch.uint8, device=dev) if workspace is None else workspace
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    kernels.latent_attention(q, cache, table, lens, scale, out, lse, workspace=workspace, status=st)
    want, wlse, mag, err = attention64(q, cache, table, lens, scale)
    longest = max(1, int(lens.max()))
    ds = ROW * 2.0 ** -23 * err + 2.0 ** -20
    rel = (2 * ds + u(q.dtype) + longest * 2.0 ** -24).unsqueeze(-1)
    assert_rounded(out, want, rel * mag)
    empty = wlse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and not bool(lse.isnan().any())
    off = torch.where(empty, 0.0, (lse.double() - torch.where(empty, 0.0, wlse)).abs())
    assert bool((off <= ds + longest * 2.0 ** -24 + 2.0 ** -22 * wlse.abs().nan_to_num(posinf=0.0)).all())
    assert bool((out[empty] == 0).all())
    assert int(st) == status
    return out, lse


def paged(dev, lens, page, dtype, seed, spare=3, fill=None, row_pad=0):
    g = gen(dev, seed)
    per = [-(-max(n, 0) // page) for n in lens]
    total = sum(per) + spare
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(lens), max(1, max(per)), dtype=torch.int32, device=dev)
    store = torch.randn(total, page, ROW + row_pad, generator=g, device=dev).to(dtype)
    cache = store[..., :ROW]
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    if fill is not None:         # whatever lies behind the sequences
        live = torch.zeros(total, page, dtype=torch.bool, device=dev)
        for b, n in enumerate(lens):
            k = torch.arange(max(n, 0), device=dev)
            live[table[b].long()[k // page], k % page] = True
        store[~live] = fill
        store[..., ROW:] = fill
    return cache, table, torch.tensor(lens, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("lens,q_len,heads,page,dt", [
    ([1], 1, 1, 64, "bf16"), ([1, 2, 0, 3], 1, 64, 16, "bf16"), ([63, 64, 65, 127, 128, 129], 1, 64, 64, "fp16"),
    ([40], 1, 8, 8, "fp16"), ([700, 31, 1999], 1, 16, 24, "bf16"), ([4001], 1, 64, 64, "bf16"), ([300, 5], 1, 128, 128, "fp16"),
    ([513, 2000], 1, 101, 40, "bf16"), ([3, 0, 700], 5, 16, 16, "fp16"), ([1000, 66], 9, 64, 64, "bf16"), ([129], 129, 3, 32, "bf16"),
    ([300, 1000, 0, 700, 59], 60, 64, 64, "bf16"), ([2000, 33], 33, 128, 16, "fp16"), ([12000] * 3, 1, 64, 64, "bf16"), ([50] * 200, 1, 32, 64, "fp16"), ([70, 2500] * 40, 2, 64, 320, "bf16"), ([5, 100], 8, 7, 56, "fp16")])
def test_attention_matches_the_formula(cuda_dev, lens, q_len, heads, page, dt):
    cache, table, lens = paged(cuda_dev, lens, page, DT[dt], len(lens) + heads)
    q = torch.randn(lens.numel() * q_len, heads, ROW, generator=gen(cuda_dev, 3), device=cuda_dev).to(DT[dt])
    check_attention(q, cache, table, lens, 192 ** -0.5)


@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("page", [16, 64, 200])
def test_attention_ignores_what_lies_behind_a_sequence(cuda_dev, fill, page):
    cache, table, lens = paged(cuda_dev, [1, 65, 130, 0, 777], page, torch.bfloat16, 4, fill=fill, row_pad=8)
    table = torch.nn.functional.pad(table, (0, 3), value=2 ** 31 - 1)[:, :table.shape[1]]      # (a strided table, too)
    q = torch.randn(5 * 2, 64, ROW + 8, generator=gen(cuda_dev, 5), device=cuda_dev).to(torch.bfloat16)[..., :ROW]
    check_attention(q, cache, table, lens, 0.07)


def test_attention_with_sharp_and_growing_scores(cuda_dev):
    """Scores of some hundred that grow along the sequence (the running maximum moves in every tile), fall, and are all alike."""
    n, dt = 1500, torch.bfloat16
    cache, table, lens = paged(cuda_dev, [n, n, n], 64, dt, 6)
    q = torch.randn(3, 64, ROW, generator=gen(cuda_dev, 7), device=cuda_dev).to(dt)
    ramp = torch.linspace(0.0, 1.0, n, device=cuda_dev)
    for b, r in enumerate((ramp, ramp.flip(0), torch.zeros_like(ramp))):
        k = torch.arange(n, device=cuda_dev)
        rows = (q[b, :, :].float().mean(0) * 300.0 * r[:, None]).to(dt)
        cache[table[b].long()[k // 64], k % 64] = rows
    check_attention(q, cache, table, lens, 0.3)


def test_attention_negative_scale_and_broadcast_query(cuda_dev):
    cache, table, lens = paged(cuda_dev, [300, 80], 64, torch.float16, 8)
    q = torch.randn(1, 1, ROW, generator=gen(cuda_dev, 9), device=cuda_dev).to(torch.float16).expand(2, 20, ROW)
    check_attention(q, cache, table, lens, -0.05)


def test_attention_leaves_out_pages_that_are_absent(cuda_dev):
    cache, table, lens = paged(cuda_dev, [500, 200, 64], 32, torch.bfloat16, 10)
    table[0, 3], table[0, 15], table[1, 0], table[2, 0], table[2, 1] = -1, 10 ** 6, cache.shape[0], -5, -(2 ** 31)
    q = torch.randn(3, 64, ROW, generator=gen(cuda_dev, 11), device=cuda_dev).to(torch.bfloat16)
    check_attention(q, cache, table, lens, 0.07, status=1)
    # a length beyond the table: the keys without an entry are left out
    check_attention(q, cache, table[:, :1].contiguous(), lens, 0.07, status=1)


def test_attention_writes_its_own_rows_only(cuda_dev):
    cache, table, lens = paged(cuda_dev, [100, 9], 16, torch.bfloat16, 12)
    q = torch.randn(2, 5, ROW, generator=gen(cuda_dev, 13), device=cuda_dev).to(torch.bfloat16)
    store = torch.full((3, 6, RANK + 8), 7.0, dtype=torch.bfloat16, device=cuda_dev)
    lse = torch.full((3, 5), 7.0, device=cuda_dev)
    check_attention(q, cache, table, lens, 0.07, out=store[:2, :5, :RANK], lse=lse[:2])
    assert bool((lse[2] == 7.0).all())
    store[:2, :5, :RANK] = 7.0
    assert bool((store == 7.0).all())


def test_attention_without_lse_is_the_same_and_repeats_bit_for_bit(cuda_dev):
    from vic_b200 import kernels
    cache, table, lens = paged(cuda_dev, [9000, 17, 3000], 64, torch.bfloat16, 14)
    q = torch.randn(3, 64, ROW, generator=gen(cuda_dev, 15), device=cuda_dev).to(torch.bfloat16)
    ws = torch.full((kernels.latent_attention_workspace_bytes(),), 255, dtype=torch.uint8, device=cuda_dev)    # NaN everywhere
    a, _ = check_attention(q, cache, table, lens, 0.07, workspace=ws)
    for _ in range(3):
        b = torch.empty_like(a)
        kernels.latent_attention(q, cache, table, lens, 0.07, b, workspace=ws)
        assert torch.equal(a, b)


def test_a_step_on_a_side_stream_and_in_a_graph_with_new_lengths(cuda_dev):
    """append -> query -> attention -> value as a decode loop runs them: captured once, replayed as the sequences grow."""
    from vic_b200 import kernels
    B, H, n, v, page, dt = 6, 16, 128, 128, 32, torch.bfloat16
    g = gen(cuda_dev, 16)
    cache, table, lens = paged(cuda_dev, [90, 1, 33, 64, 200, 31], page, dt, 17, spare=0)
    table = torch.arange(B * 10, dtype=torch.int32, device=cuda_dev).view(B, 10)
    cache = torch.randn(B * 10, page, ROW, generator=g, device=cuda_dev).to(dt)
    f = inv_freq(cuda_dev)
    kv_b = (torch.randn(H, n + v, RANK, generator=g, device=cuda_dev) * 0.06).to(dt)
    norm = torch.ones(RANK, dtype=dt, device=cuda_dev)
    x, qin = torch.empty(B, ROW, dtype=dt, device=cuda_dev), torch.empty(B, H, n + ROPE, dtype=dt, device=cuda_dev)
    pos, slots = torch.empty(B, dtype=torch.int32, device=cuda_dev), torch.empty(B, dtype=torch.int64, device=cuda_dev)
    q, o, y = (torch.empty(B, H, w, dtype=dt, device=cuda_dev) for w in (ROW, RANK, v))
    lse = torch.empty(B, H, device=cuda_dev)
    ws = torch.empty(kernels.latent_attention_workspace_bytes(), dtype=torch.uint8, device=cuda_dev)

    def step():
        kernels.latent_append(x, norm, 1e-6, pos, slots, f, cache)
        kernels.latent_query(qin, kv_b[:, :n], pos, f, q)
        kernels.latent_attention(q, cache, table, lens, 0.07, o, lse, workspace=ws)
        kernels.latent_value(o, kv_b[:, n:], y)

    def feed(i):
        x.copy_(torch.randn(B, ROW, generator=g, device=cuda_dev))
        qin.copy_(torch.randn(B, H, n + ROPE, generator=g, device=cuda_dev))
        pos.copy_(lens)
        slots.copy_(table.gather(1, (lens // page).long()[:, None])[:, 0].long() * page + lens % page)
        lens.add_(1)

    def verify():
        want, wlse, mag, _ = attention64(q, cache, table, lens, 0.07)
        assert bool(((lse.double() - wlse).abs() < 1e-3).all())
        assert_rounded(o, want, (u(dt) + 1e-4) * mag)
        a, b = o.double().transpose(0, 1), kv_b[:, n:].double().transpose(1, 2)
        assert_rounded(y, torch.bmm(a, b).transpose(0, 1), RANK * 2.0 ** -23 * torch.bmm(a.abs(), b.abs()).transpose(0, 1))
        at = slots
        lat = x[:, :RANK].double()
        lat = lat / (lat.square().mean(1, keepdim=True) + 1e-6).sqrt()
        assert_rounded(cache.view(-1, ROW)[at][:, :RANK], lat, 1e-5 * lat.abs())

    side = torch.cuda.Stream()
    feed(0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    verify()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        feed(i)
        graph.replay()
        verify()


@pytest.mark.parametrize("lens,q_len,heads", [
    ([0, 0, 0], 1, 64), ([0] * 40 + [64] * 3 + [0] * 50 + [1], 1, 8), ([64, 0, 128, 0, 0, 64] * 30, 1, 64), ([1, 0] * 300, 1, 4),
    ([192, 0, 0, 64 * 37, 0], 2, 40), ([0, 5] * 20, 70, 16), ([64] * 148, 1, 64), ([128] * 149 + [0], 1, 64)])
def test_attention_with_sequences_of_no_tokens_between_others(cuda_dev, lens, q_len, heads):
    """Empty sequences stand at the borders of the CTAs' shares too: each of their rows is written by somebody."""
    cache, table, lens = paged(cuda_dev, lens, 64, torch.bfloat16, 21)
    q = torch.randn(lens.numel() * q_len, heads, ROW, generator=gen(cuda_dev, 22), device=cuda_dev).to(torch.bfloat16)
    check_attention(q, cache, table, lens, 0.07)


@pytest.mark.parametrize("which", ["tokens", "heads", "weights", "overlapping"])
def test_products_of_broadcast_and_overlapping_operands(cuda_dev, which):
    from vic_b200 import kernels
    T, H, n, dt, g = 5, 3, 128, torch.bfloat16, gen(cuda_dev, 31)
    q, w = torch.randn(T, H, n + ROPE, generator=g, device=cuda_dev).to(dt), (torch.randn(H, n, RANK, generator=g, device=cuda_dev) * n ** -0.5).to(dt)
    if which == "tokens":
        q = q[:1].expand(T, H, n + ROPE)
    elif which == "heads":
        q = q[:, :1].expand(T, H, n + ROPE)
    elif which == "weights":
        w = w[:1].expand(H, n, RANK)
    else:
        q = torch.randn(4096, generator=g, device=cuda_dev).to(dt).as_strided((T, H, n + ROPE), (8, 200, 1))
    out, f, pos = torch.empty(T, H, ROW, dtype=dt, device=cuda_dev), inv_freq(cuda_dev), torch.arange(T, dtype=torch.int32, device=cuda_dev)
    kernels.latent_query(q, w, pos, f, out)
    a, b = q[..., :n].double().transpose(0, 1), w.double()
    assert_rounded(out[..., :RANK], torch.bmm(a, b).transpose(0, 1), n * 2.0 ** -23 * torch.bmm(a.abs(), b.abs()).transpose(0, 1))
    assert_rounded(out[..., RANK:], rotate64(q[..., n:], pos, f, True), 16 * 2.0 ** -24 * 2 * q[..., n:].double().abs().amax(-1, keepdim=True))


def test_products_leave_the_status_as_it_was(cuda_dev):
    from vic_b200 import kernels as K
    status = torch.tensor([1 << 20], dtype=torch.int32, device=cuda_dev)
    for tokens in (1, 300):
        q, w = (torch.ones(*s, dtype=torch.bfloat16, device=cuda_dev) for s in ((tokens, 8, 192), (8, 256, 512)))
        lat, out = torch.zeros(tokens, 8, 576, dtype=q.dtype, device=cuda_dev), torch.zeros(tokens, 8, 128, dtype=q.dtype, device=cuda_dev)
        K.latent_query(q, w[:, :128], torch.zeros(tokens, dtype=torch.int32, device=cuda_dev), torch.ones(32, dtype=torch.float64, device=cuda_dev),
                       lat, status=status)
        K.latent_value(lat[:, :, :512], w[:, 128:], out, status=status)
        assert lat[:, :, :512].unique().tolist() == [128.0] and out.unique().tolist() == [65536.0]
    assert status.tolist() == [1 << 20]


@pytest.mark.parametrize("tokens", [127, 128, 129, 256, 257])
@pytest.mark.parametrize("heads", [1, 8, 64])
def test_products_at_the_borders_of_their_tiles(cuda_dev, tokens, heads):
    """128 tokens a tile, 64 to 256 columns by the number of heads: rows of another tile or head in their place would show."""
    from vic_b200 import kernels
    g, dt = gen(cuda_dev, tokens * heads), torch.float16
    q, w = torch.randn(tokens, heads, 64 + ROPE, generator=g, device=cuda_dev).to(dt), (torch.randn(heads, 64, RANK, generator=g, device=cuda_dev) / 8).to(dt)
    out, f, pos = torch.full((tokens, heads, ROW), 9.0, dtype=dt, device=cuda_dev), inv_freq(cuda_dev), torch.arange(tokens, dtype=torch.int32, device=cuda_dev)
    kernels.latent_query(q, w, pos, f, out, pairs=False)
    a, b = q[..., :64].double().transpose(0, 1), w.double()
    assert_rounded(out[..., :RANK], torch.bmm(a, b).transpose(0, 1), 64 * 2.0 ** -23 * torch.bmm(a.abs(), b.abs()).transpose(0, 1))
    assert_rounded(out[..., RANK:], rotate64(q[..., 64:], pos, f, False), 16 * 2.0 ** -24 * 2 * q[..., 64:].double().abs().amax(-1, keepdim=True))
    o, v = torch.randn(tokens, heads, RANK, generator=g, device=cuda_dev).to(dt), (torch.randn(heads, 144, RANK, generator=g, device=cuda_dev) / 20).to(dt)
    y = torch.full((tokens, heads, 144), 9.0, dtype=dt, device=cuda_dev)
    kernels.latent_value(o, v, y)
    a, b = o.double().transpose(0, 1), v.double().transpose(1, 2)
    assert_rounded(y, torch.bmm(a, b).transpose(0, 1), RANK * 2.0 ** -23 * torch.bmm(a.abs(), b.abs()).transpose(0, 1))


@pytest.mark.parametrize("others,long,heads", [(0, 30000, 64), (1, 20000, 128), (5, 30000, 64), (30, 40000, 64), (100, 60000, 16), (200, 50000, 64)])
def test_one_long_sequence_among_short_ones(cuda_dev, others, long, heads):
    """From two to about 148 parts of one sequence, beside sequences of one part, in every form of the adding launch."""
    cache, table, lens = paged(cuda_dev, [3 + i % 40 for i in range(others)] + [long], 64, torch.bfloat16, 23)
    q = torch.randn(lens.numel(), heads, ROW, generator=gen(cuda_dev, 24), device=cuda_dev).to(torch.bfloat16)
    check_attention(q, cache, table, lens, 0.07)


@pytest.mark.parametrize("B,n,heads,q_len", [(64, 2500, 64, 1), (200, 500, 16, 1), (30, 3000, 64, 2), (120, 700, 128, 1)])
def test_shared_sequences_give_the_same_bits_every_time(cuda_dev, B, n, heads, q_len):
    """The CTAs that share a sequence meet in whatever order; who adds up the parts must not show.  A graph's replays too."""
    from vic_b200 import kernels
    cache, table, lens = paged(cuda_dev, [n - (37 * b) % 400 for b in range(B)], 64, torch.bfloat16, 25)
    q = torch.randn(B * q_len, heads, ROW, generator=gen(cuda_dev, 26), device=cuda_dev).to(torch.bfloat16)
    ws = torch.randint(0, 256, (kernels.latent_attention_workspace_bytes(),), dtype=torch.uint8, device=cuda_dev)
    want, wlse = check_attention(q, cache, table, lens, 0.07, workspace=ws)
    out, lse = torch.empty_like(want), torch.empty_like(wlse)
    load = torch.randn(4096, 4096, device=cuda_dev)
    side = torch.cuda.Stream()
    for i in range(60):
        out.fill_(7.0)
        if i % 3 == 1:      # another stream's work takes SMs away meanwhile
            with torch.cuda.stream(side):
                load = torch.tanh(load @ load)
        kernels.latent_attention(q, cache, table, lens, 0.07, out, lse, workspace=ws)
        assert torch.equal(out, want) and torch.equal(lse, wlse), i
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.latent_attention(q, cache, table, lens, 0.07, out, lse, workspace=ws)
    for i in range(20):
        out.fill_(7.0)
        graph.replay()
        assert torch.equal(out, want) and torch.equal(lse, wlse), i
    lens.sub_(100)          # (the replays read the lengths again)
    graph.replay()
    again = torch.empty_like(out)
    kernels.latent_attention(q, cache, table, lens, 0.07, again, workspace=ws)
    assert torch.equal(out, again)


def test_without_programmatic_launches_the_results_are_the_same(cuda_dev):
    from vic_b200 import kernels
    from vic_b200.lib import lib
    cache, table, lens = paged(cuda_dev, [3000, 65, 900], 64, torch.bfloat16, 41)
    g = gen(cuda_dev, 42)
    qin, w = torch.randn(3, 64, 192, generator=g, device=cuda_dev).to(torch.bfloat16), (torch.randn(64, 256, RANK, generator=g, device=cuda_dev) / 12).to(torch.bfloat16)
    pos, f, kv = lens - 1, inv_freq(cuda_dev), torch.randn(3, ROW, generator=g, device=cuda_dev).to(torch.bfloat16)
    slots = table.gather(1, (pos // 64).long()[:, None])[:, 0].long() * 64 + pos % 64
    ws = torch.empty(kernels.latent_attention_workspace_bytes(), dtype=torch.uint8, device=cuda_dev)
    start, got = cache.clone(), []
    try:
        for pdl in (1, 0):
            lib().vib3_config_set(1, pdl)
            cache.copy_(start)
            q, o, y = (torch.empty(3, 64, n, dtype=torch.bfloat16, device=cuda_dev) for n in (ROW, RANK, 128))
            kernels.latent_append(kv, None, 0.0, pos, slots, f, cache)
            kernels.latent_query(qin, w[:, :128], pos, f, q)
            kernels.latent_attention(q, cache, table, lens, 0.07, o, workspace=ws)
            kernels.latent_value(o, w[:, 128:], y)
            got.append((cache.clone(), q, o, y))
    finally:
        lib().vib3_config_set(1, 1)
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_two_streams_with_workspaces_of_their_own(cuda_dev):
    """Two attentions and the products of another step at the same time: nothing is shared but the cache that they read."""
    from vic_b200 import kernels
    cache, table, lens = paged(cuda_dev, [5000, 65, 900, 20000], 64, torch.bfloat16, 43)
    q = torch.randn(4, 64, ROW, generator=gen(cuda_dev, 44), device=cuda_dev).to(torch.bfloat16)
    want, _ = check_attention(q, cache, table, lens, 0.07)
    w = (torch.randn(64, 128, RANK, generator=gen(cuda_dev, 45), device=cuda_dev) / 20).to(torch.bfloat16)
    y0 = torch.empty(4, 64, 128, dtype=torch.bfloat16, device=cuda_dev)
    kernels.latent_value(want, w, y0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    ws = [torch.empty(kernels.latent_attention_workspace_bytes(), dtype=torch.uint8, device=cuda_dev) for _ in range(2)]
    outs = [[torch.empty_like(want) for _ in range(20)] for _ in range(2)]
    ys = [torch.empty_like(y0) for _ in range(20)]
    for i in range(20):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                kernels.latent_attention(q, cache, table, lens, 0.07, outs[s][i], workspace=ws[s])
        with torch.cuda.stream(streams[2]):
            kernels.latent_value(want, w, ys[i])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for s in outs for o in s) and all(torch.equal(y, y0) for y in ys)


def test_operands_off_the_device_are_refused(cuda_dev):
    from vic_b200 import kernels
    cache, table, lens = paged(cuda_dev, [10], 8, torch.bfloat16, 46)
    q, out = (torch.zeros(1, 4, n, dtype=torch.bfloat16, device=cuda_dev) for n in (ROW, RANK))
    ws = torch.empty(kernels.latent_attention_workspace_bytes(), dtype=torch.uint8, device=cuda_dev)
    with pytest.raises(ValueError):
        kernels.latent_attention(q, cache, table.cpu(), lens, 0.1, out, workspace=ws)
    with pytest.raises(ValueError):
        kernels.latent_value(out, torch.zeros(4, 16, RANK, dtype=torch.bfloat16), torch.zeros(1, 4, 16, dtype=torch.bfloat16, device=cuda_dev))


def test_nothing_beyond_the_workspace_and_the_table_is_touched(cuda_dev):
    """Guard bytes on both sides of the workspace, guard entries around the table and the lengths."""
    from vic_b200 import kernels
    n = kernels.latent_attention_workspace_bytes()
    big = torch.full((n + 512,), 0x5A, dtype=torch.uint8, device=cuda_dev)
    cache, table, lens = paged(cuda_dev, [9000] * 40 + [0, 1], 64, torch.bfloat16, 47)
    q = torch.randn(42, 64, ROW, generator=gen(cuda_dev, 48), device=cuda_dev).to(torch.bfloat16)
    check_attention(q, cache, table, lens, 0.07, workspace=big[256:256 + n])
    assert bool((big[:256] == 0x5A).all()) and bool((big[256 + n:] == 0x5A).all())
