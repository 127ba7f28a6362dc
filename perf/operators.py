"""The latent-attention operators of a decode step as cases that can be timed, beside the MoE sublayer's uses in cases.py.

A layer with latent attention keeps ONE vector of 576 values per token for all heads: 512 values that are key and value at
once (the latent) and 64 rotated ones that are key only.  Four operators take a step's tokens through such a layer between
its projections (the case's ``op``):

  append     normalise the latents, rotate the 64 position values and store the rows into a paged cache
  query      per head: the part without positions into the latent space (a product with the head's key matrix), the rest rotated
  attention  every head of every token over the cache of its sequence, softmax in the latent space, with the log of the sum
  value      per head: the weighted latent through the head's value matrix

With ``own`` they are the calls of vic_b200.kernels, without it their formulas in elementary torch operations, 32 bits
throughout (64 for the angles of positions) and rounded once at the end.
"""
from __future__ import annotations

import math
import random

import torch

own = False

RANK, ROPE = 512, 64
WIDTH = RANK + ROPE
THETA = 50000.0
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _append(tokens, kv, cache, page, pairs=True, **more):
    return {"op": "append", "tokens": tokens, "kv": kv, "cache": cache, "page": page, "pairs": pairs, **more}


def _query(tokens, heads, nope, dtype, pairs=True, **more):
    return {"op": "query", "tokens": tokens, "heads": heads, "nope": nope, "dtype": dtype, "pairs": pairs, **more}


def _attention(batch, q_len, heads, len_lo, len_hi, page, dtype, lens_seed=0, **more):
    return {"op": "attention", "batch": batch, "q_len": q_len, "heads": heads, "len_lo": len_lo, "len_hi": len_hi, "page": page,
            "dtype": dtype, "lens_seed": lens_seed, **more}


def _value(tokens, heads, value, dtype, **more):
    return {"op": "value", "tokens": tokens, "heads": heads, "value": value, "dtype": dtype, **more}


def listed():
    return [
        # the smallest call: the new tokens of a decode batch of odd size, where the launch is the cost
        _append(29, "bf16", "bf16", 64, name="append_29"),
        # a long prompt's rows from a projection that leaves fp32, into small pages
        _append(8191, "fp32", "fp16", 16, pairs=False, name="append_8191"),
        # decode of one request: the heads' key matrices are read for one token
        _query(1, 64, 128, "bf16", name="query_1"),
        # a decode batch of odd size
        _query(47, 64, 128, "fp16", name="query_47"),
        # the chunk of a prompt, where the result's rows are most of the bytes
        _query(500, 64, 128, "bf16", pairs=False, name="query_500"),
        # decode of one request with an ordinary context: the length alone has to fill the card
        _attention(1, 1, 64, 4001, 4001, 64, "bf16", name="attention_1x4001"),
        # decode of one request with a long context
        _attention(1, 1, 64, 131071, 131071, 64, "bf16", name="attention_1x131071"),
        # a decode batch whose sequences are anywhere between a word and a document
        _attention(32, 1, 64, 1, 16384, 64, "bf16", lens_seed=5, name="attention_32_ragged"),
        # the largest decode batch of a step
        _attention(128, 1, 64, 3900, 4300, 128, "bf16", lens_seed=6, name="attention_128x4100"),
        # one rank's heads of drafted tokens, several per sequence, pages smaller than a tile
        _attention(13, 5, 16, 40, 6000, 16, "fp16", lens_seed=7, name="attention_draft_13x5"),
        # decode of one request: the heads' value matrices are read for one token
        _value(1, 64, 128, "bf16", name="value_1"),
        # the largest decode batch of a step
        _value(128, 64, 128, "fp16", name="value_128"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: any of the operators, from one token to a prompt's chunk, contexts from one token to a book."""
    op = rng.choice(["append", "query", "attention", "attention", "attention", "value"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    heads = rng.choice([8, 16, 32, 64, 64, rng.randint(1, 128)])
    if op == "append":
        return _append(_log_int(rng, 1, 8192), rng.choice(["bf16", "fp16", "fp32"]), dtype, 8 * rng.randint(1, 32), rng.random() < 0.6)
    if op == "query":
        return _query(_log_int(rng, 1, 512), heads, 16 * rng.randint(2, 12), dtype, rng.random() < 0.6)
    if op == "value":
        return _value(_log_int(rng, 1, 512), heads, 16 * rng.randint(2, 12), dtype)
    while True:
        batch, q_len, hi = _log_int(rng, 1, 160), rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 2, 128)]), _log_int(rng, 1, 131072)
        lo = rng.choice([1, hi, max(1, hi // 2)])
        # no more work than the largest batch above, and a plain form whose padded scores stay within some gigabytes
        if batch * hi <= 500000 and batch * hi * q_len * max(heads, 16) <= 32e6:
            return _attention(batch, q_len, heads, lo, hi, rng.choice([16, 32, 64, 64, 128, 8 * rng.randint(1, 40)]), dtype, rng.randint(0, 10 ** 6))


def _lens(case):
    """The sequences' lengths, spread over their logarithm; the first one is the longest that the case allows."""
    rng = random.Random(case["lens_seed"])
    lens = [_log_int(rng, case["len_lo"], case["len_hi"]) for _ in range(case["batch"])]
    lens[0] = case["len_hi"]
    return lens


def _inv_freq(dev):
    return THETA ** (-torch.arange(0, ROPE, 2, dtype=torch.float64, device=dev) / ROPE)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(shape, dtype, std=1.0):
        return (torch.randn(shape, generator=g, device=dev) * std).to(dtype)

    s = dict(case)
    if case["op"] == "append":
        T, page = case["tokens"], case["page"]
        pages = -(-T // page) + 3
        s["x"] = normal((T, WIDTH), DTYPES[case["kv"]], 0.7)
        s["norm"] = (1.0 + 0.1 * torch.randn(RANK, generator=g, device=dev)).to(DTYPES[case["cache"]])
        s["positions"] = torch.randint(0, 200000, (T,), generator=g, device=dev, dtype=torch.int32)
        s["slots"] = torch.randperm(pages * page, generator=g, device=dev)[:T].contiguous()
        s["pages"] = normal((pages, page, WIDTH), DTYPES[case["cache"]])
        s["inv_freq"] = _inv_freq(dev)
    elif case["op"] == "query":
        T, H, dt = case["tokens"], case["heads"], DTYPES[case["dtype"]]
        s["q"] = normal((T, H, case["nope"] + ROPE), dt)
        s["w"] = normal((H, case["nope"], RANK), dt, case["nope"] ** -0.5)
        s["positions"] = torch.randint(0, 200000, (T,), generator=g, device=dev, dtype=torch.int32)
        s["inv_freq"] = _inv_freq(dev)
        s["out"] = torch.zeros(T, H, WIDTH, dtype=dt, device=dev)
    elif case["op"] == "value":
        T, H, dt = case["tokens"], case["heads"], DTYPES[case["dtype"]]
        s["o"] = normal((T, H, RANK), dt, 0.2)
        s["w"] = normal((H, case["value"], RANK), dt, RANK ** -0.5)
        s["out"] = torch.zeros(T, H, case["value"], dtype=dt, device=dev)
    else:
        B, H, page, dt, lens = case["batch"], case["heads"], case["page"], DTYPES[case["dtype"]], _lens(case)
        per_seq = [-(-n // page) for n in lens]
        spare = 5
        order = torch.randperm(sum(per_seq) + spare, generator=g, device=dev).to(torch.int32)
        # (pages that no sequence has yet are entry 0 of the table, any valid page will do)
        s["table"] = torch.zeros(B, max(per_seq), dtype=torch.int32, device=dev)
        at = 0
        for b, n in enumerate(per_seq):
            s["table"][b, :n] = order[at:at + n]
            at += n
        s["pages"] = normal((sum(per_seq) + spare, page, WIDTH), dt)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["q"] = normal((B * case["q_len"], H, WIDTH), dt)
        s["scale"] = (128 + ROPE) ** -0.5
        s["out"] = torch.zeros(B * case["q_len"], H, RANK, dtype=dt, device=dev)
        s["lse"] = torch.zeros(B * case["q_len"], H, device=dev)
        # scratch for the parts of sequences that several blocks share
        s["workspace"] = torch.empty(64 << 20, dtype=torch.uint8, device=dev)
    return s


def run(s):
    return {"append": _run_append, "query": _run_query, "attention": _run_attention, "value": _run_value}[s["op"]](s)


def _rotated(x, positions, inv_freq, pairs):
    """x [..., 64] turned by its position's angles, one frequency per two values: neighbours (``pairs``) or 32 apart."""
    angle = positions.double().unsqueeze(1) * inv_freq
    cos, sin = angle.cos().float(), angle.sin().float()
    if x.dim() == 3:
        cos, sin = cos.unsqueeze(1), sin.unsqueeze(1)
    x = x.float()
    a, b = (x[..., 0::2], x[..., 1::2]) if pairs else (x[..., :ROPE // 2], x[..., ROPE // 2:])
    u, v = a * cos - b * sin, b * cos + a * sin
    return torch.stack((u, v), -1).flatten(-2) if pairs else torch.cat((u, v), -1)


def _run_append(s):
    if own:
        from vic_b200 import kernels
        kernels.latent_append(s["x"], s["norm"], EPS, s["positions"], s["slots"], s["inv_freq"], s["pages"], pairs=s["pairs"])
        return s["pages"]
    x = s["x"][:, :RANK].float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["norm"].float()
    row = torch.cat((x, _rotated(s["x"][:, RANK:], s["positions"], s["inv_freq"], s["pairs"])), -1)
    s["pages"].view(-1, WIDTH)[s["slots"]] = row.to(s["pages"].dtype)
    return s["pages"]


def _run_query(s):
    if own:
        from vic_b200 import kernels
        kernels.latent_query(s["q"], s["w"], s["positions"], s["inv_freq"], s["out"], pairs=s["pairs"])
        return s["out"]
    nope = s["nope"]
    lat = torch.matmul(s["q"][..., :nope].transpose(0, 1).float(), s["w"].float()).transpose(0, 1)
    return torch.cat((lat, _rotated(s["q"][..., nope:], s["positions"], s["inv_freq"], s["pairs"])), -1).to(s["q"].dtype)


def _run_value(s):
    if own:
        from vic_b200 import kernels
        kernels.latent_value(s["o"], s["w"], s["out"])
        return s["out"]
    return torch.matmul(s["o"].transpose(0, 1).float(), s["w"].float().transpose(1, 2)).transpose(0, 1).to(s["o"].dtype)


def _run_attention(s):
    if own:
        from vic_b200 import kernels
        kernels.latent_attention(s["q"], s["pages"], s["table"], s["lens"], s["scale"], s["out"], s["lse"], workspace=s["workspace"])
        return s["out"], s["lse"]
    B, Q, H, longest = s["batch"], s["q_len"], s["heads"], s["len_hi"]
    keys = s["pages"][s["table"].long()].flatten(1, 2)[:, :longest].float()                    # [B, L, 576], padded
    at = torch.arange(longest, device=keys.device)
    keys = torch.where((at < s["lens"].unsqueeze(1)).unsqueeze(-1), keys, 0.0)
    q = s["q"].float().view(B, Q * H, WIDTH)
    scores = (torch.matmul(q, keys.transpose(1, 2)) * s["scale"]).view(B, Q, H, longest)
    # token j of the q_len newest ones sees the keys up to its own
    last = s["lens"].unsqueeze(1) - Q + torch.arange(Q, device=keys.device)
    seen = (at <= last.unsqueeze(-1)).unsqueeze(2)
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3.0e38)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Q * H, longest), keys[..., :RANK]).view(B, Q, H, RANK)
    o = torch.where(total > 0, o / total, 0.0)
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)
    return o.view(B * Q, H, RANK).to(s["q"].dtype), lse.view(B * Q, H)


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "append":
        T = case["tokens"]
        return {"bytes": T * (WIDTH * (size[case["kv"]] + size[case["cache"]]) + 4 + 8) + RANK * 2, "flops": T * (4 * RANK + 6 * ROPE)}
    T, H = case.get("tokens"), case["heads"]
    if case["op"] == "query":
        n = case["nope"]
        return {"bytes": 2 * (T * H * (n + ROPE) + H * n * RANK + T * H * WIDTH) + 4 * T, "flops": 2 * T * H * n * RANK + 6 * T * H * ROPE // 2}
    if case["op"] == "value":
        v = case["value"]
        return {"bytes": 2 * (T * H * RANK + H * v * RANK + T * H * v), "flops": 2 * T * H * v * RANK}
    lens, Q = _lens(case), case["q_len"]
    rows = case["batch"] * Q * H
    pairs = sum(max(0, n - Q + j + 1) for n in lens for j in range(Q))
    table = sum(-(-n // case["page"]) for n in lens)
    return {"bytes": 2 * (sum(lens) * WIDTH + rows * (WIDTH + RANK)) + 4 * (rows + table + len(lens)), "flops": 2 * pairs * H * (WIDTH + RANK)}


def exact(case, seed):
    """The operators from their definitions, sequence by sequence and head by head in 64 bits."""
    s = prepare(case, seed)
    d = torch.float64

    def turn(x, positions):
        half = ROPE // 2
        z = torch.view_as_complex(x.to(d).reshape(*x.shape[:-1], half, 2)) if case["pairs"] else torch.complex(x[..., :half].to(d), x[..., half:].to(d))
        angle = torch.outer(positions.to(d), torch.tensor([THETA ** (-2 * i / ROPE) for i in range(half)], dtype=d, device=x.device))
        z = z * torch.polar(torch.ones_like(angle), angle).reshape(angle.shape[0], *(1,) * (x.dim() - 2), half)
        return torch.view_as_real(z).flatten(-2) if case["pairs"] else torch.cat((z.real, z.imag), -1)

    if case["op"] == "append":
        pages = s["pages"].to(d)
        lat = s["x"][:, :RANK].to(d)
        lat = lat / torch.sqrt(torch.linalg.vector_norm(lat, dim=1, keepdim=True) ** 2 / RANK + EPS)
        pages.view(-1, WIDTH).index_copy_(0, s["slots"], torch.cat((lat * s["norm"].to(d), turn(s["x"][:, RANK:], s["positions"])), 1))
        return pages
    if case["op"] == "query":
        out = torch.empty(s["out"].shape, dtype=d, device=s["q"].device)
        for h in range(case["heads"]):
            out[:, h, :RANK] = s["q"][:, h, :case["nope"]].to(d) @ s["w"][h].to(d)
        out[..., RANK:] = turn(s["q"][..., case["nope"]:], s["positions"])
        return out
    if case["op"] == "value":
        return torch.stack([s["o"][:, h].to(d) @ s["w"][h].to(d).T for h in range(case["heads"])], 1)
    Q, H, page = case["q_len"], case["heads"], case["page"]
    out = torch.zeros(s["out"].shape, dtype=d, device=s["q"].device)
    lse = torch.full(s["lse"].shape, -math.inf, dtype=d, device=s["q"].device)
    for b, n in enumerate(_lens(case)):
        keys = s["pages"][s["table"][b, :-(-n // page)].long()].reshape(-1, WIDTH)[:n].to(d)
        for j in range(Q):
            seen = n - Q + j + 1
            if seen > 0:
                t = b * Q + j
                scores = s["q"][t].to(d) @ keys[:seen].T * s["scale"]
                lse[t] = torch.logsumexp(scores, 1)
                out[t] = torch.softmax(scores, 1) @ keys[:seen, :RANK]
    return out, lse
