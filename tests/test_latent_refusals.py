"""What the latent-attention launchers refuse, before any launch: no GPU is needed."""
import pytest
import torch

F16, BF16, F32 = 1, 2, 0
P = 1 << 20            # an aligned address that no refused call reads


def lib():
    from vic_b200.lib import lib as load
    return load()


def append(**k):
    a = dict(kv=P, kv_dtype=BF16, kv_stride=576, norm=P, eps=1e-6, positions=P, slots=P, inv_freq=P, rope_scale=1.0, pairs=1, n_tokens=1,
             cache=P, cache_dtype=BF16, num_pages=4, page_size=16, page_stride=16 * 576, row_stride=576, status=0, stream=0)
    a.update(k)
    return lib().vib3_launch_latent_append_paged(*a.values())


def query(**k):
    a = dict(q=P, q_token=2 * 192, q_head=192, w=P, w_head=128 * 512, positions=P, inv_freq=P, rope_scale=1.0, pairs=1, out=P,
             out_token=2 * 576, out_head=576, n_tokens=2, heads=2, nope=128, dtype=BF16, status=0, stream=0)
    a.update(k)
    return lib().vib3_launch_latent_query(*a.values())


def value(**k):
    a = dict(o=P, o_token=1024, o_head=512, w=P, w_head=128 * 512, out=P, out_token=256, out_head=128, n_tokens=2, heads=2, value=128,
             dtype=F16, status=0, stream=0)
    a.update(k)
    return lib().vib3_launch_latent_value(*a.values())


def attention(**k):
    a = dict(q=P, q_token=2 * 576, q_head=576, cache=P, num_pages=9, page_size=16, page_stride=16 * 576, row_stride=576, table=P,
             table_stride=4, max_pages=4, lens=P, batch=2, q_len=1, heads=2, scale=0.1, dtype=BF16, out=P, out_token=1024, out_head=512,
             lse=0, workspace=P, workspace_bytes=lib().vib3_latent_attention_workspace_bytes(), status=0, stream=0)
    a.update(k)
    return lib().vib3_launch_latent_attention_paged(*a.values())


UNSUPPORTED, COUNT, NULL, ALIGN, SHAPE, CAPACITY = -1, -2, -3, -4, -5, -8


@pytest.mark.parametrize("call,change,code", [
    *[(append, {n: 0}, NULL) for n in ("kv", "positions", "slots", "inv_freq", "cache")],
    (append, {"kv_dtype": 3}, UNSUPPORTED), (append, {"cache_dtype": F32}, UNSUPPORTED), (append, {"n_tokens": -1}, COUNT),
    (append, {"num_pages": 0}, COUNT), (append, {"page_size": 0}, COUNT), (append, {"row_stride": 568}, SHAPE),
    (append, {"n_tokens": 2, "kv_stride": 568}, SHAPE), (append, {"page_stride": 15 * 576}, SHAPE), (append, {"page_stride": 0}, SHAPE), (append, {"kv": P + 2}, ALIGN), (append, {"kv_stride": 580}, ALIGN),
    (append, {"kv_dtype": F32, "kv_stride": 578}, ALIGN), (append, {"row_stride": 580}, ALIGN), (append, {"cache": P + 8}, ALIGN),
    (append, {"page_stride": 16 * 576 + 4}, ALIGN), (append, {"norm": P + 2}, ALIGN),
    *[(query, {n: 0}, NULL) for n in ("q", "w", "positions", "inv_freq", "out")],
    (query, {"nope": 8}, UNSUPPORTED), (query, {"nope": 120}, UNSUPPORTED), (query, {"nope": 272}, UNSUPPORTED), (query, {"dtype": F32}, UNSUPPORTED),
    (query, {"heads": 0}, COUNT), (query, {"heads": 129}, COUNT), (query, {"n_tokens": -1}, COUNT), (query, {"q": P + 4}, ALIGN),
    (query, {"q_head": 196}, ALIGN), (query, {"out_head": 580}, ALIGN), (query, {"w_head": 4}, ALIGN), (query, {"out_head": 512}, SHAPE),
    (query, {"out_token": 0}, SHAPE), (query, {"q_token": -576}, SHAPE),
    *[(value, {n: 0}, NULL) for n in ("o", "w", "out")],
    (value, {"value": 24}, UNSUPPORTED), (value, {"value": 0}, UNSUPPORTED), (value, {"dtype": 7}, UNSUPPORTED), (value, {"heads": 200}, COUNT),
    (value, {"out_head": 120}, SHAPE), (value, {"o": P + 8}, ALIGN), (value, {"out_token": 260}, ALIGN),
    *[(attention, {n: 0}, NULL) for n in ("q", "cache", "table", "lens", "out", "workspace")],
    (attention, {"dtype": F32}, UNSUPPORTED), (attention, {"page_size": 12}, UNSUPPORTED), (attention, {"heads": 0}, COUNT),
    (attention, {"heads": 129}, COUNT), (attention, {"batch": -1}, COUNT), (attention, {"q_len": -1}, COUNT), (attention, {"num_pages": 0}, COUNT),
    (attention, {"num_pages": 1 << 32}, COUNT), (attention, {"max_pages": 0}, COUNT), (attention, {"max_pages": 1 << 28, "table_stride": 1 << 28}, COUNT),
    (attention, {"q_len": 1 << 20}, COUNT), (attention, {"page_size": 0}, COUNT), (attention, {"row_stride": 512}, SHAPE),
    (attention, {"page_stride": 15 * 576}, SHAPE), (attention, {"table_stride": 3}, SHAPE), (attention, {"out_head": 504}, SHAPE),
    (attention, {"out_token": 8}, SHAPE), (attention, {"q": P + 2}, ALIGN), (attention, {"cache": P + 8}, ALIGN), (attention, {"row_stride": 580, "page_stride": 16 * 580}, ALIGN),
    (attention, {"workspace": P + 4}, ALIGN), (attention, {"q_head": 580}, ALIGN), (attention, {"workspace_bytes": 1 << 20}, CAPACITY),
])
def test_refusals(call, change, code):
    assert call(**change) == code


@pytest.mark.parametrize("page_size,max_pages", [(16, (1 << 27) - 16), (8, (1 << 28) - 256), (1 << 20, 2047), (64, 0x7ffff000 // 64 + 1)])
def test_lengths_whose_key_numbers_pass_32_bits_are_refused(page_size, max_pages):
    # a table entry is looked up for 32 boxes of up to 64 keys at once: the last key number of that look is up to 2048 beyond the length
    change = dict(page_size=page_size, page_stride=page_size * 576, max_pages=max_pages, table_stride=max_pages)
    if (max_pages * page_size - 1) // 64 * 64 + 31 * 64 >= 1 << 31 or max_pages * page_size > 0x7ffff000:
        assert attention(**change) == COUNT
    else:
        assert attention(**{**change, "workspace_bytes": 0}) == CAPACITY


def test_a_call_without_tokens_launches_nothing():
    assert append(n_tokens=0) == 0 and query(n_tokens=0) == 0 and value(n_tokens=0) == 0
    assert attention(batch=0) == 0 and attention(q_len=0) == 0


def test_wrappers_refuse_wrong_shapes_and_types():
    from vic_b200 import kernels
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    i32, i64, f64 = torch.int32, torch.int64, torch.float64
    good = dict(kv=z(2, 576), norm_weight=z(512), eps=1e-6, positions=z(2, dtype=i32), slots=z(2, dtype=i64), inv_freq=z(32, dtype=f64), cache=z(3, 8, 576))
    for name, bad in (("kv", z(2, 575)), ("kv", z(3, 576)), ("kv", z(2, 576, dtype=f64)), ("norm_weight", z(512, dtype=torch.float16)),
                      ("norm_weight", z(511)), ("positions", z(2, dtype=i64)), ("slots", z(2, dtype=i32)), ("inv_freq", z(32, dtype=torch.float32)),
                      ("cache", z(3, 8, 512)), ("cache", z(3, 8, 576, dtype=torch.float32)), ("cache", z(3, 576, 8).transpose(1, 2))):
        with pytest.raises(ValueError):
            kernels.latent_append(**{**good, name: bad})
    good = dict(q=z(2, 4, 192), w_uk=z(4, 128, 512), positions=z(2, dtype=i32), inv_freq=z(32, dtype=f64), out=z(2, 4, 576))
    for name, bad in (("q", z(2, 4, 190)), ("q", z(2, 3, 192)), ("w_uk", z(4, 128, 512, dtype=torch.float16)), ("w_uk", z(4, 512, 128).transpose(1, 2)),
                      ("out", z(2, 4, 512)), ("positions", z(3, dtype=i32))):
        with pytest.raises(ValueError):
            kernels.latent_query(**{**good, name: bad})
    good = dict(o=z(2, 4, 512), w_uv=z(4, 128, 512), out=z(2, 4, 128))
    for name, bad in (("o", z(2, 4, 576)), ("w_uv", z(3, 128, 512)), ("out", z(2, 4, 64)), ("out", z(2, 4, 128, dtype=torch.float32))):
        with pytest.raises(ValueError):
            kernels.latent_value(**{**good, name: bad})
    good = dict(q=z(4, 4, 576), cache=z(9, 8, 576), page_table=z(2, 4, dtype=i32), seq_lens=z(2, dtype=i32), scale=0.1, out=z(4, 4, 512),
                workspace=z(16, dtype=torch.uint8))
    for name, bad in (("q", z(3, 4, 576)), ("q", z(4, 4, 512)), ("cache", z(9, 8, 576, dtype=torch.float16)), ("page_table", z(3, 4, dtype=i32)),
                      ("page_table", z(2, 4, dtype=i64)), ("seq_lens", z(2, dtype=i64)), ("out", z(4, 4, 576)), ("lse", z(4, 4)), ("lse", z(4, 5, dtype=torch.float32))):
        with pytest.raises(ValueError):
            kernels.latent_attention(**{**good, name: bad})
