"""The limit on a call's tiles that the header states, from its far side (a call within it would be launched).  No GPU is needed."""
import pytest

from tests.test_latent_refusals import COUNT, attention


@pytest.mark.parametrize("batch,q_len,heads,pages", [(4096, 256, 128, 4096), (8192, 128, 64, 1 << 13), (100000, 9, 64, 1 << 14), (1 << 20, 1, 1, 1 << 13)])
def test_more_tiles_than_32_bits_count_are_refused(batch, q_len, heads, pages):
    blocks = -(-q_len * heads // 64)
    blocks = 1 if blocks <= 8 else blocks
    assert batch * blocks * (pages * 16 // 64 + 4) > 2 ** 31 - 256
    assert attention(batch=batch, q_len=q_len, heads=heads, max_pages=pages, table_stride=pages, q_token=heads * 576, out_token=heads * 512) == COUNT
