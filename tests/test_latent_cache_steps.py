"""Steps that follow one another in the same device buffers (no GPU needed)."""
import torch

from tests.test_latent_cache import make, slots_of


def test_slots_behind_a_smaller_step_are_none():
    """A captured step of more rows than the one laid out must not append over rows in use: it finds no slot behind the step's."""
    c = make(pages=12, max_tokens=24)
    assert c.slots.tolist() == [-1] * 24
    for new in ([4, 4, 4], [1, 1, 1], [2, 0, 3], [0, 0, 0], [7, 1, 1], [1, 0, 0], [8, 8, 8]):
        before = list(c.host_lens)
        c.begin_step(new)
        q = max(new)
        want = sum(([-1] * (q - k) + slots_of(c, b, before[b], before[b] + k) for b, k in enumerate(new)), [])
        assert c.step_rows == len(want) and c.slots.tolist() == want + [-1] * (24 - len(want)), new
        assert c.positions[len(want):].eq(0).all(), new
