"""The host side of the latent cache: pages, slots and positions of a step's tokens (no GPU needed)."""
import pytest
import torch


def make(**k):
    from vic_b200.attention import LatentCache
    a = dict(layers=2, pages=6, page_size=8, max_sequences=3, max_pages=4, dtype=torch.bfloat16, device="cpu", max_tokens=64)
    a.update(k)
    return LatentCache(**a)


def slots_of(cache, b, lo, hi):
    return [int(cache.table[b, p // cache.page_size]) * cache.page_size + p % cache.page_size for p in range(lo, hi)]


def test_steps_give_every_token_a_slot_of_its_own():
    c = make()
    c.begin_step([5, 0, 9])                                     # a chunk of 9 rows per sequence, the shorter ones padded in front
    assert c.lens.tolist() == [5, 0, 9]
    assert c.slots[:27].tolist() == [-1] * 4 + slots_of(c, 0, 0, 5) + [-1] * 9 + slots_of(c, 2, 0, 9)
    assert c.positions[:27].tolist() == [0] * 4 + list(range(5)) + [0] * 9 + list(range(9))
    seen = set(slots_of(c, 0, 0, 5) + slots_of(c, 2, 0, 9))
    assert len(seen) == 14
    for step in range(4):
        c.begin_step([1, 1, 0])
        assert c.slots[:3].tolist() == slots_of(c, 0, 5 + step, 6 + step) + slots_of(c, 1, step, step + 1) + [-1]
        assert c.positions[:3].tolist() == [5 + step, step, 0]
        new = [s for s in c.slots[:3].tolist() if s >= 0]
        assert not seen & set(new)
        seen |= set(new)
    assert c.lens.tolist() == [9, 4, 9]


def test_a_full_cache_refuses_the_step_and_stays_as_it_was():
    from vic_b200.lib import Vib3Error
    c = make()
    c.begin_step([16, 16, 8], q_len=16)
    before = (c.lens.tolist(), c.table.tolist(), list(c._free))
    with pytest.raises(Vib3Error):
        c.begin_step([1, 1, 0])                                 # two pages wanted, one left
    with pytest.raises(ValueError):
        c.begin_step([1, 1])
    with pytest.raises(ValueError):
        c.begin_step([2, 0, 0], q_len=1)
    with pytest.raises(ValueError):
        c.begin_step([-1, 0, 0], q_len=1)
    with pytest.raises(ValueError):
        c.begin_step([30, 0, 0])
    assert before == (c.lens.tolist(), c.table.tolist(), list(c._free)) and c.host_lens == [16, 16, 8]
    c.begin_step([1, 0, 0])
    with pytest.raises(Vib3Error):
        c.begin_step([0, 1, 0])
    c.release(2)
    c.begin_step([0, 1, 1], q_len=1) if len(c._free) > 1 else c.begin_step([0, 1, 0], q_len=1)
    assert c.host_lens[1] == 17


def test_a_sequence_has_no_more_pages_than_its_table():
    from vic_b200.lib import Vib3Error
    c = make(pages=100, max_tokens=200)
    c.begin_step([32, 0, 0])
    with pytest.raises(Vib3Error):
        c.begin_step([1, 0, 0])
    c.release(0)
    c.begin_step([1, 0, 0])
    assert c.lens.tolist() == [1, 0, 0]


def test_the_table_follows_pages_that_come_and_go():
    c = make(pages=12)
    steps = [[9, 8, 1], [0, 1, 0], "release 1", [8, 3, 0], "release 0", "release 2", [1, 0, 20], [0, 0, 0], [7, 1, 1], [1, 0, 0]]
    for s in steps:
        if isinstance(s, str):
            c.release(int(s[-1]))
            continue
        c.begin_step(s)
        used = [p for own in c._pages_of for p in own]
        assert len(used) == len(set(used)) and not set(used) & set(c._free) and len(used) + len(c._free) == 12
        for b, own in enumerate(c._pages_of):
            assert len(own) == -(-c.host_lens[b] // 8) and c.table[b].tolist() == own + [0] * (4 - len(own))


def test_a_layer_takes_the_rows_of_the_step_and_no_others():
    from vic_b200.attention import LatentAttention
    from vic_b200.core_types import LatentShape
    c = make(max_tokens=12)
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    sh = LatentShape("small", 64, 2, 16, 16, 10000.0, 1e-6)
    layer = LatentAttention(sh, z(2 * 80, 64), z(576, 64), z(512), z(2, 32, 512), z(64, 32), max_tokens=12, workspace=torch.zeros(16, dtype=torch.uint8))
    with pytest.raises(ValueError, match="rows"):
        layer.forward(z(3, 64), c, 0)                           # no step yet
    c.begin_step([4, 4, 4])
    c.begin_step([1, 1, 1])
    for rows in (6, 12):                                        # the slots behind row 3 are the older step's
        with pytest.raises(ValueError, match="rows"):
            layer.forward(z(rows, 64), c, 0)
    with pytest.raises(Exception):
        c.begin_step([30, 0, 0])                                # refused: the step stays the one before
    assert c.step_rows == 3


def test_bad_layouts_are_refused():
    with pytest.raises(ValueError):
        make(page_size=12)
    with pytest.raises(ValueError):
        make(max_tokens=2)
