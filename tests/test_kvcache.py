"""The page pool's host side. CPU only."""
from __future__ import annotations

import pytest

from techjam2026_b200.kvcache import PagePool, main


def test_pages_are_handed_out_once_and_come_back():
    pool = PagePool(pages=7, batch=2, blocks=3, block=16, device="cpu")
    pool.reserve([1, 33])
    assert [len(r) for r in pool.rows] == [1, 3] and len(pool.free) == 3
    pool.reserve([16, 40])                        # still the same pages
    assert [len(r) for r in pool.rows] == [1, 3]
    used = [p for r in pool.rows for p in r]
    assert len(set(used + pool.free)) == 7
    assert pool.table[0, 0] == pool.rows[0][0]
    assert pool.table[1].tolist() == pool.rows[1]
    rows = [pool.take(1), pool.take(2)]
    pool.replace(rows)
    assert pool.rows == rows and len(pool.free) == 4
    assert sorted(pool.free + rows[0] + rows[1]) == list(range(7))


def test_a_full_pool_and_a_long_sequence_are_refused():
    pool = PagePool(pages=3, batch=2, blocks=3, block=16, device="cpu")
    with pytest.raises(RuntimeError):
        pool.reserve([0, 49])
    with pytest.raises(RuntimeError):
        pool.reserve([33, 17])


def test_a_refused_reservation_changes_nothing():
    """The first sequence's pages are there, the second one's are not: neither
    gets any, and a later reservation that fits is on the table."""
    pool = PagePool(pages=3, batch=2, blocks=3, block=16, device="cpu")
    pool.table.fill_(-1)
    with pytest.raises(RuntimeError):
        pool.reserve([33, 17])
    assert pool.rows == [[], []] and len(pool.free) == 3
    pool.reserve([33, 0])
    assert sorted(pool.rows[0]) == [0, 1, 2] and pool.rows[1] == []
    assert pool.table[0].tolist() == pool.rows[0]
    with pytest.raises(RuntimeError):
        pool.reserve([33, 1])
    assert pool.rows[1] == [] and pool.table[0].tolist() == pool.rows[0]


def test_pages_of_some_sequences_are_replaced():
    pool = PagePool(pages=9, batch=3, blocks=3, block=16, device="cpu")
    pool.reserve([40, 20, 33])
    before = [list(r) for r in pool.rows]
    rows = [pool.take(1)]
    pool.replace(rows, [1])
    assert pool.rows == [before[0], rows[0], before[2]]
    assert sorted(pool.free) == sorted(before[1])
    assert pool.table[0].tolist() == before[0] and pool.table[2].tolist() == before[2]
    assert pool.table[1, 0] == rows[0][0]


@pytest.mark.parametrize("argv", [["--config", "c3a"], ["--config", "c3b"], ["--tokens", "0"],
                                  ["--config", "c1", "--tokens", "64"]])
def test_the_example_refuses_what_it_cannot_run(argv, capsys):
    """Heads of 8 and 256, no single token, no prompt: a usage error, not a
    traceback from inside the cache."""
    with pytest.raises(SystemExit) as told:
        main(argv)
    assert told.value.code == 2
    said = capsys.readouterr().err
    assert argv[-2] in said and "usage" in said
