"""Forking, freeing and compacting the page pool, host side. CPU only."""
from __future__ import annotations

import random

import pytest

from techjam2026_b200.kvcache import PagePool, main


def consistent(pool):
    """Every page is free or used as often as rows name it; the table says the same."""
    count = [0] * len(pool.uses)
    for row in pool.rows:
        assert len(set(row)) == len(row)
        for p in row:
            count[p] += 1
    assert count == pool.uses
    assert sorted(pool.free) == [p for p, n in enumerate(count) if n == 0]
    for i, row in enumerate(pool.rows):
        assert pool.table[i, :len(row)].tolist() == row


def test_children_share_full_pages_and_copy_the_last_one():
    pool = PagePool(pages=12, batch=3, blocks=4, block=16, device="cpu")
    pool.reserve([40, 5, 0])
    a = list(pool.rows[0])
    copies = pool.fork([0, 0, 0], [40, 5, 0])
    consistent(pool)
    assert pool.rows[0] == a and [r[:2] for r in pool.rows] == [a[:2]] * 3
    assert [c[0] for c in copies] == [a[2]] * 2 and [c[2] for c in copies] == [8, 8]
    assert [c[1] for c in copies] == [pool.rows[1][2], pool.rows[2][2]]
    starts, shared, each = pool.groups
    assert starts.tolist() == [0, 3] and shared.tolist() == [32] and each == [32] * 3


def test_a_full_last_page_needs_no_copy_and_the_next_tokens_go_elsewhere():
    pool = PagePool(pages=6, batch=2, blocks=3, block=16, device="cpu")
    pool.reserve([32, 0])
    assert pool.fork([0, 0], [32, 0]) == []
    assert pool.rows[0] == pool.rows[1]
    pool.reserve([33, 33])
    consistent(pool)
    assert pool.rows[0][:2] == pool.rows[1][:2] and pool.rows[0][2] != pool.rows[1][2]


def test_a_parent_without_children_ends_and_an_only_child_moves():
    pool = PagePool(pages=8, batch=3, blocks=2, block=16, device="cpu")
    pool.reserve([20, 30, 10])
    b = list(pool.rows[1])
    assert pool.fork([1, 2, 1], [20, 30, 10])[0][0] == b[1]
    consistent(pool)
    assert pool.rows[0] == b and pool.rows[2][0] == b[0]
    # rows 0 and 2 share, but row 1 stands between them
    assert pool.groups is None


def test_whole_copies_share_nothing():
    pool = PagePool(pages=9, batch=3, blocks=3, block=16, device="cpu")
    pool.reserve([40, 0, 0])
    copies = pool.fork([0, 0, 0], [40, 0, 0], whole=True)
    consistent(pool)
    assert [c[2] for c in copies] == [16, 16, 8] * 2 and pool.groups is None
    assert max(pool.uses) == 1


def test_a_fork_that_does_not_fit_changes_nothing():
    pool = PagePool(pages=4, batch=4, blocks=3, block=16, device="cpu")
    pool.reserve([17, 17, 0, 0])
    before = [list(r) for r in pool.rows], list(pool.free), list(pool.uses)
    with pytest.raises(RuntimeError):
        pool.fork([0, 0, 1, 1], [17, 17, 0, 0])
    assert before == ([list(r) for r in pool.rows], list(pool.free), list(pool.uses))
    # pages of a sequence that ends serve the copies
    pool.fork([0, 0, 0, 0][:1] + [0, 0, 2], [17, 17, 0, 0])
    consistent(pool)


def test_compaction_moves_the_highest_pages_into_the_lowest_holes():
    pool = PagePool(pages=10, batch=3, blocks=3, block=16, device="cpu")
    pool.reserve([33, 33, 33])
    pool.replace([[]], [0])
    moves = pool.compact()
    consistent(pool)
    assert sorted(p for r in pool.rows for p in r) == list(range(6))
    assert all(a >= 6 > b for a, b in moves) and pool.compact() == []
    pool.reserve([33, 33, 33])
    consistent(pool)


def test_random_histories_keep_the_books():
    rng = random.Random(0)
    pool = PagePool(pages=60, batch=5, blocks=6, block=16, device="cpu")
    held = [0] * 5
    for _ in range(300):
        what = rng.choice(["grow", "fork", "free", "compact"])
        if what == "grow":
            want = [min(96, n + rng.randint(0, 20)) for n in held]
            pool.reserve(want)
            held = want
            # no sequence writes into a page that another one has
            for i, row in enumerate(pool.rows):
                if held[i] % 16:
                    assert pool.uses[row[held[i] // 16]] == 1
        elif what == "fork":
            parents = [rng.randrange(5) for _ in range(5)]
            old = [list(r) for r in pool.rows]
            copies = pool.fork(parents, held)
            for a, b, n in copies:
                assert any(a in r for r in old) and 0 < n < 16 and pool.uses[b] == 1
            held = [held[p] for p in parents]
            for i, p in enumerate(parents):
                full = held[i] // 16
                assert pool.rows[i][:full] == old[p][:full]
        elif what == "free":
            i = rng.randrange(5)
            pool.replace([[]], [i])
            held[i] = 0
        else:
            pool.compact()
        consistent(pool)
        if pool.groups is not None:
            starts, shared, each = (x if isinstance(x, list) else x.tolist() for x in pool.groups)
            assert starts[0] == 0 and starts[-1] == 5 and starts == sorted(starts)
            for a, z, n in zip(starts, starts[1:], shared):
                assert len({tuple(r[:n // 16]) for r in pool.rows[a:z]}) == 1
                assert all(each[i] == n <= held[i] for i in range(a, z))


def rows_that_share(common, own=2, block=16):
    """A pool in which row i has common[i] leading pages in common with row i - 1."""
    B, blocks = len(common), max(common) + own + 1
    pool = PagePool(pages=B * blocks, batch=B, blocks=blocks, block=block, device="cpu")
    rows = [pool.take(blocks)]
    for n in common[1:]:
        rows.append(rows[-1][:n] + pool.take(blocks - n))
    pool.replace(rows)
    consistent(pool)
    return pool


@pytest.mark.parametrize("common,starts,shared", [
    ([0, 10, 10, 1], [0, 3, 4], [10, 0]),           # the last one has only the beginning
    ([0, 1, 10, 10], [0, 1, 4], [0, 10]),           # the first one
    ([0, 10, 10, 1, 10, 10], [0, 3, 6], [10, 10]),  # two prompts behind one beginning
    ([0, 10, 9, 10], [0, 4], [9]),                  # nearly the same: one group
    ([0, 3, 0, 5], [0, 2, 4], [3, 5]),
    ([0, 2, 2, 2, 9], [0, 3, 5], [2, 9]),           # 4 * 2 or 2 * 2 + 9 reads saved
    ([0, 5, 11, 6, 5], [0, 5], [5]),                # 4 * 5 or 11 and less
    ([0, 0, 4], [0, 1, 3], [0, 4]),
])
def test_a_sequence_with_little_in_common_takes_nothing_from_a_group(common, starts, shared):
    pool = rows_that_share(common)
    assert pool.groups[0].tolist() == starts
    assert pool.groups[1].tolist() == [16 * n for n in shared]
    assert pool.groups[2] == [16 * n for (a, z), n in zip(zip(starts, starts[1:]), shared)
                              for _ in range(z - a)]


def test_groups_save_at_least_as_much_as_one_for_each_first_page():
    """Against groups of all consecutive rows that begin with one page."""
    rng = random.Random(1)
    for _ in range(500):
        common = [0] + [rng.choice([0, 1, 2, 3, 5, 6, 8, 11]) for _ in range(rng.randint(1, 9))]
        pool = rows_that_share(common)
        saved = 0
        if pool.groups is not None:
            starts, shared = pool.groups[0].tolist(), pool.groups[1].tolist()
            for a, z, n in zip(starts, starts[1:], shared):
                assert len({tuple(r[:n // 16]) for r in pool.rows[a:z]}) == 1
                assert z - a > 1 or n == 0
                saved += (z - a - 1) * n // 16
        plain, run = 0, []
        for n in common[1:] + [0]:
            if n:
                run.append(n)
            else:
                plain += len(run) * min(run, default=0)
                run = []
        assert saved >= plain


@pytest.mark.parametrize("argv", [["--beams", "129"], ["--beams", "-1"],
                                  ["--beams", "2", "--vocab", "3"]])
def test_the_example_refuses_beams_it_cannot_run(argv, capsys):
    with pytest.raises(SystemExit) as told:
        main(argv)
    assert told.value.code == 2
    assert "--beams" in capsys.readouterr().err
