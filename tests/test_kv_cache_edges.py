"""Steps of ls.KvCache in orders and with arguments that the other tests do not make (no GPU: device=-1)."""

import numpy as np
import pytest

import layerstream_b200 as ls
from test_kv_cache import cache, refuses


def prompts(n, seqs=8, M=128, page=64):
    """Sequences forked under the same n positions."""
    kv = cache(seqs=seqs, page=page, num_pages=n // page + 1 + seqs * 8, max_ctx=n + 512, max_rows=seqs * M, heads=14, kv_heads=2)
    kv.set_table(0, range(-(-n // page)), n)
    kv.fork(0, range(1, seqs))
    return kv


@pytest.mark.parametrize("n", [4096, 4100])
@pytest.mark.parametrize("rows", [[128, 1, 1], [1, 128, 1], [1, 32, 5, 128, 128, 2], [33, 40, 33]])
def test_what_a_step_shares_depends_on_its_own_rows_alone(n, rows):
    # (32, 33 or 128 rows of 7 heads fill four fifths of their pairs of tiles and are planned alone, the others are not)
    kv = prompts(n)
    for r in rows:
        kv.begin([r] * 8, 128)
        kv.self_check()
        fresh = prompts(n)
        fresh.begin([r] * 8, 128)
        assert kv.info.shared_positions == fresh.info.shared_positions == (0 if r in (32, 33, 128) else 4096), r
        kv.end()


def test_sequences_with_many_rows_beside_sequences_with_few():
    kv = prompts(4096)
    for counts in ([128] * 4 + [1] * 4, [1] * 4 + [128] * 4, [1] * 8, [0, 0, 0, 1, 0, 0, 128, 128], [2] * 8):
        kv.begin(counts, 128)
        kv.self_check()
        few = sum(1 for c in counts if 0 < c < 100)
        assert kv.info.shared_positions == (4096 if few > 1 else 0), counts


@pytest.mark.parametrize("M", [2**62, 2**63, 2**63 + 1, 2**64 - 1, 5])
def test_begin_refuses_more_rows_than_the_workspaces_hold(M):
    # seqs x M of the large ones is 0, 0, 4 and -4 modulo 2^64
    kv = cache(seqs=4, max_rows=16)
    refuses(kv.begin, [1, 1, 1, 1], M, match="max_rows")
    assert kv.info.pages_used == 0
    kv.self_check()


@pytest.mark.parametrize("seed", range(6))
def test_a_begin_that_fails_changes_nothing(seed):
    # forks, rollbacks and dropped steps; now and then a begin fails at its launches, and is then made again: the
    # tables are always those of a cache where none failed
    rng = np.random.default_rng(seed)
    a, b = (cache(seqs=5, page=8, num_pages=60, max_ctx=96, max_rows=60) for _ in range(2))
    both = (a, b)
    for step in range(50):
        what = rng.integers(0, 5)
        if what == 0:
            src = int(rng.integers(5))
            dst = [int(d) for d in rng.permutation(5)[:2] if d != src]
            n = int(rng.integers(0, a.length(src) + 1))
            for kv in both:
                kv.fork(src, dst, n)
        elif what == 1:
            s = int(rng.integers(5))
            n = int(rng.integers(0, a.length(s) + 1))
            for kv in both:
                kv.truncate(s, n)
        else:
            counts = [int(min(rng.integers(0, 13), 96 - a.length(s))) for s in range(5)]
            before, info = a.tables(), a.info
            a.inject_error()
            refuses(a.begin, counts, 12, match="test hook", code=-3)
            a.self_check()
            assert np.array_equal(a.tables(), before)
            assert (a.info.pages_used, a.info.pages_shared) == (info.pages_used, info.pages_shared)
            refuses(a.end, match="no step")
            for kv in both:
                kv.begin(counts, 12)
            a.self_check()
            assert a.info.shared_positions == b.info.shared_positions
            assert np.array_equal(a.tables(), b.tables())
            if what < 4:
                keep = [int(rng.integers(0, c + 1)) for c in counts]
                for kv in both:
                    kv.end(keep)
        a.self_check()
        assert np.array_equal(a.tables(), b.tables()), step
    a.inject_error()
    a.inject_error(0)
    a.begin([0] * 5, 1)
    for code in (-1, 2, 3):
        refuses(a.inject_error, code)


@pytest.mark.parametrize("heads,hd", [(14, 64), (16, 128), (6, 64)])
@pytest.mark.parametrize("prefix", [512, 2048, 8192, 32768])
def test_no_cta_gets_the_rest_of_the_work(heads, hd, prefix):
    # (self_check compares every CTA's share with the mean) shared tiles in pairs and single ones, long and short ranges
    for seqs in (1, 2, 4, 8, 32):
        for M in (1, 3, 5, 9, 12, 16, 20, 33, 40, 48, 64):
            kv = cache(seqs=seqs, page=64, num_pages=prefix // 64 + 3 * seqs, max_ctx=prefix + 192, max_rows=seqs * M, heads=heads, hd=hd)
            for s in range(seqs):
                kv.set_table(s, [*range(prefix // 64), *range(prefix // 64 + 3 * s, prefix // 64 + 3 * s + 3)], prefix + 100)
            kv.begin([M] * seqs, M)
            kv.self_check()
            kv.close()


def test_fork_takes_any_integer_and_any_sequence_of_them():
    kv = cache(seqs=6)
    kv.begin([5, 0, 0, 0, 0, 0], 5)
    kv.end()
    for dst in (np.int64(1), np.uint32(2), [np.int32(3)], (5,), np.array([1, 2]), range(3, 5)):
        kv.fork(0, dst)
    assert [kv.length(s) for s in range(6)] == [5] * 6
    for dst in (-1, [1, -2], np.int64(-1)):
        with pytest.raises(ValueError):
            kv.fork(0, dst)
    for dst in (1.0, [1.5], "12"):
        with pytest.raises(TypeError):
            kv.fork(0, dst)
    kv.self_check()


def test_pages_that_are_no_integers_are_refused():
    kv = cache()
    kv.set_table(1, [3, np.int64(4)], 9)
    before = kv.tables()
    for ids in ([0.5], [1.0], np.array([1.5, 2.5]), ["1"], [None]):
        with pytest.raises(TypeError):
            kv.set_table(0, ids, 0)
        with pytest.raises(TypeError):
            ls.kv_copy_pages(1 << 20, 1 << 20, 1, 1, 64, 16, 8, ids, list(range(len(ids))))
        with pytest.raises(TypeError):
            ls.kv_copy_pages(1 << 20, 1 << 20, 1, 1, 64, 16, 8, list(range(len(ids))), list(range(4, 4 + len(ids))), ids)
    for ids in ((5, 6), range(5, 7), np.array([5, 6], np.uint8), [np.int32(5), 6]):
        kv.set_table(0, ids, 9)
        assert kv.tables()[0, :3].tolist() == [5, 6, -1]
    assert np.array_equal(kv.tables()[1], before[1])
    ls.kv_copy_pages(1 << 20, 1 << 20, 1, 1, 64, 16, 8, [], [], [])
