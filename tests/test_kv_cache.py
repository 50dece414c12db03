"""The page bookkeeping of ls.KvCache and the plans of attention over shared pages (no GPU: device=-1).

The tables are checked against a Python restatement (lowest free page first, a page copied when one of
several holders is about to write into it, the last holder writes in place), and every step's plan by
the library's own check: each row's positions are covered exactly once, through the pages of its own
table, inside the workspaces.
"""

import numpy as np
import pytest

import layerstream_b200 as ls

ARG = -1


def cache(seqs=4, page=8, num_pages=64, max_ctx=128, max_rows=256, heads=4, kv_heads=2, hd=64, **kw):
    return ls.KvCache(0, 0, layers=2, heads=heads, kv_heads=kv_heads, hd=hd, page=page, num_pages=num_pages, seqs=seqs, max_ctx=max_ctx,
                      max_rows=max_rows, device=-1, **kw)


class Restated:
    """Page tables as lists, page counts recomputed from them."""

    def __init__(self, seqs, page, num_pages):
        self.t, self.n, self.page, self.num_pages = [[] for _ in range(seqs)], [0] * seqs, page, num_pages

    def refs(self):
        return np.bincount([p for t in self.t for p in t], minlength=self.num_pages)

    def need(self, n):
        return -(-n // self.page)

    def take(self):
        return int(np.flatnonzero(self.refs() == 0)[0])

    def fork(self, src, dst, n):
        for d in dst:
            self.t[d], self.n[d] = self.t[src][: self.need(n)], n

    def truncate(self, s, n):
        self.n[s] = n
        self.t[s] = self.t[s][: self.need(n)]

    def begin(self, counts):
        for s, c in enumerate(counts):
            if not c:
                continue
            for i in range(self.n[s] // self.page, self.need(self.n[s] + c)):
                if i >= len(self.t[s]):
                    self.t[s].append(self.take())
                elif self.refs()[self.t[s][i]] > 1:
                    self.t[s][i] = self.take()

    def end(self, counts, keep):
        for s, c in enumerate(counts):
            if c:
                self.truncate(s, self.n[s] + keep[s])

    def tables(self, max_pages):
        return np.array([t + [-1] * (max_pages - len(t)) for t in self.t], np.int32)


@pytest.mark.parametrize("seed", range(8))
def test_tables_follow_forks_steps_truncation_and_compaction(seed):
    rng = np.random.default_rng(seed)
    seqs, page = int(rng.integers(2, 9)), int(rng.choice([8, 16, 64]))
    max_ctx, M = 40 * 8, int(rng.integers(1, 20))
    num_pages = seqs * (-(-max_ctx // page))
    kv = cache(seqs=seqs, page=page, num_pages=num_pages, max_ctx=max_ctx, max_rows=seqs * M)
    py = Restated(seqs, page, num_pages)
    for step in range(60):
        what = rng.integers(0, 6)
        if what == 0:
            src = int(rng.integers(seqs))
            dst = [int(d) for d in rng.permutation(seqs)[: rng.integers(1, seqs)] if d != src]
            n = int(rng.integers(0, py.n[src] + 1))
            kv.fork(src, dst, n)
            py.fork(src, dst, n)
        elif what == 1:
            s = int(rng.integers(seqs))
            n = int(rng.integers(0, py.n[s] + 1))
            kv.truncate(s, n)
            py.truncate(s, n)
        elif what == 2:
            used = np.flatnonzero(py.refs())
            free_low = [p for p in range(len(used)) if p not in set(used.tolist())]
            to = dict(zip([int(p) for p in used if p >= len(used)], free_low))
            assert kv.compact() == len(to)
            py.t = [[to.get(p, p) for p in t] for t in py.t]
        else:
            counts = [int(min(rng.integers(0, M + 1), max_ctx - n)) for n in py.n]
            kv.begin(counts, M)
            py.begin(counts)
            kv.self_check()
            assert np.array_equal(kv.tables(), py.tables(kv.max_pages))
            if what < 5:  # otherwise the step is dropped: its pages stay with the sequences
                keep = [int(rng.integers(0, c + 1)) for c in counts]
                kv.end(keep)
                py.end(counts, keep)
        kv.self_check()
        assert np.array_equal(kv.tables(), py.tables(kv.max_pages)), (step, what)
        assert [kv.length(s) for s in range(seqs)] == py.n
        i = kv.info
        assert (i.pages_used, i.pages_shared) == (int((py.refs() > 0).sum()), int((py.refs() > 1).sum()))


@pytest.mark.parametrize("seed", range(12))
def test_plans_cover_every_rows_positions_once(seed):
    # prompts forked, forks forked again, ragged rows, long and short tails, pages below and above a chunk
    rng = np.random.default_rng(100 + seed)
    heads, kv_heads = [(14, 2), (16, 2), (4, 4), (5, 1), (32, 8)][seed % 5]
    page = int(rng.choice([8, 32, 64, 128, 512]))
    seqs, M = int(rng.integers(2, 14)), int(rng.choice([1, 3, 9, 40]))
    max_ctx = 6000
    num_pages = seqs * (-(-max_ctx // page))
    kv = cache(seqs=seqs, page=page, num_pages=num_pages, max_ctx=max_ctx, max_rows=seqs * M, heads=heads, kv_heads=kv_heads)
    ids = rng.permutation(num_pages)
    base = int(rng.integers(0, 4000))
    kv.set_table(0, ids[: -(-(base + 1) // page)], base)
    lens = [base] + [0] * (seqs - 1)
    for s in range(1, seqs):
        src = int(rng.integers(0, s))
        n = int(rng.integers(0, lens[src] + 1)) if rng.random() < 0.3 else lens[src]
        kv.fork(src, s, n)
        lens[s] = n
        for _ in range(int(rng.integers(0, 4))):  # some rows of its own
            c = int(rng.integers(1, M + 1))
            kv.begin([c if i == s else 0 for i in range(seqs)], M)
            kv.end()
            lens[s] += c
    for counts in ([M] * seqs, rng.integers(0, M + 1, seqs).tolist(), [0] * (seqs - 1) + [1], [0] * seqs):
        kv.begin(counts, M)
        kv.self_check()
        shared = kv.info.shared_positions
        assert shared <= max(lens) * 2
    kv.close()


def test_a_long_shared_prefix_is_read_once():
    kv = cache(seqs=16, page=64, num_pages=200, max_ctx=6000, max_rows=16)
    kv.set_table(0, range(64), 4096)
    kv.fork(0, range(1, 16))
    kv.begin([1] * 16, 1)
    kv.self_check()
    assert kv.info.shared_positions == 4096
    kv.end()
    kv.begin([1] * 16, 1)  # the grown tails are not shared
    kv.self_check()
    assert kv.info.shared_positions == 4096
    kv.end()
    # two prompts under one system prompt: the common part, then each prompt's own part
    kv = cache(seqs=8, page=64, num_pages=400, max_ctx=6000, max_rows=8)
    kv.set_table(0, range(32), 2048)
    kv.set_table(4, list(range(16)) + list(range(100, 132)), 48 * 64)
    kv.fork(0, range(1, 4))
    kv.fork(4, range(5, 8))
    kv.begin([1] * 8, 1)
    kv.self_check()
    assert kv.info.shared_positions == 1024 + 1024 + 2048


def test_the_last_holder_of_a_page_writes_in_place():
    kv = cache(seqs=3, page=8, num_pages=16)
    kv.begin([5, 0, 0], 5)
    kv.end()
    kv.fork(0, [1, 2])
    kv.begin([1, 1, 1], 1)
    assert kv.tables()[:, 0].tolist() == [1, 2, 0]
    kv.self_check()


def refuses(fn, *a, match=None, code=ARG, **kw):
    with pytest.raises(ls.LayerstreamError, match=match) as e:
        fn(*a, **kw)
    assert e.value.code == code


def test_refusals_leave_the_tables_as_they_were():
    kv = cache(seqs=3, page=8, num_pages=6, max_ctx=40, max_rows=9)
    kv.begin([3, 3, 0], 3)
    kv.end()
    kv.fork(0, 2)
    before = kv.tables()
    refuses(kv.fork, 0, 0, match="onto itself")
    refuses(kv.fork, 0, [1, 1], match="named twice")
    refuses(kv.fork, 0, [1, 3], match="outside the cache")
    refuses(kv.fork, 5, 1, 0, match="outside the cache")
    refuses(kv.fork, 0, 1, 4, match="holds 3 positions")
    refuses(kv.truncate, 0, 4, match="cannot truncate")
    refuses(kv.truncate, 3, 0, match="outside the cache")
    refuses(kv.set_table, 1, [0, 6], 9, match="outside the pool")
    refuses(kv.set_table, 1, [-1], 1, match="outside the pool")
    refuses(kv.set_table, 1, [2, 2], 9, match="named twice")
    refuses(kv.set_table, 1, [2], 9, match="fewer than n")
    refuses(kv.set_table, 1, [0, 1, 2, 3, 4, 5], 9, match="more pages")
    refuses(kv.begin, [1, 1, 4], 3, match="more than M")
    refuses(kv.begin, [1, 1, 1], 0, match="max_rows")
    refuses(kv.begin, [1, 1, 1], 4, match="max_rows")
    refuses(kv.end, match="no step")
    kv.begin([1, 0, 0], 1)
    refuses(kv.end, [2, 0, 0], match="keep more")
    refuses(kv.attention, 0, 16, 16, match="pages only")
    kv.truncate(1, 3)
    refuses(kv.end, match="no step")  # the table changed since
    with pytest.raises(ValueError):
        kv.begin([1, 1], 1)
    with pytest.raises(ValueError):
        kv.begin([1, -1, 0], 1)
    assert np.array_equal(kv.tables()[1], before[1])
    kv.self_check()


def test_an_exhausted_pool_refuses_the_step_and_changes_nothing():
    kv = cache(seqs=3, page=8, num_pages=4, max_ctx=32, max_rows=24)
    kv.begin([8, 8, 0], 8)
    kv.end()
    kv.truncate(0, 5)
    kv.fork(0, 2)
    # free pages: 2. Needed: 0 and 2 write into one shared page (one copy), 1 takes one page; then 0 and 2 grow
    before = kv.tables()
    refuses(kv.begin, [8, 1, 8], 8, match="exhausted")
    assert np.array_equal(kv.tables(), before)
    kv.self_check()
    kv.begin([1, 1, 1], 8)
    kv.self_check()
    assert kv.info.pages_used == 4
    kv = cache(seqs=1, page=8, num_pages=64, max_ctx=16, max_rows=16)
    refuses(kv.begin, [17], 17, match="max_rows")
    kv.begin([16], 16)
    kv.end()
    refuses(kv.begin, [1], 1, match="context is full")


@pytest.mark.parametrize("kw", [dict(hd=32), dict(hd=96), dict(page=4), dict(page=48), dict(page=1 << 17), dict(num_pages=0), dict(seqs=0),
                                dict(seqs=5000), dict(max_ctx=0), dict(max_rows=0), dict(heads=5), dict(heads=0), dict(kv_heads=0),
                                dict(num_pages=1 << 29), dict(max_rows=1 << 20)])
def test_open_refuses(kw):
    refuses(cache, **kw)


def test_copy_pages_refuses_before_it_touches_the_gpu():
    def call(src, dst, rows=None, k=1 << 20, v=1 << 20, layers=2, kv_heads=2, hd=64, page=8, num_pages=16):
        ls.kv_copy_pages(k, v, layers, kv_heads, hd, page, num_pages, src, dst, rows)

    call([], [])
    refuses(call, [0], [0], match="both read and written|also read")
    refuses(call, [0, 1], [2, 2], match="written twice")
    refuses(call, [0, 2], [2, 3], match="both read and written")
    refuses(call, [0, 3], [3, 1], match="both read and written")
    refuses(call, [1, 2], [3, 1], match="also read")
    refuses(call, [16], [0], match="outside the pool")
    refuses(call, [0], [16], match="outside the pool")
    refuses(call, [-1], [0], match="outside the pool")
    refuses(call, [0], [1], [9], match="rows must")
    refuses(call, [0], [1], [-1], match="rows must")
    refuses(call, [0], [1], k=0, match="NULL")
    refuses(call, [0], [1], k=8, match="aligned")
    refuses(call, [0], [1], hd=12, match="head size")
    refuses(call, [0], [1], page=12, match="page")
    refuses(call, [0], [1], layers=0, match="layers")
    refuses(call, list(range(16)) + [0], list(range(17)), match="more copies|outside")
    with pytest.raises(ValueError):
        call([0, 1], [2])


def test_page_ids_that_do_not_fit_32_bits_are_refused():
    kv = cache()
    for ids in ([2**32], np.array([2**32]), np.array([2**31], np.uint64)):
        with pytest.raises(OverflowError):
            kv.set_table(0, ids, 0)
        with pytest.raises(OverflowError):
            ls.kv_copy_pages(1 << 20, 1 << 20, 1, 1, 64, 16, 8, ids, [0])
    with pytest.raises(ValueError, match="same length"):
        ls.kv_copy_pages(1 << 20, 1 << 20, 1, 1, 64, 16, 8, [1, 2], [0])
