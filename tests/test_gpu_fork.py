"""Forked sequences of a batch (needs a B200): Batch.fork shares the prompt's K/V pages, the verify passes copy a
page before one of several holders writes into it, and read the shared prefix once for all sequences.

Each sequence must decode as it would alone: bit for bit on the tiny model (head size 16, where forks
share pages and every sequence reads its own context), and at the 0.5B and 3B widths (head sizes 64 and
128, attention over shared pages) wherever the top-2 margins of a single-sequence model exceed 2e-2.
"""

import os

import numpy as np
import pytest

import fixtures as F
import layerstream_b200 as ls
from layerstream_b200 import synth
from oracle import oracle as O

pytestmark = pytest.mark.gpu

TOL = 2e-2
ROOT = os.environ.get("LS_BENCH_ROOT", "/tmp/ls_b200_bench")


@pytest.fixture(scope="module")
def tiny():
    d = F.TempDir("gpu-fork").path
    F.write_tiny_model(d, 13)
    p = os.path.join(d, "q8g32.lsq")
    O.quantize_model(d, p, (8, 32), (8, 32), clip=True)
    yield p


def with_page(page, f):
    old = os.environ.get("LS_KV_PAGE")
    os.environ["LS_KV_PAGE"] = str(page)
    try:
        return f()
    finally:
        if old is None:
            del os.environ["LS_KV_PAGE"]
        else:
            os.environ["LS_KV_PAGE"] = old


@pytest.mark.parametrize("page", [8, 64])
def test_forked_sequences_decode_like_separately_prefilled_ones(tiny, page):
    prompt = F.PROMPT + list(range(200, 231))
    base = ls.Model(tiny, max_ctx=256)
    forked = with_page(page, lambda: ls.Batch(base, 4, max_ctx=160, max_block=5))
    plain = with_page(page, lambda: ls.Batch(base, 4, max_ctx=160, max_block=5))
    first = forked.prefill(0, prompt)
    forked.fork(0, [1, 2, 3])
    held = -(-len(prompt) // page)
    assert forked.pages() == {"used": held, "shared": held}
    assert [forked.pos(i) for i in range(4)] == [len(prompt)] * 4
    assert [plain.prefill(i, prompt) for i in range(4)] == [first] * 4
    rng = np.random.default_rng(page)
    nxt = [first] * 4
    for step in range(6):
        blocks = np.array([[t] + rng.integers(0, 600, 4).tolist() for t in nxt], np.uint32)
        if step == 2:  # perfect drafts now and then: different accepted counts
            blocks[1, 1:] = blocks[0, 1:]
        got, want = forked.verify(blocks), plain.verify(blocks)
        assert got == want, step
        assert [forked.pos(i) for i in range(4)] == [plain.pos(i) for i in range(4)]
        nxt = got[1]
        if step == 3:  # a fork of a fork, from the middle of a page; sequence 3's own pages go back
            n = forked.pos(1) - 3
            forked.fork(1, 3, n)
            plain.truncate(3, 0)
            hist = prompt + hist1[: n - len(prompt)] if n > len(prompt) else prompt[:n]
            plain.prefill(3, hist)
            nxt[3] = 7
        if step == 0:
            hist1 = []
        hist1 += [int(x) for x in blocks[1, : got[0][1] + 1]]
    # rolled back into the shared prompt: the pages are copied before they are written
    for i in (0, 2):
        forked.truncate(i, 11)
        plain.truncate(i, 11)
    blocks = np.array([[5, 6, 7, 8, 9]] * 4, np.uint32)
    assert forked.verify(blocks) == plain.verify(blocks)
    for i in range(4):
        forked.truncate(i, 0)
    assert forked.pages() == {"used": 0, "shared": 0}
    forked.close()
    plain.close()
    base.close()


def test_bad_forks_are_errors(tiny):
    m = ls.Model(tiny, max_ctx=64)
    b = ls.Batch(m, 3, max_ctx=40, max_block=3)
    b.prefill(0, [1, 2, 3])
    for src, dst, n in [(0, [0], 1), (0, [1, 1], 1), (0, [3], 1), (3, [0], 0), (0, [1], 4)]:
        with pytest.raises(ls.LayerstreamError) as e:
            b.fork(src, dst, n)
        assert e.value.code == -1
    assert b.pages() == {"used": 1, "shared": 0} and b.pos(1) == 0
    b.fork(0, 1, 0)
    assert b.pos(1) == 0
    b.close()


def margins(rows):
    top = np.partition(rows, -2, axis=1)[:, -2:]
    return top[:, 1] - top[:, 0]


@pytest.mark.parametrize("shape,prompt_len,B,M", [("0.5b", 300, 6, 4), ("0.5b", 700, 20, 9), ("3b-2l", 400, 5, 5)])
def test_a_shared_prefix_read_once_decodes_as_each_sequence_alone(shape, prompt_len, B, M):
    os.makedirs(ROOT, exist_ok=True)
    path = synth.ensure_lsq(ROOT, shape, 0, (4, 32), (4, 32), clip=True)
    rng = np.random.default_rng(prompt_len)
    prompt = rng.integers(0, 150000, prompt_len).tolist()
    model = ls.Model(path, max_ctx=prompt_len + 64)
    b = ls.Batch(model, B, max_ctx=prompt_len + 64, max_block=M)
    alone = ls.Model(path, max_ctx=prompt_len + 64)
    first = b.prefill(0, prompt)
    b.fork(0, range(1, B))
    alone.forward(prompt, want_logits=False)
    hist, nxt = [[] for _ in range(B)], [first] * B
    checked = skipped = 0
    for step in range(3):
        blocks = np.array([[t] + rng.integers(0, 150000, M - 1).tolist() for t in nxt], np.uint32)
        m, got = b.verify(blocks)
        assert b.pages()["shared"] == prompt_len // 64
        for i in range(B):
            alone.truncate(prompt_len)
            if hist[i]:
                alone.forward(hist[i], want_logits=False)
            rows = alone.forward_multi(blocks[i], M)
            am, mg = rows.argmax(1), margins(rows)
            k = 0
            while k < M - 1 and am[k] == blocks[i, k + 1]:
                k += 1
            if (mg[: k + 1] > TOL).all():
                checked += 1
                assert (m[i], got[i]) == (k, int(am[k])), (step, i)
            else:
                skipped += 1
            hist[i] += [int(x) for x in blocks[i, : m[i] + 1]]
            assert b.pos(i) == prompt_len + len(hist[i])
        nxt = got
    # (the first step's first row is the same in every sequence: one near tie there skips all of them)
    assert checked >= B
    b.close()
    alone.close()
    model.close()
