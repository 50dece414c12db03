"""Batch.fork and the passes over shared pages (needs a B200): what runs beside them and in which order, at the 0.5B widths."""

import os

import numpy as np
import pytest
import torch

import layerstream_b200 as ls
from layerstream_b200 import synth

pytestmark = pytest.mark.gpu

ROOT = os.environ.get("LS_BENCH_ROOT", "/tmp/ls_b200_bench")


@pytest.fixture(scope="module")
def model():
    os.makedirs(ROOT, exist_ok=True)
    m = ls.Model(synth.ensure_lsq(ROOT, "0.5b", 0, (4, 32), (4, 32), clip=True), max_ctx=64)
    yield m
    m.close()


def forked(model, B, M, n, seed=0, groups=1):
    """A batch whose sequences hold the same n positions (groups of them: one prompt each)."""
    rng = np.random.default_rng(seed)
    b = ls.Batch(model, B, max_ctx=n + 64, max_block=M)
    for g in range(groups):
        seqs = range(g * B // groups, (g + 1) * B // groups)
        b.prefill(seqs[0], rng.integers(0, 150000, n).tolist())
        b.fork(seqs[0], seqs[1:])
    return b, rng


def test_the_first_shared_pass_beside_a_busy_default_stream(model):
    B, M, n = 6, 4, 700
    results = []
    for busy in (False, True):
        b, rng = forked(model, B, M, n)
        a = torch.randn(4096, 4096, device="cuda", dtype=torch.bfloat16)
        torch.cuda.synchronize()
        if busy:
            for _ in range(100):  # about 10 ms on the legacy stream: a few passes
                a = torch.mm(a, a)
        results.append([b.verify(rng.integers(0, 150000, (B, M)).astype(np.uint32)) for _ in range(10)])
        torch.cuda.synchronize()
        b.close()
    assert results[0] == results[1]


def test_a_pass_that_failed_at_its_page_copies_is_made_again(model):
    B, M, n = 5, 4, 410  # not a whole page: four of the five sequences copy the last one
    results = []
    for fail in (False, True):
        b, rng = forked(model, B, M, n)
        blocks = rng.integers(0, 150000, (4, B, M)).astype(np.uint32)
        before = b.pages()
        for _ in range(2 * fail):
            b.inject_error(6)
            with pytest.raises(ls.LayerstreamError, match="test hook") as e:
                b.verify(blocks[0])
            assert e.value.code == -3 and b.pages() == before and [b.pos(i) for i in range(B)] == [n] * B
        got = [b.verify(x) for x in blocks]
        b.fork(0, 1, n)  # the prompt's rows are still whole in the pages that are shared
        b.truncate(0, n)
        results.append((got, b.verify(blocks[1]), b.pages()))
        b.close()
    assert results[0] == results[1]


def test_blocks_of_changing_length_read_the_prefix_once(model):
    # 32 rows of 7 heads fill tiles of their own and are planned alone, 5 rows are not
    B, n = 4, 520
    b, rng = forked(model, B, 32, n)
    assert b.shared_positions == 0  # prefilled by one sequence
    for M, shared in ((32, 0), (5, 512), (32, 0), (1, 512), (5, 512)):
        b.verify(rng.integers(0, 150000, (B, M)).astype(np.uint32))
        assert b.shared_positions == shared, M
    b.close()


def near_ties(rows):
    top = np.partition(rows, -2, axis=1)[:, -2:]
    return top[:, 1] - top[:, 0] <= 2e-2  # the bound of the framework's other token comparisons


@pytest.mark.parametrize("groups", [1, 2])
def test_shared_and_separate_reading_decode_alike(model, monkeypatch, groups):
    B, M, n = 6, 4, 700
    path = synth.ensure_lsq(ROOT, "0.5b", 0, (4, 32), (4, 32), clip=True)
    got = {}
    for shared in ("1", "0"):
        for graphs in ("1", "0"):
            monkeypatch.setenv("LS_SHARED", shared)
            monkeypatch.setenv("LS_BATCH_GRAPHS", graphs)
            b, rng = forked(model, B, M, n, seed=5, groups=groups)
            out = []
            for _ in range(3):
                blocks = rng.integers(0, 150000, (B, M)).astype(np.uint32)
                out.append((blocks, b.verify(blocks)))
                assert b.shared_positions == (groups * (n // 64 * 64) if shared == "1" else 0)
                for i in range(B):
                    b.truncate(i, n)  # every step behind the prompt alone, whatever was accepted
            got[shared, graphs] = out
            b.close()
    for shared in ("1", "0"):
        for (_, x), (_, y) in zip(got[shared, "1"], got[shared, "0"]):
            assert x == y  # a graph's replay is the eager pass
    alone = ls.Model(path, max_ctx=n + 64)
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, 150000, n).tolist() for _ in range(groups)]
    same = 0
    for g in range(groups):
        alone.truncate(0)
        alone.forward(prompts[g], want_logits=False)
        for (blocks, (m1, t1)), (_, (m0, t0)) in zip(got["1", "1"], got["0", "1"]):
            for i in range(g * B // groups, (g + 1) * B // groups):
                alone.truncate(n)
                rows = alone.forward_multi(blocks[i], M)
                k = 0
                while k < M - 1 and rows[k].argmax() == blocks[i, k + 1]:
                    k += 1
                if not near_ties(rows[: k + 1]).any():
                    same += 1
                    assert (m1[i], t1[i]) == (m0[i], t0[i]) == (k, int(rows[k].argmax())), i
    assert same >= 2 * B
    alone.close()
