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
