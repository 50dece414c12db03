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
