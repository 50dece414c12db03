"""Attention over shared pages at its edges (needs a B200): what a row must not see, plans of more levels and segments, and
calls in orders that the other tests do not make. Tolerances are those of test_gpu_kv.py."""

import math

import pytest
import torch

import layerstream_b200 as ls
from test_gpu_kv import Setup, run_layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,dtype,n,M", [(64, "f16", 100, 6), (128, "bf16", 125, 9), (64, "bf16", 0, 40), (128, "bf16", 10, 130)])
def test_the_largest_values_in_new_rows_reach_only_the_rows_that_see_them(hd, dtype, n, M):
    s = Setup(4, 2, hd, dtype, 16, 2, M, n + M, seed=3)
    s.fill_fast(0, list(range(-(-n // 16))), n)
    s.fill_fast(1, list(range(-(-n // 16), 2 * -(-n // 16))), n)
    s.kv.begin([M, M], M)
    qkv = s.randn(2 * M, s.W)
    ref = run_layer(s, 0, [M, M], qkv).view(2, M, 4, hd)
    big = torch.finfo(s.dt).max
    v = (4 + 2) * hd
    for t0 in (M // 2, M - 1):  # every row from t0 on, in some columns of both kv heads
        bad = qkv.clone()
        bad[t0:M, v + 3] = big
        bad[t0:M, v + hd + 5] = -big
        got = run_layer(s, 0, [M, M], bad, check=False).view(2, M, 4, hd)
        assert torch.equal(got[1], ref[1])
        assert torch.equal(got[0, :t0], ref[0, :t0]), t0


@pytest.mark.parametrize("hd,dtype", [(64, "f16"), (64, "bf16"), (128, "bf16")])
def test_a_weight_of_zero_takes_nothing_from_the_largest_value(hd, dtype):
    # eight neighbouring keys whose scores are 2 hd below zero: their weights are zero in 32 bits
    s = Setup(4, 2, hd, dtype, 16, 3, 2, 330, seed=9)
    s.fill_fast(0, list(range(20)), 300)
    s.k[0, :, 3, 4:12] = -2 * math.sqrt(hd)
    s.kv.fork(0, [1, 2])
    s.kv.begin([2, 2, 2], 2)
    qkv = s.randn(6, s.W)
    qkv[:, : 4 * hd] = 1
    s.v[0, :, 3, 4:12] = 0
    ref = run_layer(s, 0, [2, 2, 2], qkv, rope=False, check=False)
    s.v[0, :, 3, 4:12] = torch.finfo(s.dt).max
    got = run_layer(s, 0, [2, 2, 2], qkv, rope=False, check=False)
    assert torch.isfinite(ref).all() and torch.equal(got, ref)


def test_steps_without_rows_between_steps_with_rows():
    # queued without a wait: the rows that an empty step's kernels find are never those of the step behind it
    pools = []
    for empty in (False, True):
        s = Setup(8, 2, 64, "f16", 16, 4, 3, 700, layers=2, seed=13)
        s.fill_fast(0, list(range(20)), 310)
        s.kv.fork(0, [1, 2, 3])
        qkv, other, out = s.randn(100, 12, s.W), s.randn(12, s.W), torch.zeros(12, 8 * 64, device="cuda", dtype=s.dt)
        torch.cuda.synchronize()
        outs = []
        for i in range(100):
            if empty:
                s.kv.begin([0, 0, 0, 0], 3)
                for layer in (0, 1):
                    s.kv.attention(layer, other.data_ptr(), out.data_ptr(), s.rope.data_ptr())
            s.kv.begin([3, 2, 0, 1], 3)
            for layer in (0, 1):
                s.kv.attention(layer, qkv[i].data_ptr(), out.data_ptr(), s.rope.data_ptr())
            outs.append(out.clone())
            s.kv.end([1, 2, 0, 1])
        torch.cuda.synchronize()
        pools.append([torch.stack(outs), s.k.view(torch.int16), s.v.view(torch.int16)])
    for a, b in zip(*pools):
        assert torch.equal(a, b)


@pytest.mark.parametrize("heads,hd,dtype", [(14, 64, "f16"), (16, 128, "bf16")])
def test_prompts_continued_under_a_shared_prompt_then_single_rows(heads, hd, dtype):
    # blocks that are planned by themselves, then steps that read the prefix once, and back
    s = Setup(heads, 2, hd, dtype, 64, 4, 128, 1400, seed=17)
    s.fill_fast(0, list(range(16)), 1000)
    s.kv.fork(0, [1, 2, 3])
    for counts, shared in (([128] * 4, 0), ([1] * 4, 960), ([2, 1, 2, 1], 960), ([128, 1, 128, 1], 960), ([128] * 4, 0), ([1] * 4, 960)):
        s.kv.begin(counts, 128)
        s.kv.self_check()
        assert s.kv.info.shared_positions == shared, counts
        run_layer(s, 0, counts)
        s.kv.end()


def test_a_begin_that_failed_is_made_again_with_its_copies():
    s = Setup(4, 2, 64, "f16", 16, 4, 3, 400, layers=2, seed=19)
    s.fill_fast(0, list(range(20)), 309)  # the last page is shared in part: three of the four holders copy it
    s.kv.fork(0, [1, 2, 3])
    before = s.kv.tables()
    for _ in range(2):
        s.kv.inject_error()
        with pytest.raises(ls.LayerstreamError, match="test hook") as e:
            s.kv.begin([3, 1, 2, 3], 3)
        assert e.value.code == -3 and (s.kv.tables() == before).all()
    s.kv.begin([3, 1, 2, 3], 3)
    s.kv.self_check()
    for layer in (0, 1):
        run_layer(s, layer, [3, 1, 2, 3])
    s.kv.end()


@pytest.mark.parametrize("heads,kvh,hd,dtype,M", [(14, 2, 64, "f16", 1), (16, 2, 128, "bf16", 5), (8, 2, 128, "f16", 9), (6, 2, 64, "bf16", 3)])
def test_prompts_under_a_system_prompt_are_two_shared_levels(heads, kvh, hd, dtype, M):
    # 512 positions of all nine sequences, then 640 and 768 of four each; the ninth has only the first range
    s = Setup(heads, kvh, hd, dtype, 64, 9, M, 1600, seed=23)
    s.fill_fast(0, list(range(22)), 512 + 640 + 70)
    s.fill_fast(4, list(range(8)) + list(range(30, 45)), 512 + 768 + 5)
    s.fill_fast(8, list(range(8)) + [60, 61], 512 + 33)
    s.kv.fork(0, [1, 2, 3], 512 + 640 + 9)
    s.kv.fork(4, [5, 6, 7])
    for counts in ([M] * 9, [M, 0, 1, M, 0, M, M, 1, M], [M] * 9):
        s.kv.begin(counts, M)
        s.kv.self_check()
        assert s.kv.info.shared_positions == 512 + 640 + 768
        run_layer(s, 0, counts)
        s.kv.end()


def test_more_segments_than_a_lane_keeps_near():
    # 700 sequences x 16 kv heads, each with a tile of its own: 11200 segments on the 296 lanes of 148 SMs, more than 32
    # on some lane whatever the split
    s = Setup(16, 16, 64, "f16", 16, 700, 1, 64, seed=29, num_pages=2810)
    for i in range(700):
        s.fill_fast(i, [0, 1, 2 + 4 * i, 3 + 4 * i], 32 + i % 31)
    s.kv.begin([1] * 700, 1)
    s.kv.self_check()
    assert s.kv.info.shared_positions == 32
    run_layer(s, 0, [1] * 700)


def test_after_a_wait_ran_out_a_new_cache_goes_on_over_the_same_pools():
    args = (4, 2, 64, "f16", 16, 3, 2, 400)
    s = Setup(*args, seed=31)
    s.fill_fast(0, list(range(20)), 300)
    s.kv.fork(0, [1, 2])
    s.kv.begin([2, 1, 2], 2)
    run_layer(s, 0, [2, 1, 2])
    s.kv.end()
    s.kv.begin([1, 1, 1], 2)
    s.kv.inject_error(2)
    x = s.randn(6, s.W)
    for _ in range(2):
        for call in (lambda: s.kv.begin([1, 1, 1], 2), lambda: s.kv.attention(0, x.data_ptr(), x.data_ptr()), s.kv.compact):
            with pytest.raises(ls.LayerstreamError, match="bounded wait") as e:
                call()
            assert e.value.code == -4
    s.kv.truncate(1, 300)
    lens, tables = [s.kv.length(i) for i in range(3)], s.kv.tables()
    assert lens == [302, 300, 302]
    s.kv.close()
    s.kv = ls.KvCache(s.k.data_ptr(), s.v.data_ptr(), layers=1, heads=4, kv_heads=2, hd=64, page=16, num_pages=s.num_pages, seqs=3,
                      max_ctx=400, max_rows=6, dtype="f16")
    for i, n in enumerate(lens):
        s.kv.set_table(i, tables[i][: -(-n // 16)], n)
    s.kv.begin([2, 2, 0], 2)
    s.kv.self_check()
    run_layer(s, 0, [2, 2, 0])
