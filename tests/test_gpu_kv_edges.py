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


@pytest.mark.parametrize("heads,kvh,hd,dtype,page,n,M", [
    (14, 2, 64, "f16", 64, 70, 1500),      # a long block: 83 tiles of one sequence, rows that see chunks of new rows alone
    (8, 1, 128, "bf16", 128, 1000, 700),
    (128, 1, 64, "f16", 16, 200, 3),       # a row's heads fill a tile, or more than one
    (200, 1, 128, "bf16", 32, 300, 2),
    (1024, 8, 64, "bf16", 64, 40, 1),
    (4, 1, 64, "f16", 65536, 3000, 2),     # the largest page
    (3, 3, 128, "bf16", 2048, 2047, 3),    # rows on both sides of a page's end
])
def test_sizes_at_the_ends_of_the_range(heads, kvh, hd, dtype, page, n, M):
    s = Setup(heads, kvh, hd, dtype, page, 2, M, n + M, seed=37)
    s.fill_fast(0, list(range(-(-n // page))), n)
    s.kv.fork(0, [1], n - n % 16)
    counts = [M, max(1, M // 3)]
    s.kv.begin(counts, M)
    s.kv.self_check()
    run_layer(s, 0, counts)


def test_pools_of_more_than_2_to_the_31_elements():
    # 19.2 million rows of 128: pages at both ends of the pools, in the second layer's half of them; copied pages too
    s = Setup(4, 1, 128, "f16", 64, 3, 2, 700, layers=2, seed=41, num_pages=150000)
    ids = [149999, 0, 149990, 75000, 149998, 1, 149997, 149996, 2, 149995]
    s.fill_fast(0, ids, 620)
    s.kv.fork(0, [1, 2], 600)
    s.kv.begin([2, 2, 1], 2)
    s.kv.self_check()
    assert s.kv.info.shared_positions == 576
    run_layer(s, 1, [2, 2, 1])
    s.kv.end()
    t, lens = s.kv.tables(), [s.kv.length(i) for i in range(3)]
    assert lens == [622, 602, 601]
    old = [s.k[:, :, t[i, : -(-lens[i] // 64)].tolist()].clone() for i in range(3)]
    moved = s.kv.compact()
    torch.cuda.synchronize()
    t = s.kv.tables()
    assert moved > 5 and t.max() == s.kv.info.pages_used - 1
    for i in range(3):
        new = s.k[:, :, t[i, : -(-lens[i] // 64)].tolist()]
        assert torch.equal(new.view(torch.int16), old[i].view(torch.int16))
    s.kv.begin([1, 1, 1], 2)
    run_layer(s, 1, [1, 1, 1])


def test_a_step_begun_on_one_stream_and_read_on_another():
    s = Setup(8, 2, 64, "f16", 32, 4, 2, 900, layers=2, seed=43)
    s.fill_fast(0, list(range(25)), 790)
    s.kv.fork(0, [1, 2, 3])
    qkv, outs = s.randn(8, s.W), []
    torch.cuda.synchronize()
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    for a, b in ((first, second), (second, first)) * 5:
        s.kv.begin([2, 2, 1, 2], 2, a.cuda_stream)
        b.wait_stream(a)
        out = torch.zeros(8, 8 * 64, device="cuda", dtype=s.dt)
        b.wait_stream(torch.cuda.current_stream())
        s.kv.attention(1, qkv.data_ptr(), out.data_ptr(), s.rope.data_ptr(), stream=b.cuda_stream)
        a.wait_stream(b)
        outs.append(out)  # the step is dropped: every turn begins the same one again
    torch.cuda.synchronize()
    s.kv.begin([2, 2, 1, 2], 2)
    want = run_layer(s, 1, [2, 2, 1, 2], qkv)
    rows = [0, 1, 2, 3, 4, 6, 7]
    for out in outs:
        assert torch.equal(out[rows], want[rows])


def test_page_copies_in_a_captured_graph():
    k, v = (torch.randn(2, 2, 12, 16, 64, device="cuda").half() for _ in range(2))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        ls.kv_copy_pages(k.data_ptr(), v.data_ptr(), 2, 2, 64, 16, 12, [0, 0, 3], [5, 6, 7], [16, 16, 3], st.cuda_stream)
    for _ in range(2):
        k.copy_(torch.randn(k.shape, device="cuda"))
        v.copy_(torch.randn(v.shape, device="cuda"))
        want = [x.clone() for x in (k, v)]
        for w in want:
            w[:, :, 5] = w[:, :, 6] = w[:, :, 0]
            w[:, :, 7, :3] = w[:, :, 3, :3]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])
