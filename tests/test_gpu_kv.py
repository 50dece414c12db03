"""Attention over shared pages, forks, page copies and compaction of ls.KvCache (needs a B200).

Attention is compared with a float64 restatement of its definition (rotate, round k and v into the
pages, causal softmax(q . k / sqrt(hd)) v per sequence through its own page table, without any sharing).

Tolerance, with u = eps / 2 of the cache's type (2^-11 for f16, 2^-8 for bf16): the output is rounded
once (u |o|); each softmax weight is rounded once (u sum p|v|; in f16, weights below 2^-14 of the largest
are off by at most 2^-25 of it each); each rotated q component is rounded once, which moves a score by at most
d = u max_p sum_e |q_e k_pe| / sqrt(hd) and a normalised weight by at most a factor e^(2 d). The f32 steps
(sums over up to a few thousand positions, 2^x to 2^-22) are given 2^-14 of sum p|v|.
"""

import math

import numpy as np
import pytest
import torch

import layerstream_b200 as ls

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def rope_table(hd, positions):
    inv = 1e6 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return torch.stack([ang.cos(), ang.sin()], -1).float().cuda().contiguous()


def rotate64(x, cs):
    """x [rows, heads, hd], cs [rows, hd / 2, 2]."""
    a, b = x.chunk(2, -1)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


class Setup:
    """Pools with finite rows where sequences have positions and NaN everywhere else."""

    def __init__(self, heads, kvh, hd, dtype, page, seqs, M, max_ctx, layers=1, spare=3, seed=0, num_pages=None):
        self.g = torch.Generator("cuda").manual_seed(seed)
        self.heads, self.kvh, self.hd, self.dt, self.page, self.seqs, self.M = heads, kvh, hd, DT[dtype], page, seqs, M
        self.num_pages = num_pages or seqs * -(-max_ctx // page) + spare
        self.u = torch.finfo(self.dt).eps / 2
        self.k = torch.full((layers, kvh, self.num_pages, page, hd), math.nan, device="cuda", dtype=self.dt)
        self.v = self.k.clone()
        self.layers = layers
        self.kv = ls.KvCache(self.k.data_ptr(), self.v.data_ptr(), layers=layers, heads=heads, kv_heads=kvh, hd=hd, page=page,
                             num_pages=self.num_pages, seqs=seqs, max_ctx=max_ctx, max_rows=seqs * M, dtype=dtype)
        self.rope = rope_table(hd, max_ctx)
        self.W = (heads + 2 * kvh) * hd

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda").to(self.dt)

    def fill(self, seq, pages, n):
        """Sequence seq: these pages, n cached positions with values."""
        for p in range(n):
            a, b = int(pages[p // self.page]), p % self.page
            if torch.isnan(self.k[0, 0, a, b, 0]):
                self.k[:, :, a, b] = self.randn(self.layers, self.kvh, self.hd)
                self.v[:, :, a, b] = self.randn(self.layers, self.kvh, self.hd)
        self.kv.set_table(seq, pages, n)

    def fill_fast(self, seq, pages, n):
        full = torch.as_tensor(np.asarray(pages[: -(-n // self.page)], np.int64), device="cuda")
        k, v = self.randn(self.layers, self.kvh, len(full), self.page, self.hd), self.randn(self.layers, self.kvh, len(full), self.page, self.hd)
        if n % self.page:
            k[:, :, -1, n % self.page:] = math.nan
            v[:, :, -1, n % self.page:] = math.nan
        new = torch.isnan(self.k[0, 0, full, 0, 0]) if n else torch.zeros(0, dtype=torch.bool, device="cuda")
        self.k[:, :, full[new]] = k[:, :, new]
        self.v[:, :, full[new]] = v[:, :, new]
        self.kv.set_table(seq, pages, n)


def want_attention(s, layer, qkv, counts, lens, tables, rope, k_before, v_before):
    """(out, bound) in float64 of the valid rows, and the pools' expected contents; s.k / s.v hold what the call left."""
    H, kvh, hd, G = s.heads, s.kvh, s.hd, s.heads // s.kvh
    out, bound = {}, {}
    for i, (c, n) in enumerate(zip(counts, lens)):
        if c == 0:
            continue
        x = qkv[i * s.M: i * s.M + c, : s.W].double().view(c, H + 2 * kvh, hd)
        q, kn, vn = x[:, :H], x[:, H:H + kvh], x[:, H + kvh:]
        if rope is not None:
            cs = rope[n:n + c].double()
            mag = (kn.abs() + kn.roll(hd // 2, -1).abs())
            q, kn = rotate64(q, cs), rotate64(kn, cs)
        else:
            mag = torch.zeros_like(kn)
        at = torch.arange(n + c, device="cuda")
        pages = torch.as_tensor(tables[i].astype(np.int64), device="cuda")[at // s.page]
        K, V = s.k[layer][:, pages, at % s.page].double(), s.v[layer][:, pages, at % s.page].double()  # [kvh, n + c, hd]
        # the new rows were rounded into their pages
        fin = torch.isfinite(vn)
        assert torch.equal(V[:, n:].transpose(0, 1)[fin], vn[fin].to(s.dt).double())
        assert ((K[:, n:].transpose(0, 1) - kn).abs() <= s.u * kn.abs() * 1.001 + 2**-21 * mag + 1e-7).all()
        for t in range(c):
            e = n + t + 1
            qt = q[t].view(kvh, G, hd)
            sc = torch.einsum("gjd,gpd->gjp", qt, K[:, :e]) / math.sqrt(hd)
            p = torch.softmax(sc, -1)
            o = torch.einsum("gjp,gpd->gjd", p, V[:, :e])
            a = torch.einsum("gjp,gpd->gjd", p, V[:, :e].abs())
            d = s.u * (torch.einsum("gjd,gpd->gjp", qt.abs(), K[:, :e].abs()) / math.sqrt(hd)).amax(-1, keepdim=True)
            tiny = e * 2.0**-25 * V[:, :e].abs().amax(1, keepdim=True) if s.dt == torch.float16 else 0.0
            out[i, t] = o.reshape(-1)
            bound[i, t] = (s.u * o.abs() + (s.u + torch.expm1(2 * d) + 2**-14) * a + tiny + 1e-7).reshape(-1)
    return out, bound


def run_layer(s, layer, counts, qkv=None, rope=True, pad=0, out_pad=0, check=True):
    """One begun step through one layer, checked; returns out."""
    lens, tables = [s.kv.length(i) for i in range(s.seqs)], s.kv.tables()
    if qkv is None:
        qkv = s.randn(s.seqs * s.M, s.W + pad)
    out = torch.full((s.seqs * s.M, s.heads * s.hd + out_pad), 7.0, device="cuda", dtype=s.dt)
    kb, vb = s.k.clone(), s.v.clone()
    st = torch.cuda.current_stream().cuda_stream
    s.kv.attention(layer, qkv.data_ptr(), out.data_ptr(), s.rope.data_ptr() if rope else 0, qkv.stride(0), out.stride(0), stream=st)
    torch.cuda.synchronize()
    if not check:
        return out
    want, bound = want_attention(s, layer, qkv, counts, lens, tables, s.rope if rope else None, kb, vb)
    for (i, t), w in want.items():
        got = out[i * s.M + t, : s.heads * s.hd].double()
        over = (got - w).abs() / bound[i, t]
        assert torch.isfinite(got).all() and over.max() <= 1, (i, t, float(over.max()), float((got - w).abs().max()))
    # nothing else was written: rows past each count, the row padding, other positions and pages
    valid = torch.zeros(s.seqs * s.M, dtype=torch.bool, device="cuda")
    for i, c in enumerate(counts):
        valid[i * s.M: i * s.M + c] = True
    assert (out[~valid] == 7).all() and (out[:, s.heads * s.hd:] == 7).all()
    new = torch.zeros(s.num_pages, s.page, dtype=torch.bool, device="cuda")
    for i, (c, n) in enumerate(zip(counts, lens)):
        for p in range(n, n + c):
            new[int(tables[i][p // s.page]), p % s.page] = True
    for pool, before in ((s.k, kb), (s.v, vb)):
        same = (pool.view(torch.int16) == before.view(torch.int16)).all(-1)  # [layers, kvh, pages, page]
        same[layer] |= new
        assert same.all()
    return out


CASES = [
    # heads kvh hd dtype page groups seqs M prefix tail ragged
    (14, 2, 64, "f16", 64, 1, 2, 1, 128, 40, False),
    (14, 2, 64, "f16", 64, 1, 5, 9, 512, 100, False),
    (16, 2, 128, "bf16", 64, 1, 4, 5, 640, 200, False),
    (16, 2, 128, "f16", 256, 2, 6, 3, 512, 300, True),
    (6, 2, 64, "bf16", 8, 2, 7, 5, 1000, 77, True),
    (8, 8, 128, "f16", 16, 1, 3, 1, 304, 1, False),   # one q head per kv head, tails of zero or one position
    (5, 1, 128, "bf16", 128, 1, 9, 2, 256, 129, True),
    (24, 1, 64, "f16", 32, 1, 3, 33, 320, 60, False),  # tiles across many rows of one sequence
    (4, 4, 64, "f16", 8, 1, 2, 70, 256, 9, False),     # blocks longer than a chunk boundary
    (14, 2, 64, "f16", 64, 3, 24, 1, 256, 64, False),
    (32, 8, 128, "bf16", 64, 1, 20, 2, 1536, 30, True),
    (14, 2, 64, "bf16", 64, 1, 40, 9, 256, 20, False),  # several pairs of tiles over one prefix
    (2, 2, 64, "f16", 512, 1, 3, 4, 1024, 700, False),
]


@pytest.mark.parametrize("heads,kvh,hd,dtype,page,groups,seqs,M,prefix,tail,ragged", CASES)
def test_attention_matches_the_definition(heads, kvh, hd, dtype, page, groups, seqs, M, prefix, tail, ragged):
    rng = np.random.default_rng(prefix + seqs + M)
    s = Setup(heads, kvh, hd, dtype, page, seqs, M, prefix + tail + M, seed=seqs * M)
    ids = rng.permutation(s.num_pages)
    shared = prefix // page
    at = groups * shared
    lens = []
    for i in range(seqs):
        n = prefix + int(rng.integers(0, tail + 1))
        own = -(-(n + M) // page) - shared
        g = i * groups // seqs
        s.fill_fast(i, list(ids[g * shared:(g + 1) * shared]) + list(ids[at:at + own]), n)
        at += own
        lens.append(n)
    counts = rng.integers(0, M + 1, seqs).tolist() if ragged else [M] * seqs
    counts[-1] = M
    s.kv.begin(counts, M)
    s.kv.self_check()
    live = {i * groups // seqs for i in range(seqs) if counts[i]}
    many = [g for g in live if sum(1 for i in range(seqs) if counts[i] and i * groups // seqs == g) > 1]
    if prefix >= 256:
        assert s.kv.info.shared_positions == prefix * len(many)  # the shared path is what runs
    run_layer(s, 0, counts, rope=seqs % 2 == 0)


@pytest.mark.parametrize("hd,dtype", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("n,M", [(0, 1), (0, 5), (1, 1), (7, 1), (8, 3), (127, 1), (127, 2), (128, 1), (129, 40), (255, 130)])
def test_short_contexts(hd, dtype, n, M):
    s = Setup(6, 2, hd, dtype, 8, 2, M, n + M, seed=n + M)
    s.fill_fast(0, list(range(-(-n // 8))), n)
    s.fill_fast(1, list(range(-(-n // 8), -(-n // 8) + -(-(n // 2) // 8))), n // 2)
    s.kv.begin([M, max(1, M // 2)], M)
    run_layer(s, 0, [M, max(1, M // 2)])


def test_rows_that_nobody_has_may_hold_anything():
    # (the pools of every test are NaN outside the sequences) here: infinities, and a step of no rows
    s = Setup(4, 2, 64, "f16", 16, 3, 2, 100)
    s.k.fill_(math.inf)
    s.v.fill_(-math.inf)
    s.k[:, :, :5], s.v[:, :, :5] = s.randn(1, 2, 5, 16, 64), s.randn(1, 2, 5, 16, 64)
    s.k[:, :, 4, 6:] = math.inf
    s.v[:, :, 4, 6:] = math.inf
    s.kv.set_table(0, [0, 1, 2, 3, 4], 70)
    s.kv.fork(0, [1, 2])
    s.kv.begin([2, 0, 1], 2)
    run_layer(s, 0, [2, 0, 1])
    s.kv.begin([0, 0, 0], 2)
    run_layer(s, 0, [0, 0, 0])


@pytest.mark.parametrize("hd,dtype,n,M", [(64, "f16", 100, 6), (128, "bf16", 125, 9), (64, "bf16", 0, 4), (128, "f16", 10, 130)])
def test_infinities_in_a_new_row_reach_only_the_rows_that_see_it(hd, dtype, n, M):
    s = Setup(4, 2, hd, dtype, 16, 2, M, n + M, seed=3)
    s.fill_fast(0, list(range(-(-n // 16))), n)
    s.fill_fast(1, list(range(-(-n // 16), 2 * -(-n // 16))), n)
    s.kv.begin([M, M], M)
    qkv = s.randn(2 * M, s.W)
    clean = run_layer(s, 0, [M, M], qkv)
    bad = qkv.clone()
    t0, kv_head, H = M // 2, 1, 4 * hd
    vcol = H + 2 * hd + kv_head * hd
    bad[t0, vcol + 3] = math.inf
    bad[t0, vcol + 5] = math.nan
    bad[M - 1, vcol + 7] = -math.inf
    bad[t0, H + 0 * hd + 1] = math.nan  # a key of the other kv head
    got = run_layer(s, 0, [M, M], bad, check=False).view(2, M, 4, hd)
    ref = clean.view(2, M, 4, hd)
    assert torch.equal(got[1], ref[1])  # the other sequence
    assert torch.equal(got[0, :t0], ref[0, :t0])  # the rows before it
    seen = got[0, t0:, 2:]  # q heads of kv head 1
    assert (seen[..., 3] == math.inf).all() and torch.isnan(seen[..., 5]).all()
    assert (seen[-1, :, 7] == -math.inf).all() and torch.isfinite(seen[:-1, :, 7]).all()
    rest = [d for d in range(hd) if d not in (3, 5, 7)]
    assert torch.equal(seen[..., rest], ref[0, t0:, 2:][..., rest])
    assert torch.isnan(got[0, t0:, :2]).all()  # the NaN key: every later row of its heads


def test_large_scores_move_the_maximum():
    # keys whose scores grow along the context, so that the running maximum keeps rising, and fall
    for sign in (1.0, -1.0):
        s = Setup(4, 2, 64, "bf16", 64, 3, 2, 1300, seed=9)
        n = 1200
        s.fill_fast(0, list(range(-(-n // 64) + 1)), n)
        ramp = torch.linspace(0.05, 6.0, 19 * 64, device="cuda").view(1, 1, 19, 64, 1)
        s.k[:, :, :19] = (s.k[:, :, :19].float() * (ramp if sign > 0 else ramp.flip(2, 3))).to(s.dt)
        s.kv.fork(0, [1, 2], 1152)
        s.kv.begin([2, 2, 2], 2)
        run_layer(s, 0, [2, 2, 2])


def test_strides_streams_and_repeated_calls():
    s = Setup(6, 2, 64, "f16", 32, 5, 3, 400, seed=4)
    s.fill_fast(0, list(range(10)), 300)
    s.kv.fork(0, [1, 2, 3, 4])
    qkv = s.randn(15, s.W + 24)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.kv.begin([3, 3, 3, 3, 3], 3, side.cuda_stream)
        a = run_layer(s, 0, [3] * 5, qkv, out_pad=16)
        b = run_layer(s, 0, [3] * 5, qkv, out_pad=16)
    assert torch.equal(a, b)


def test_a_captured_layer_replays_over_later_steps():
    s = Setup(6, 2, 64, "f16", 16, 4, 2, 400, layers=2, seed=5)
    s.fill_fast(0, list(range(12)), 190)
    s.kv.fork(0, [1, 2, 3])
    qkv, out = s.randn(8, s.W), torch.zeros(8, 6 * 64, device="cuda", dtype=s.dt)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        s.kv.begin([2, 2, 2, 2], 2, st.cuda_stream)
        s.kv.attention(1, qkv.data_ptr(), out.data_ptr(), s.rope.data_ptr(), stream=st.cuda_stream)
        st.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            s.kv.attention(1, qkv.data_ptr(), out.data_ptr(), s.rope.data_ptr(), stream=st.cuda_stream)
            with pytest.raises(ls.LayerstreamError, match="captured"):
                s.kv.begin([1, 1, 1, 1], 2, st.cuda_stream)
            with pytest.raises(ls.LayerstreamError, match="captured"):
                s.kv.compact(st.cuda_stream)
        for step, counts in enumerate([[2, 2, 2, 2], [1, 2, 0, 2], [2, 1, 2, 0], [2, 2, 2, 2]]):
            qkv.copy_(s.randn(8, s.W))
            s.kv.begin(counts, 2, st.cuda_stream)
            s.kv.self_check()
            graph.replay()
            st.synchronize()
            replayed = out.clone()
            direct = run_layer(s, 1, counts, qkv)
            for i, c in enumerate(counts):
                assert torch.equal(replayed[2 * i:2 * i + c], direct[2 * i:2 * i + c]), step
            s.kv.end(counts if step % 2 else [min(c, 1) for c in counts])


def test_forks_steps_rollbacks_and_compaction_together():
    """Decode under forks: every sequence's attention equals the definition over its own history, in every
    layer, while pages are shared, copied on write, returned, reused and moved."""
    rng = np.random.default_rng(8)
    layers, seqs, M = 3, 6, 4
    s = Setup(4, 2, 64, "f16", 16, seqs, M, 500, layers=layers, seed=6)
    hist = [[torch.zeros(0, 2, 64, dtype=torch.double, device="cuda")] * (2 * layers) for _ in range(seqs)]  # K, V rows by layer

    def check_history():
        t = s.kv.tables()
        for i in range(seqs):
            n = s.kv.length(i)
            at = torch.arange(n, device="cuda")
            pg = torch.as_tensor(t[i].astype(np.int64), device="cuda")[at // 16]
            for l in range(layers):
                assert torch.equal(s.k[l][:, pg, at % 16].double().transpose(0, 1), hist[i][2 * l])
                assert torch.equal(s.v[l][:, pg, at % 16].double().transpose(0, 1), hist[i][2 * l + 1])

    def step(counts, keep):
        s.kv.begin(counts, M)
        s.kv.self_check()
        t = s.kv.tables()
        for l in range(layers):
            run_layer(s, l, counts)
            for i, c in enumerate(counts):
                n = s.kv.length(i)
                at = torch.arange(n, n + c, device="cuda")
                pg = torch.as_tensor(t[i].astype(np.int64), device="cuda")[at // 16]
                for j, pool in enumerate((s.k, s.v)):
                    hist[i][2 * l + j] = torch.cat([hist[i][2 * l + j], pool[l][:, pg, at % 16].double().transpose(0, 1)[: keep[i]]])
        s.kv.end(keep)

    for _ in range(45):  # sequence 0's prompt
        step([M] + [0] * 5, [M] + [0] * 5)
    s.kv.fork(0, range(1, 5))
    for i in range(1, 5):
        hist[i] = list(hist[0])
    check_history()
    for r in range(5):
        counts = [int(c) for c in rng.integers(0, M + 1, seqs)]
        step(counts, [int(rng.integers(0, c + 1)) for c in counts])
        check_history()
    s.kv.truncate(2, 100)
    hist[2] = [h[:100] for h in hist[2]]
    s.kv.fork(2, [5], 97)
    hist[5] = [h[:97] for h in hist[2]]
    s.kv.fork(3, [1])
    hist[1] = list(hist[3])
    before = s.kv.tables()
    moved = s.kv.compact(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert moved > 0 and s.kv.tables().max() == s.kv.info.pages_used - 1 < before.max()
    check_history()
    for r in range(3):
        step([M] * seqs, [int(k) for k in rng.integers(0, M + 1, seqs)])
        check_history()


@pytest.mark.parametrize("layers,kvh,hd,page,num_pages,n,partial", [(3, 2, 64, 64, 40, 6, True), (2, 2, 64, 64, 40, 20, False),
                                                                  (1, 3, 72, 8, 5000, 2400, True), (2, 1, 8, 16, 9, 1, False),
                                                                  (1, 2, 128, 256, 20, 10, True), (1, 1, 128, 4096, 3, 1, True)])
def test_copy_pages(layers, kvh, hd, page, num_pages, n, partial):
    rng = np.random.default_rng(n)
    g = torch.Generator("cuda").manual_seed(n)
    k, v = (torch.randint(-2**15, 2**15, (layers, kvh, num_pages, page, hd), generator=g, device="cuda", dtype=torch.int16) for _ in range(2))
    ids = rng.permutation(num_pages)
    src, dst = ids[:n].copy(), ids[n:2 * n]
    src[n // 2:] = src[: n - n // 2]  # sources repeat
    rows = rng.integers(0, page + 1, n) if partial else np.full(n, page)
    wk, wv = k.clone(), v.clone()
    for a, b, r in zip(src, dst, rows):
        wk[:, :, b, :r] = k[:, :, a, :r]
        wv[:, :, b, :r] = v[:, :, a, :r]
    ls.kv_copy_pages(k.data_ptr(), v.data_ptr(), layers, kvh, hd, page, num_pages, src, dst, rows if partial else None,
                     torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_refusals_with_a_gpu():
    s = Setup(4, 2, 64, "f16", 16, 2, 2, 64)
    qkv, out = s.randn(4, s.W + 8), torch.zeros(4, 256 + 8, device="cuda", dtype=s.dt)

    def refused(match, layer=0, q=qkv.data_ptr(), o=out.data_ptr(), rope=0, qs=0, os_=0):
        with pytest.raises(ls.LayerstreamError, match=match) as e:
            s.kv.attention(layer, q, o, rope, qs, os_)
        assert e.value.code == -1

    refused("no step")
    s.kv.begin([1, 1], 2)
    refused("outside the cache", layer=1)
    refused("NULL", q=0)
    refused("NULL", o=0)
    refused("qkv must be 16-byte", q=qkv.data_ptr() + 2)
    refused("out must be 16-byte", o=out.data_ptr() + 8)
    refused("rope must be 16-byte", rope=s.rope.data_ptr() + 4)
    refused("strides", qs=s.W - 8)
    refused("strides", qs=s.W + 4)
    refused("strides", os_=248)
    refused("strides", os_=260)
    s.kv.end([0, 0])
    refused("no step")
    host = np.zeros(1 << 16, np.uint16)
    with pytest.raises(ls.LayerstreamError, match="device memory"):
        ls.KvCache(host.ctypes.data & ~15, s.v.data_ptr(), layers=1, heads=4, kv_heads=2, hd=64, page=16, num_pages=4, seqs=1, max_ctx=64,
                   max_rows=4)
    with pytest.raises(ls.LayerstreamError, match="device memory"):
        ls.kv_copy_pages(host.ctypes.data & ~15, s.v.data_ptr(), 1, 2, 64, 16, 4, [0], [1])


@pytest.mark.parametrize("heads,kvh,hd,dtype,seqs,M,prefix,tail", [
    (2, 1, 64, "f16", 1, 1, 40000, 0),     # one row over all CTAs: the join's four warps hold more than 32 partials each
    (2, 1, 128, "bf16", 1, 3, 20000, 0),
    (15, 1, 64, "bf16", 4, 20, 33000, 30),  # many rows of few tiles: one warp joins about 30 partials
])
def test_long_contexts(heads, kvh, hd, dtype, seqs, M, prefix, tail):
    s = Setup(heads, kvh, hd, dtype, 64, seqs, M, prefix + tail * seqs + M, seed=11)
    shared = list(range(prefix // 64))
    at = len(shared)
    for i in range(seqs):
        n = prefix // 64 * 64 + tail * (i + 1)
        own = -(-n // 64) - len(shared)
        s.fill_fast(i, shared + list(range(at, at + own)), n)
        at += own
    s.kv.begin([M] * seqs, M)
    run_layer(s, 0, [M] * seqs)


@pytest.mark.parametrize("hd,dtype,n", [(64, "f16", 500), (128, "bf16", 700), (128, "f16", 1000)])
def test_a_row_does_not_depend_on_its_neighbours(hd, dtype, n):
    # NaN, and scores that outgrow the running maximum, in one row of a tile: the others keep every bit
    M = 8
    s = Setup(8, 2, hd, dtype, 32, 2, M, n + M, seed=5)
    pages = list(range(-(-n // 32)))
    s.fill_fast(0, pages, n)
    s.kv.fork(0, [1])
    s.kv.begin([M, M], M)
    qkv = s.randn(2 * M, s.W)
    clean = run_layer(s, 0, [M, M], qkv, check=False).view(2, M, 8, hd)
    big = qkv.clone()
    big[2, : 8 * hd] *= 30
    big[M + 5, hd: 2 * hd] = math.nan
    got = run_layer(s, 0, [M, M], big, check=False).view(2, M, 8, hd)
    assert torch.isnan(got[1, 5, 1]).all()
    same = torch.ones(2, M, 8, dtype=torch.bool, device="cuda")
    same[0, 2] = False
    same[1, 5, 1] = False
    assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize("hd,dtype", [(64, "f16"), (128, "bf16")])
def test_an_infinite_key(hd, dtype):
    # its score is +inf for the rows that are NaN by the definition too, -inf (weight 0) for the others
    s = Setup(4, 2, hd, dtype, 16, 2, 2, 330, seed=9)
    s.fill_fast(0, list(range(20)), 300)
    s.k[0, 0, 3, 5, 7] = math.inf
    s.kv.fork(0, [1])
    s.kv.begin([2, 2], 2)
    lens, tables = [300, 300], s.kv.tables()
    qkv = s.randn(4, s.W)
    got = run_layer(s, 0, [2, 2], qkv, rope=False, check=False)
    qz = qkv.view(4, -1, hd)[:, :2, 7].float()  # kv head 0's q heads: sign of q . k
    nan = qz > 0
    out = got.view(4, 4, hd)
    assert torch.isnan(out[:, :2][nan]).all() and torch.isfinite(out[:, 2:]).all() and torch.isfinite(out[:, :2][~nan]).all()
    at = torch.arange(302, device="cuda")
    for i in range(2):
        pg = torch.as_tensor(tables[i].astype(np.int64), device="cuda")[at // 16]
        K, V = s.k[0][0, pg, at % 16].double(), s.v[0][0, pg, at % 16].double()
        for t in range(2):
            e = lens[i] + t + 1
            seen = torch.ones(e, dtype=torch.bool, device="cuda")
            seen[3 * 16 + 5] = False
            for j in range(2):
                if nan[2 * i + t, j]:
                    continue
                q = qkv[2 * i + t].view(-1, hd)[j].double()
                p = torch.softmax(K[:e][seen] @ q / math.sqrt(hd), 0)
                o, a = p @ V[:e][seen], p @ V[:e][seen].abs()
                d = s.u * ((K[:e][seen].abs() @ q.abs()) / math.sqrt(hd)).max()
                tiny = e * 2.0**-25 * V[:e].abs().amax() if s.dt == torch.float16 else 0.0
                assert ((out[2 * i + t, j].double() - o).abs() <= s.u * o.abs() + (s.u + torch.expm1(2 * d) + 2**-14) * a + tiny + 1e-7).all()


def test_two_caches_on_two_streams():
    setups = [Setup(8, 2, 64, "f16", 16, 4, 3, 900, seed=21), Setup(4, 2, 128, "bf16", 32, 6, 2, 1500, seed=22)]
    streams, qkvs, alone = [torch.cuda.Stream() for _ in setups], [], []
    for s, n in zip(setups, (800, 1400)):
        s.fill_fast(0, list(range(-(-n // s.page))), n)
        s.kv.fork(0, range(1, s.seqs))
        s.kv.begin([s.M] * s.seqs, s.M)
        qkvs.append(s.randn(s.seqs * s.M, s.W))
        alone.append(run_layer(s, 0, [s.M] * s.seqs, qkvs[-1]))
    outs = [torch.zeros_like(a) for a in alone]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, st, q, o in zip(setups, streams, qkvs, outs):
            s.kv.attention(0, q.data_ptr(), o.data_ptr(), s.rope.data_ptr(), stream=st.cuda_stream)
    torch.cuda.synchronize()
    for a, o in zip(alone, outs):
        assert torch.equal(a, o)
