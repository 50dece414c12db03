// Attention over a paged K/V cache whose sequences share pages, and copies of its pages.
//
// One layer's call is three launches:
//
//   kv_prep_kernel   the block's rows: q rotated and rounded into the query operand, k rotated and v
//                    rounded into their pages
//   kv_attn_kernel   one CTA per SM works its program of segments (ls_kv.h): for a tile of 128 query
//                    rows and a run of 128-position chunks
//                        S = Q K^T            tcgen05, Q and K in shared memory (128-byte swizzle)
//                        P = 2^(S c - m)      one query row per thread, c = log2(e) / sqrt(hd), f32
//                        O += P V             tcgen05, P in tensor memory, V as the pages hold it
//                    and leaves (m, l, O). A prefix shared by several sequences is a segment over the
//                    rows of all of them, so its K/V are read once for up to 256 rows (two tiles)
//                    instead of once per sequence.
//   kv_merge_kernel  per query row: O = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i over its partials
//
// Warp roles of kv_attn_kernel: two softmax warpgroups (one per lane of the CTA), one MMA issuer warp
// per lane, one TMA producer warp. O stays in tensor memory and is rescaled only when a row's maximum
// has grown by more than 2^8 over the one its exponents are taken against.
//
// Rounding: q (after rotation) and P enter the tensor core in the cache's 16-bit type, the type that
// its operands K and V have; scores, maxima, sums, O and the partials stay f32; the output is rounded
// once. Infinities and NaN in V rows that only some of a tile's rows may see (the block's own rows)
// are replaced by zeros for the MMA, since 0 x inf would reach the rows that do not see them, and the
// merge adds them back to the rows that do.
#include <cuda_bf16.h>

#include <algorithm>

#include "layerstream.h"
#include "ls_device.cuh"
#include "ls_kv.h"

namespace ls {

constexpr int KV_THREADS = 352;  // 2 softmax warpgroups, 2 issuer warps, 1 producer warp
constexpr float KV_RESCALE = 8.0f;  // log2 growth of a row's maximum that O is rescaled for

template <int HD>
struct KvSmem {
  static constexpr int kTile = 128 * HD * 2;      // Q tile, K chunk, V chunk
  static constexpr int kStages = HD == 64 ? 4 : 2;  // of K and of V, even: in the lanes' own phase lane t owns those of parity t
  static constexpr int kQ = 0, kK = 2 * kTile, kV = kK + kStages * kTile;
  static constexpr int kTotal = kV + kStages * kTile + 1024;  // + alignment
};

// ---- small device helpers -----------------------------------------------------------------------

__device__ __forceinline__ float kv_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool BF16>
__device__ __forceinline__ uint32_t kv_pack(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <bool BF16>
__device__ __forceinline__ float2 kv_unpack(uint32_t v) {
  if constexpr (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  const __half2 h = *reinterpret_cast<const __half2*>(&v);
  return __half22float2(h);
}
// Mask of the halves of v that are infinities or NaN (all exponent bits set).
template <bool BF16>
__device__ __forceinline__ uint32_t kv_nonfinite(uint32_t v) {
  constexpr uint32_t E = BF16 ? 0x7F80u : 0x7C00u;
  uint32_t m = 0;
  if ((v & E) == E) m |= 0x0000FFFFu;
  if ((v & (E << 16)) == (E << 16)) m |= 0xFFFF0000u;
  return m;
}
__device__ __forceinline__ void kv_ld32(uint32_t taddr, float* f) {
  uint32_t* v = reinterpret_cast<uint32_t*>(f);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
      "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
        "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
        "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void kv_tma2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(tc::su32(bar))
      : "memory");
}
// Shared-memory matrix descriptor of a 128-byte-swizzled tile: 8-row groups 1024 bytes apart; lbo = bytes
// between 64-element blocks of the contiguous dimension when that is the operand's M or N.
__device__ __forceinline__ uint64_t kv_sdesc(uint32_t saddr, uint32_t lbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}
// kind::f16, f32 accumulators, M = 128, N = n; b_mn: B's N dimension is the contiguous one.
template <bool BF16>
__host__ __device__ constexpr uint32_t kv_idesc(int n, bool b_mn) {
  return tc::idesc_f16(n) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u);
}

// ---- the block's rows -----------------------------------------------------------------------------

// Eight consecutive elements as f32.
template <bool BF16, bool F32>
__device__ __forceinline__ void kv_load8(const void* base, size_t at, float (&x)[8]) {
  if constexpr (F32) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + at);
    const float4 a = p[0], b = p[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + at);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float2 f = kv_unpack<BF16>(w[e]);
      x[2 * e] = f.x;
      x[2 * e + 1] = f.y;
    }
  }
}
template <bool BF16>
__device__ __forceinline__ uint4 kv_pack8(const float (&x)[8]) {
  return make_uint4(kv_pack<BF16>(x[0], x[1]), kv_pack<BF16>(x[2], x[3]), kv_pack<BF16>(x[4], x[5]), kv_pack<BF16>(x[6], x[7]));
}

struct KvArgs {
  const uint8_t* plan;
  const void* qkv;
  const float2* rope;
  uint16_t *q, *k, *v;
  const int32_t* tables;
  float* part;
  int* flags;
  int* err;
  uint16_t* out;
  size_t qkv_stride, out_stride;
  int G, kv_heads, hd, shift, num_pages, out_bt_n;
};

// One thread per 16 elements of a row: dims [8 i, 8 i + 8) and their rotation partners hd / 2 further
// on for q and k, 16 consecutive ones for v. Latency-bound: every row is read and written once.
template <bool BF16, bool F32>
__global__ void __launch_bounds__(256) kv_prep_kernel(const KvArgs a) {
  pdl_trigger();
  const KvHdr& h = *reinterpret_cast<const KvHdr*>(a.plan);
  const KvSeq* sq = reinterpret_cast<const KvSeq*>(a.plan + h.off_seq);
  const int G = a.G, kvh = a.kv_heads, H = G * kvh, hd = a.hd, half = hd / 2, per = hd / 16;
  const int units = (H + 2 * kvh) * per;
  const int M = h.M;
  const size_t total = (size_t)h.nseq * M * units;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
    const int row = (int)(i / units), u = (int)(i - (size_t)row * units);
    const int s = row / M, t = row - s * M;
    const KvSeq q = sq[s];
    if (t >= q.cnt) continue;
    const int head = u / per, c = u - head * per;
    const size_t src = (size_t)row * a.qkv_stride + (size_t)head * hd;
    const int pos = q.n + t;
    float x[8], y[8];
    if (head < H + kvh) {
      kv_load8<BF16, F32>(a.qkv, src + c * 8, x);
      kv_load8<BF16, F32>(a.qkv, src + half + c * 8, y);
      if (a.rope) {
        const float4* cs = reinterpret_cast<const float4*>(a.rope + (size_t)pos * half + c * 8);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float4 w = cs[e];
          const float x0 = x[2 * e], y0 = y[2 * e], x1 = x[2 * e + 1], y1 = y[2 * e + 1];
          x[2 * e] = x0 * w.x - y0 * w.y;
          y[2 * e] = y0 * w.x + x0 * w.y;
          x[2 * e + 1] = x1 * w.z - y1 * w.w;
          y[2 * e + 1] = y1 * w.z + x1 * w.w;
        }
      }
    } else {
      kv_load8<BF16, F32>(a.qkv, src + c * 16, x);
      kv_load8<BF16, F32>(a.qkv, src + c * 16 + 8, y);
    }
    const uint4 xv = kv_pack8<BF16>(x), yv = kv_pack8<BF16>(y);
    if (head < H) {
      const int g = head / G, j = head - g * G;
      uint16_t* d = a.q + ((size_t)g * h.R + q.row0 + (size_t)t * G + j) * hd + c * 8;
      *reinterpret_cast<uint4*>(d) = xv;
      *reinterpret_cast<uint4*>(d + half) = yv;
    } else {
      const bool is_v = head >= H + kvh;
      const int g = head - H - (is_v ? kvh : 0);
      const int page = a.tables[q.tab + (pos >> a.shift)];
      const size_t dst = ((((size_t)g * a.num_pages + page) << a.shift) + (pos & ((1 << a.shift) - 1))) * hd;
      if (is_v) {
        *reinterpret_cast<uint4*>(a.v + dst + c * 16) = xv;
        *reinterpret_cast<uint4*>(a.v + dst + c * 16 + 8) = yv;
        if (t == 0 && c == 0) a.flags[s * kvh + g] = 0;
      } else {
        *reinterpret_cast<uint4*>(a.k + dst + c * 8) = xv;
        *reinterpret_cast<uint4*>(a.k + dst + c * 8 + half) = yv;
      }
    }
  }
}

// ---- the segments -----------------------------------------------------------------------------------

template <int HD, bool BF16>
__global__ void __launch_bounds__(KV_THREADS, 1)
    kv_attn_kernel(const KvArgs a, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap) {
  using SM = KvSmem<HD>;
  constexpr int NS = SM::kStages, CB = HD / 64;      // CB: 64-element column blocks of a row
  constexpr uint32_t BLK = 128 * 128;                // bytes of one column block of a tile
  constexpr uint32_t COL_O = 256;                    // tensor memory: S / P of lane t at 128 t, O at 256 + HD t
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t k_full[NS], k_empty[NS], v_full[NS], v_empty[NS];
  __shared__ uint64_t q_full[2], s_full[2], p_full[2], pv_done[2], o_free[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const uint32_t smem = (tc::su32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem_gen = smem_raw + (smem - tc::su32(smem_raw));

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const KvHdr& h = *reinterpret_cast<const KvHdr*>(a.plan);
  const KvProg pr = reinterpret_cast<const KvProg*>(a.plan + h.off_prog)[blockIdx.x];
  const KvSeg* const segs = reinterpret_cast<const KvSeg*>(a.plan + h.off_seg);
  pdl_trigger();
  if (pr.nseg[0] + pr.nseg[1] == 0) return;

  if (tid == 0) {
    for (int s = 0; s < NS; s++) {
      tc::mbar_init(&k_full[s], 1);
      tc::mbar_init(&v_full[s], 1);
      tc::mbar_init(&k_empty[s], 2);  // both lanes' MMAs, or one lane's and its issuer
      tc::mbar_init(&v_empty[s], 2);
    }
    for (int t = 0; t < 2; t++) {
      tc::mbar_init(&q_full[t], 1);
      tc::mbar_init(&s_full[t], 1);
      tc::mbar_init(&p_full[t], 4);
      tc::mbar_init(&pv_done[t], 1);
      tc::mbar_init(&o_free[t], 4);
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::su32(&s_tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = s_tmem;
  pdl_wait();  // the query operand and the block's K/V rows

  // Ring use of lane t's chunk: pair chunk i is in stage i % NS of K and of V; chunk j of a lane's own
  // phase in stage (2 j + t) % NS, so that each lane's own stages advance with that lane alone. Its
  // phase is the number of uses the stage had before.
  auto ring = [&](int chunk, int t, int& stage, uint32_t& phase) {
    if (chunk < pr.pair_ch) {
      stage = chunk % NS;
      phase = (uint32_t)(chunk / NS);
    } else {
      const int v = 2 * (chunk - pr.pair_ch) + t;
      stage = v % NS;
      phase = (uint32_t)((pr.pair_ch - stage + NS - 1) / NS + v / NS);
    }
  };

  if (warp == 10) {
    // ---- producer: K and V chunks through the page tables, one box per page and column block ----
    const int page = 1 << a.shift, pg_rows = min(page, KV_CHUNK);
    struct Cursor {
      int seg, end, j, chunk;
    };
    Cursor cur[2] = {{pr.seg[0], pr.seg[0] + pr.nseg[0], 0, 0}, {pr.seg[1] + pr.npair, pr.seg[1] + pr.nseg[1], 0, pr.pair_ch}};
    bool ok = true;
    uint32_t issued = 0, parity = 0;  // per ring slot (K stages, then V stages): a copy was issued, its phase's parity
    int t = 0;
    while (ok && (cur[0].seg < cur[0].end || cur[1].seg < cur[1].end)) {
      if (cur[t].seg >= cur[t].end) t ^= 1;
      Cursor& c = cur[t];
      const KvSeg s = segs[c.seg];
      const int pc = s.p0 + c.j * KV_CHUNK;
      const int npg = (min(KV_CHUNK, s.p1 - pc) + pg_rows - 1) / pg_rows;
      const int i = lane / CB, cb = lane - i * CB;
      const int pid = i < npg ? a.tables[s.tab + ((pc + i * pg_rows) >> a.shift)] : 0;
      const int y = ((s.kv_head * a.num_pages + pid) << a.shift) + (pc & (page - 1));
      int st;
      uint32_t ph;
      ring(c.chunk, t, st, ph);
      const uint32_t off = (uint32_t)st * SM::kTile + cb * BLK + (uint32_t)(i * pg_rows) * 128u;
#pragma unroll
      for (int kv = 0; kv < 2; kv++) {
        uint64_t* full = kv ? &v_full[st] : &k_full[st];
        uint64_t* empty = kv ? &v_empty[st] : &k_empty[st];
        if (ph > 0) ok = ok && tc::mbar_wait_fast(empty, (ph - 1) & 1, &s_abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) tc::mbar_expect_tx(full, (uint32_t)(npg * pg_rows) * HD * 2);
        __syncwarp();
        issued |= 1u << (kv * NS + st);
        parity = (parity & ~(1u << (kv * NS + st))) | ((ph & 1) << (kv * NS + st));
        if (i < npg) kv_tma2d(smem + (kv ? SM::kV : SM::kK) + off, kv ? &vmap : &kmap, cb * 64, y, full);
      }
      c.chunk++;
      if (++c.j == s.nch) {
        c.j = 0;
        c.seg++;
      }
      if (c.chunk > pr.pair_ch || (c.chunk == pr.pair_ch && t == 0)) t = c.chunk == pr.pair_ch ? 0 : t ^ 1;
    }
    if (!ok) {  // copies in flight land before the CTA leaves
      int never = 0;
      for (int s = 0; s < 2 * NS; s++)
        if (issued >> s & 1) (void)tc::mbar_wait(s < NS ? &k_full[s] : &v_full[s - NS], parity >> s & 1, &never);
    }
  } else if (warp >= 8) {
    // ---- MMA issuer of lane t ----
    const int t = warp - 8;
    if (lane == 0 && pr.nseg[t] > 0) {
      const uint32_t sq = smem + SM::kQ + t * SM::kTile;
      const uint32_t t_s = tmem + t * 128, t_o = tmem + COL_O + t * HD;
      auto load_q = [&](int seg) {
        tc::mbar_expect_tx(&q_full[t], SM::kTile);
        const int y = segs[seg].qrow;
#pragma unroll
        for (int cb = 0; cb < CB; cb++) kv_tma2d(sq + cb * BLK, &qmap, cb * 64, y, &q_full[t]);
      };
      load_q(pr.seg[t]);
      int chunk = 0, nq = 1;
      bool ok = true;
      for (int i = 0; ok && i < pr.nseg[t]; i++) {
        const int nch = segs[pr.seg[t] + i].nch;
        for (int j = 0; j < nch; j++, chunk++) {
          int st;
          uint32_t ph;
          ring(chunk, t, st, ph);
          const bool pair = chunk < pr.pair_ch;
          // scores: Q and the K chunk are in shared memory, the last P has been read
          if (j == 0) ok = ok && tc::mbar_wait_fast(&q_full[t], i & 1, &s_abort);
          ok = ok && tc::mbar_wait_fast(&k_full[st], ph & 1, &s_abort);
          if (chunk > 0) ok = ok && tc::mbar_wait_fast(&pv_done[t], (chunk - 1) & 1, &s_abort);
          if (!ok) break;
          tc::fence_after();
          const uint32_t sk = smem + SM::kK + st * SM::kTile;
#pragma unroll
          for (int k = 0; k < HD / 16; k++) {
            const uint32_t o = (k / 4) * BLK + (k % 4) * 32u;
            tc::mma_f16_ss(t_s, kv_sdesc(sq + o, 16), kv_sdesc(sk + o, 16), kv_idesc<BF16>(128, false), k > 0 ? 1u : 0u);
          }
          tc::commit(&s_full[t]);
          tc::commit(&k_empty[st]);
          if (!pair) tc::mbar_arrive(&k_empty[st]);
          // values: P is in tensor memory (and S, hence Q and K, have been read)
          ok = ok && tc::mbar_wait_fast(&p_full[t], chunk & 1, &s_abort);
          if (ok && j == nch - 1 && i + 1 < pr.nseg[t]) {
            load_q(pr.seg[t] + i + 1);
            nq++;
          }
          ok = ok && tc::mbar_wait_fast(&v_full[st], ph & 1, &s_abort);
          if (j == 0 && i > 0) ok = ok && tc::mbar_wait_fast(&o_free[t], (i - 1) & 1, &s_abort);
          if (!ok) break;
          tc::fence_after();
          const uint32_t sv = smem + SM::kV + st * SM::kTile;
#pragma unroll
          for (int k = 0; k < KV_CHUNK / 16; k++)
            tc::mma_f16_ts(t_o, t_s + k * 8, kv_sdesc(sv + k * 2048u, BLK), kv_idesc<BF16>(HD, true), (j > 0 || k > 0) ? 1u : 0u);
          tc::commit(&pv_done[t]);
          tc::commit(&v_empty[st]);
          if (!pair) tc::mbar_arrive(&v_empty[st]);
        }
      }
      if (!ok) {  // the query tile in flight lands, the MMAs in flight end
        int never = 0;
        (void)tc::mbar_wait(&q_full[t], (nq - 1) & 1, &never);
        tc::commit(&q_full[t]);
        (void)tc::mbar_wait(&q_full[t], nq & 1, &never);
      }
    }
  } else {
    // ---- softmax of lane t: one query row per thread ----
    const int t = warp >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t t_s = tmem + ((uint32_t)(quad * 32) << 16) + t * 128;
    const uint32_t t_o = tmem + ((uint32_t)(quad * 32) << 16) + COL_O + t * HD;
    const float cs = 1.4426950408889634f / sqrtf((float)HD);
    int chunk = 0;
    bool ok = true;
    for (int i = 0; ok && i < pr.nseg[t]; i++) {
      const KvSeg s = segs[pr.seg[t] + i];
      const bool active = quad * 32 < s.nrows, row_ok = row < s.nrows;  // active: warp-uniform
      // last position the row sees
      int lim = s.p1 - 1;
      if (s.causal != INT_MAX && row_ok) lim = min(lim, s.causal + (s.trow0 + row) / a.G);
      float m_ref = -CUDART_INF_F, l = 0.f;
      for (int j = 0; j < s.nch; j++, chunk++) {
        const int pc = s.p0 + j * KV_CHUNK;
        ok = tc::mbar_wait_fast(&s_full[t], chunk & 1, &s_abort);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc::fence_after();
        if (active) {
          float x[128];
#pragma unroll
          for (int q = 0; q < 4; q++) kv_ld32(t_s + q * 32, x + q * 32);
          tc::wait_ld();
          const int vis = lim - pc;  // columns 0 .. vis are visible
          const bool all = __all_sync(0xffffffffu, vis >= KV_CHUNK - 1 || !row_ok);
          if (!all) {
#pragma unroll
            for (int c = 0; c < 128; c++) x[c] = c <= vis ? x[c] : -CUDART_INF_F;
          }
          float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
          for (int c = 0; c < 128; c++) mx[c & 3] = fmaxf(mx[c & 3], x[c]);
          const float m_new = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * cs;
          if (j == 0) {
            m_ref = m_new;
          } else if (__any_sync(0xffffffffu, row_ok && m_new > m_ref + KV_RESCALE)) {
            // O and l to the new maximum, once the last P V has been added
            ok = tc::mbar_wait_fast(&pv_done[t], (chunk - 1) & 1, &s_abort);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc::fence_after();
            const float m2 = fmaxf(m_ref, m_new);
            const float f = m2 == -CUDART_INF_F ? 1.f : kv_ex2(m_ref - m2);
            m_ref = m2;
            l *= f;
#pragma unroll 1
            for (int q = 0; q < HD / 16; q++) {
              float o[16];
              tc::ld16(t_o + q * 16, reinterpret_cast<uint32_t*>(o));
              tc::wait_ld();
#pragma unroll
              for (int e = 0; e < 16; e++) o[e] *= f;
              tc::st16(t_o + q * 16, reinterpret_cast<uint32_t*>(o));
            }
          }
          const float mb = m_ref == -CUDART_INF_F ? 0.f : m_ref;
          float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < 4; q++) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; e++) {
              const float e0 = kv_ex2(fmaf(x[q * 32 + 2 * e], cs, -mb)), e1 = kv_ex2(fmaf(x[q * 32 + 2 * e + 1], cs, -mb));
              ls[(2 * e) & 3] += e0;
              ls[(2 * e + 1) & 3] += e1;
              pk[e] = kv_pack<BF16>(e0, e1);
            }
            tc::st16(t_s + q * 16, pk);
          }
          l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
          tc::wait_st();
        }
        // V rows that nobody sees (past the range) are zeroed, and infinities and NaN of rows that
        // only some of the tile see; all four warps take part
        const bool tail = pc + KV_CHUNK > s.p1;
        const bool fresh = s.causal != INT_MAX && s.p1 > s.causal + 1 && pc + KV_CHUNK > s.causal + 1;
        if (tail || fresh) {
          int st;
          uint32_t ph;
          ring(chunk, t, st, ph);
          ok = tc::mbar_wait_fast(&v_full[st], ph & 1, &s_abort);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          uint8_t* sv = smem_gen + SM::kV + st * SM::kTile;
          const int r1 = min(KV_CHUNK, s.p1 - pc);
          const int r0 = fresh ? max(0, s.causal + 1 - pc) : r1;
          for (int k = row; k < (KV_CHUNK - r0) * CB * 8; k += 128) {
            const int r = r0 + k / (CB * 8), c = k % (CB * 8);
            uint4* p = reinterpret_cast<uint4*>(sv + (c >> 3) * BLK + r * 128 + (c & 7) * 16);
            if (r >= r1) {
              *p = make_uint4(0, 0, 0, 0);
            } else {
              uint4 v = *p;
              const uint4 n = make_uint4(kv_nonfinite<BF16>(v.x), kv_nonfinite<BF16>(v.y), kv_nonfinite<BF16>(v.z), kv_nonfinite<BF16>(v.w));
              if (n.x | n.y | n.z | n.w) {
                *p = make_uint4(v.x & ~n.x, v.y & ~n.y, v.z & ~n.z, v.w & ~n.w);
                a.flags[s.flag] = 1;
              }
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      ok = tc::mbar_wait_fast(&pv_done[t], (chunk - 1) & 1, &s_abort);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc::fence_after();
      if (active) {
        float* po = a.part + ((size_t)s.slot + row) * HD;
#pragma unroll
        for (int q = 0; q < HD / 32; q++) {
          float o[32];
          kv_ld32(t_o + q * 32, o);
          tc::wait_ld();
          if (row_ok)
#pragma unroll
            for (int e = 0; e < 8; e++)
              reinterpret_cast<float4*>(po + q * 32)[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
        if (row_ok) reinterpret_cast<float2*>(a.part + (size_t)h.nslots * HD)[s.slot + row] = make_float2(m_ref, l);
      }
      tc::fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&o_free[t]);
    }
  }

  tc::fence_before();
  __syncthreads();
  if (warp == 0) {
    tc::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  if (s_abort && tid == 0) {
    *reinterpret_cast<volatile int*>(a.err) = 1;
    __threadfence_system();
  }
}

// ---- the partials ---------------------------------------------------------------------------------

// One warp per query row: the maxima of the row's partials, then their weighted sum in plan order
// (the result does not depend on timing). BT: f16 in the batched GEMM's operand layout.
template <int HD, bool BF16, bool BT>
__global__ void __launch_bounds__(128) kv_merge_kernel(const KvArgs a) {
  constexpr int W = HD / 32;  // f32 per lane
  pdl_trigger();
  const KvHdr& h = *reinterpret_cast<const KvHdr*>(a.plan);
  const KvSeq* sqs = reinterpret_cast<const KvSeq*>(a.plan + h.off_seq);
  const KvNode* nodes = reinterpret_cast<const KvNode*>(a.plan + h.off_node);
  const int32_t* uoff = reinterpret_cast<const int32_t*>(a.plan + h.off_uoff);
  const int32_t* useg = reinterpret_cast<const int32_t*>(a.plan + h.off_useg);
  const int lane = threadIdx.x & 31;
  const int G = a.G, kvh = a.kv_heads, H = G * kvh;
  const float2* pml = reinterpret_cast<const float2*>(a.part + (size_t)h.nslots * HD);
  pdl_wait();
  const size_t total = (size_t)h.nseq * h.M * H;
  for (size_t it = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5); it < total; it += (size_t)gridDim.x * 4) {
    const int orow = (int)(it / H), head = (int)(it - (size_t)orow * H);
    const int s = orow / h.M, t = orow - s * h.M;
    const KvSeq q = sqs[s];
    if (t >= q.cnt) continue;
    const int g = head / G, row = q.row0 + t * G + (head - g * G);
    float m = -CUDART_INF_F, l = 0.f, acc[W];
#pragma unroll
    for (int e = 0; e < W; e++) acc[e] = 0.f;
#pragma unroll 1
    for (int pass = 0; pass < 2; pass++) {
#pragma unroll 1
      for (int lv = 0; lv < q.nlev; lv++) {
        const KvNode nd = nodes[q.node[lv]];
        const int lr = row - nd.row0, u = nd.unit0 + g * nd.ntile + lr / KV_TILE;
        const int k1 = uoff[u + 1];
        for (int k0 = uoff[u]; k0 < k1; k0 += 32) {
          int slot = 0;
          float2 ml = make_float2(-CUDART_INF_F, 0.f);
          if (k0 + lane < k1) {
            slot = useg[k0 + lane] + lr % KV_TILE;
            ml = __ldcg(pml + slot);
          }
          if (pass == 0) {
            m = fmaxf(m, ml.x);
            continue;
          }
          const float w = ml.x == -CUDART_INF_F ? 0.f : kv_ex2(ml.x - m);
          l += w * ml.y;
          const int n = min(32, k1 - k0);
#pragma unroll 4
          for (int k = 0; k < n; k++) {
            const float wk = __shfl_sync(0xffffffffu, w, k);
            const float* p = a.part + (size_t)__shfl_sync(0xffffffffu, slot, k) * HD + lane * W;
            if constexpr (W == 4) {
              const float4 v = __ldcg(reinterpret_cast<const float4*>(p));
              acc[0] += wk * v.x;
              acc[1] += wk * v.y;
              acc[2] += wk * v.z;
              acc[3] += wk * v.w;
            } else {
              const float2 v = __ldcg(reinterpret_cast<const float2*>(p));
              acc[0] += wk * v.x;
              acc[1] += wk * v.y;
            }
          }
        }
      }
      if (pass == 0) m = warp_max(m);
    }
    l = warp_sum(l);
    const float inv = 1.0f / l;
#pragma unroll
    for (int e = 0; e < W; e++) acc[e] *= inv;
    if (t > 0 && a.flags[s * kvh + g]) {  // infinities and NaN of the block's own V rows that this row sees
      for (int tt = 1; tt <= t; tt++) {
        const int pos = q.n + tt;
        const size_t src = ((((size_t)g * a.num_pages + a.tables[q.tab + (pos >> a.shift)]) << a.shift) + (pos & ((1 << a.shift) - 1))) * HD + lane * W;
#pragma unroll
        for (int e = 0; e < W; e += 2) {
          const uint32_t v = *reinterpret_cast<const uint32_t*>(a.v + src + e);
          const uint32_t n = kv_nonfinite<BF16>(v);
          const float2 f = kv_unpack<BF16>(v);
          if (n & 0xffffu) acc[e] += f.x;
          if (n >> 16) acc[e + 1] += f.y;
        }
      }
    }
    uint16_t* o = BT ? a.out + bt_off(orow, head * HD + lane * W, H * HD, a.out_bt_n) : a.out + (size_t)orow * a.out_stride + (size_t)head * HD + lane * W;
    if constexpr (W == 4)
      *reinterpret_cast<uint2*>(o) = make_uint2(kv_pack<BF16>(acc[0], acc[1]), kv_pack<BF16>(acc[2], acc[3]));
    else
      *reinterpret_cast<uint32_t*>(o) = kv_pack<BF16>(acc[0], acc[1]);
  }
}

// ---- page copies ------------------------------------------------------------------------------------

constexpr int KV_COPIES = 1024;  // copies of one launch (they travel in its parameters)
struct KvCopyList {
  PageCopy c[KV_COPIES];
};

// Tasks of 4 KB: (copy, layer x head, K or V, piece of the page's rows). Every lane has its eight
// 16-byte loads in flight before the first store. Bound by HBM: each byte is read and written once.
__global__ void __launch_bounds__(256) kv_copy_kernel(const __grid_constant__ KvCopyList list, int n, uint4* __restrict__ k,
                                                      uint4* __restrict__ v, int blocks, int num_pages, int page16, int row16, int pieces) {
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * 8;
  const long long tasks = (long long)n * blocks * 2 * pieces;
  for (long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); w < tasks; w += warps) {
    long long x = w;
    const int piece = (int)(x % pieces);
    x /= pieces;
    const int kv = (int)(x & 1);
    x >>= 1;
    const int b = (int)(x % blocks), i = (int)(x / blocks);
    const PageCopy c = list.c[i];
    const int end = c.rows * row16;
    const int at = piece * 256 + lane;
    if (piece * 256 >= end) continue;
    uint4* base = (kv ? v : k) + (size_t)b * num_pages * page16;
    const uint4* src = base + (size_t)c.src * page16;
    uint4* dst = base + (size_t)c.dst * page16;
    uint4 r[8];
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (at + e * 32 < end) r[e] = __ldcs(src + at + e * 32);
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (at + e * 32 < end) dst[at + e * 32] = r[e];
  }
}

void launch_page_copies(void* k, void* v, int layers, int kv_heads, int hd, int page, int num_pages, const PageCopy* c, size_t n,
                        int num_sms, cudaStream_t s) {
  const int row16 = hd / 8;
  for (size_t i = 0; i < n; i += KV_COPIES) {
    KvCopyList list;
    const int m = (int)std::min<size_t>(KV_COPIES, n - i);
    int rows = 0;
    for (int e = 0; e < m; e++) {
      list.c[e] = c[i + e];
      rows = std::max(rows, (int)c[i + e].rows);
    }
    if (rows == 0) continue;
    const int pieces = (rows * row16 + 255) / 256, blocks = layers * kv_heads;
    const long long tasks = (long long)m * blocks * 2 * pieces;
    const int grid = (int)std::min<long long>((tasks + 7) / 8, (long long)num_sms * 8);
    kv_copy_kernel<<<grid, 256, 0, s>>>(list, m, reinterpret_cast<uint4*>(k), reinterpret_cast<uint4*>(v), blocks, num_pages, page * row16,
                                        row16, pieces);
    LS_CUDA(cudaGetLastError());
  }
}

__global__ void __launch_bounds__(128) kv_table_kernel(int32_t* __restrict__ table, const KvRange* __restrict__ ranges, int n) {
  const KvRange r = ranges[blockIdx.x];
  const int32_t* vals = reinterpret_cast<const int32_t*>(ranges + n) + r.from;
  for (int i = threadIdx.x; i < r.n; i += 128) table[r.at + i] = vals[i];
}

void launch_table_update(int32_t* table, const KvRange* ranges, int nranges, cudaStream_t s) {
  kv_table_kernel<<<nranges, 128, 0, s>>>(table, ranges, nranges);
  LS_CUDA(cudaGetLastError());
}

// ---- launches ---------------------------------------------------------------------------------------

void kv_encode_map(CUtensorMap* m, const void* base, uint64_t rows, int hd, int box_rows, bool bf16) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  cudaDriverEntryPointQueryResult qr;
  void* fn = nullptr;
  LS_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qr));
  if (qr != cudaDriverEntryPointSuccess || !fn) LS_THROW(LS_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t dims[2] = {(cuuint64_t)hd, rows};
  const cuuint64_t strides[1] = {(cuuint64_t)hd * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, es[2] = {1, 1};
  const CUresult r = reinterpret_cast<Encode>(fn)(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                                                  const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) LS_THROW(LS_ERR_CUDA, "cuTensorMapEncodeTiled (K/V cache) failed: " + std::to_string((int)r));
}

void KvWork::open(const KvGeom& geom, bool is_bf16, int* err_word) {
  g = geom;
  bf16 = is_bf16;
  err = err_word;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const size_t qrows = g.rows_cap() * g.kv_heads;
  const size_t bp = up(g.plan_cap()), bq = up(qrows * g.hd * 2), bo = up(g.slots_cap() * (g.hd + 2) * 4), bf = up((size_t)g.nseq * g.kv_heads * 4);
  LS_CUDA(cudaMalloc(&mem, bp + bq + bo + bf));
  uint8_t* p = reinterpret_cast<uint8_t*>(mem);
  plan = p;
  q = p + bp;
  part = reinterpret_cast<float*>(p + bp + bq);
  flags = reinterpret_cast<int*>(p + bp + bq + bo);
  // the query operand's rows past the block's are read into tiles (and never used): finite from the start
  LS_CUDA(cudaMemset(q, 0, bq));
  LS_CUDA(cudaMemset(flags, 0, bf));
  kv_encode_map(&qmap, q, qrows, g.hd, KV_TILE, bf16);
}

void KvWork::close() {
  if (mem) cudaFree(mem);
  mem = nullptr;
}

template <int HD, bool BF16>
static void launch_kv_t(const KvWork& w, const KvAttn& a, const KvArgs& k, cudaStream_t s) {
  const int units = (w.g.heads + 2 * w.g.kv_heads) * (HD / 16);
  const size_t items = (size_t)a.rows * units;
  const int gp = (int)std::min<size_t>((items + 255) / 256, (size_t)w.g.nctas * 8);
  if (a.qkv_f32)
    kv_prep_kernel<BF16, true><<<gp, 256, 0, s>>>(k);
  else
    kv_prep_kernel<BF16, false><<<gp, 256, 0, s>>>(k);
  LS_CUDA(cudaGetLastError());
  const size_t smem = KvSmem<HD>::kTotal;
  ensure_smem(kv_attn_kernel<HD, BF16>, smem);
  launch_pdl(kv_attn_kernel<HD, BF16>, dim3(w.g.nctas), dim3(KV_THREADS), smem, s, k, w.qmap, *a.kmap, *a.vmap);
  const int gm = (int)std::min<size_t>(((size_t)a.rows * w.g.heads + 3) / 4, (size_t)w.g.nctas * 16);
  if constexpr (!BF16) {
    if (a.out_bt) return launch_pdl(kv_merge_kernel<HD, false, true>, dim3(gm), dim3(128), 0, s, k);
  }
  launch_pdl(kv_merge_kernel<HD, BF16, false>, dim3(gm), dim3(128), 0, s, k);
}

void launch_kv_attention(const KvWork& w, const KvAttn& a, cudaStream_t s) {
  KvArgs k{};
  k.plan = w.plan;
  k.qkv = a.qkv;
  k.rope = a.rope;
  k.q = reinterpret_cast<uint16_t*>(w.q);
  k.k = reinterpret_cast<uint16_t*>(a.k);
  k.v = reinterpret_cast<uint16_t*>(a.v);
  k.tables = a.tables;
  k.part = w.part;
  k.flags = w.flags;
  k.err = w.err;
  k.out = a.out_bt ? a.out_bt : reinterpret_cast<uint16_t*>(a.out);
  k.qkv_stride = a.qkv_stride;
  k.out_stride = a.out_stride;
  k.G = w.g.G();
  k.kv_heads = w.g.kv_heads;
  k.hd = w.g.hd;
  k.shift = w.g.shift;
  k.num_pages = w.g.num_pages;
  k.out_bt_n = a.out_bt_n;
  if (w.g.hd == 64) return w.bf16 ? launch_kv_t<64, true>(w, a, k, s) : launch_kv_t<64, false>(w, a, k, s);
  return w.bf16 ? launch_kv_t<128, true>(w, a, k, s) : launch_kv_t<128, false>(w, a, k, s);
}

}  // namespace ls
