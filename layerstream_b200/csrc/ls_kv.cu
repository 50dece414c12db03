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
// per lane, one TMA producer warp. K and V come in chunks of 128 positions; the softmax takes them by halves of
// 64, so that a lane's two S buffers fit beside O in tensor memory at hd 128 too, and the tensor cores work
// on one half while the softmax works on the other. (Many pair tiles: 64 sequences of 32 rows, 4096 positions
// each, 16/2 heads of 128 in bf16 or 14/2 of 64 in f16, one call in a graph. One buffer of 128 positions: 107 instead
// of 90 us at hd 128; at hd 64, where the next S could follow as soon as the last one was in registers, 75 us
// either way.) O stays in tensor memory and is rescaled only when a row's maximum has
// grown by more than 2^8 over the one its exponents are taken against.
//
// Bound, per two tiles and 128 positions: the special-function units need 2048 clocks for the exponentials
// (1536 with a quarter of them on the FMA units), the tensor cores 1024 at hd 64 and 2048 at hd 128, an
// SM's share of HBM 1450 and 2900 for K and V that nobody else reads; the kernel takes about 3400. The
// rest is the latency of a row's chain through one step (scores out of tensor memory, maximum,
// exponentials, P into tensor memory, P V, next S). More warps did not hide it: four softmax warpgroups,
// two for each tile, took 99 us for many pair tiles at hd 128 when they shared a step's columns and 100
// when they took the steps in turn, against 90 with two.
//
// Rounding: q (after rotation) and P enter the tensor core in the cache's 16-bit type, the type that
// its operands K and V have; scores, maxima, sums, O and the partials stay f32; the output is rounded
// once. (P in a high and a low part takes 8 to 20 % more time.) Infinities and NaN in V rows that only some of a tile's rows may see (the block's own rows)
// are replaced by zeros for the MMA, since 0 x inf would reach the rows that do not see them, and the
// merge adds them back to the rows that do.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "layerstream.h"
#include "ls_device.cuh"
#include "ls_kv.h"

namespace ls {

constexpr int KV_THREADS = 352;  // 2 softmax warpgroups, 2 issuer warps, 1 producer warp
constexpr int KV_HALF = KV_CHUNK / 2;  // positions that a step of the softmax takes
constexpr int KV_SEGS_NEAR = 32;    // segments of a lane that are held in shared memory
constexpr float KV_RESCALE = 8.0f;  // log2 growth of a row's maximum that O is rescaled for

template <int HD>
struct KvSmem {
  static constexpr int kTile = KV_TILE * HD * 2;    // Q tile
  static constexpr int kChunk = KV_CHUNK * HD * 2;  // K chunk, V chunk
  static constexpr int kStages = HD == 64 ? 4 : 2;  // of K and of V; even: in the lanes' own phase lane t owns those of parity t
  static constexpr int kQ = 0, kK = 2 * kTile, kV = kK + kStages * kChunk;
  static constexpr int kTotal = kV + kStages * kChunk + 1024;  // + alignment
};

// ---- small device helpers -----------------------------------------------------------------------

__device__ __forceinline__ float kv_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two f32 in one register pair.
__device__ __forceinline__ uint64_t kv_f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 kv_un2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t kv_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t kv_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float kv_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float kv_max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 2^z on the FMA units, for a share of the exponentials (the special-function units do 16 a clock and SM):
// z = n + f, n the nearest integer (Cody and Waite's reduction; it sits in the low bits of z + 1.5 * 2^23),
// 2^f by the quartic with the least largest relative error on [-1/2, 1/2] (Remez exchange, 2.7e-6), n added
// to the exponent; z up to 8 occurs. A NaN does not come through: the row's maximum carries it. In f16 z is clamped
// at -126: 2^-126 rounds to zero in P. In bf16 it would be a weight, on positions that the row does not see (z =
// -inf) too; there z is clamped at -127, where the quartic is just below 1, so that taking 127 from its exponent
// leaves a negative integer, which becomes zero (every z <= -127 then gives zero, and what lies between -127 and
// -126 is off by at most 2^-127; ex2.approx.ftz flushes it).
// Many pair tiles at hd 128 and 64: no share 93.7 and 79.8 us, a quarter 89.7 and 77.3, 3/8 90.4 and
// 77.4, half 94.1 and 80.9.
template <bool BF16>
__device__ __forceinline__ float2 kv_ex2_fma(uint64_t z) {
  constexpr float LOW = BF16 ? -127.f : -126.f;
  const float2 zf = kv_un2(z);
  z = kv_f2(fmaxf(zf.x, LOW), fmaxf(zf.y, LOW));
  const uint64_t r = kv_add2(z, kv_f2(12582912.f, 12582912.f));
  const uint64_t f = kv_fma2(kv_add2(r, kv_f2(-12582912.f, -12582912.f)), kv_f2(-1.f, -1.f), z);
  uint64_t p = kv_f2(0x1.3997d6p-7f, 0x1.3997d6p-7f);
  p = kv_fma2(p, f, kv_f2(0x1.ca1444p-5f, 0x1.ca1444p-5f));
  p = kv_fma2(p, f, kv_f2(0x1.ec06dap-3f, 0x1.ec06dap-3f));
  p = kv_fma2(p, f, kv_f2(0x1.62e0dcp-1f, 0x1.62e0dcp-1f));
  p = kv_fma2(p, f, kv_f2(0x1.ffffe8p-1f, 0x1.ffffe8p-1f));
  const float2 pf = kv_un2(p), rf = kv_un2(r);
  int x = __float_as_int(pf.x) + (__float_as_int(rf.x) << 23), y = __float_as_int(pf.y) + (__float_as_int(rf.y) << 23);
  if constexpr (BF16) x = max(x, 0), y = max(y, 0);
  return make_float2(__int_as_float(x), __int_as_float(y));
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
// Loads issued so far have landed; v (32 of their registers) is not read before.
__device__ __forceinline__ void kv_wait32(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]),
                 "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]),
                 "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]),
                 "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}
// Bounded wait on an mbarrier phase (a second or so), false and the CTA's abort flag on timeout. The loop is
// not unrolled: it stands in the code many times.
__device__ __forceinline__ bool kv_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
#pragma unroll 1
  for (uint32_t i = 0; i < (1u << 22); i++) {
    if (tc::mbar_try(bar, parity)) return true;
    if ((i & 63) == 63 && *abort) return false;
  }
  *abort = 1;
  return false;
}
__device__ __forceinline__ void kv_tma2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(tc::su32(bar))
      : "memory");
}
// Low word of the shared-memory matrix descriptor of a 128-byte-swizzled tile (8-row groups 1024 bytes apart);
// lbo = bytes between 64-element blocks of the contiguous dimension when that is the operand's M or N.
__device__ __forceinline__ uint32_t kv_desc(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | (lbo >> 4) << 16; }
constexpr uint32_t KV_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);  // row-group stride, version 1, 128-byte swizzle
// kind::f16, f32 accumulators, M = 128, N = n; b_mn: B's N dimension is the contiguous one.
template <bool BF16>
__host__ __device__ constexpr uint32_t kv_idesc(int n, bool b_mn) {
  return tc::idesc_f16(n) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u);
}
// MMAs of a converged warp, issued by its elected lane (lead), so that their operands stay warp-uniform.
__device__ __forceinline__ void kv_mma_ss(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 x, {%2, %6};\n\t"
      "mov.b64 y, {%3, %6};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%1], x, y, %4, p;\n\t}" ::"r"(lead),
      "r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "n"(KV_DESC_HI)
      : "memory");
}
__device__ __forceinline__ void kv_mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 y, {%3, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], y, %4, p;\n\t}" ::"r"(lead),
      "r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "n"(KV_DESC_HI)
      : "memory");
}
__device__ __forceinline__ void kv_commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}" ::"r"(lead),
      "r"(tc::su32(bar))
      : "memory");
}
__device__ __forceinline__ uint32_t kv_elect() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e;
}
__device__ __forceinline__ void kv_st8(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]),
               "f"(v[6]), "f"(v[7])
               : "memory");
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
  int G, kv_heads, hd, shift, num_pages, out_bt_n, rows, M;
};

// One thread per 16 elements of a row: dims [8 i, 8 i + 8) and their rotation partners hd / 2 further
// on for q and k, 16 consecutive ones for v. Latency-bound: every row is read and written once.
template <bool BF16, bool F32>
__global__ void __launch_bounds__(256) kv_prep_kernel(const KvArgs a) {
  // The rows are there, the last call's kernels have read what is overwritten here, and the step's plan is: the
  // attention and merge kernels read it before they wait for anything, so they may start from here on.
  pdl_wait();
  pdl_trigger();
  const KvHdr& h = *reinterpret_cast<const KvHdr*>(a.plan);
  const KvSeq* sq = reinterpret_cast<const KvSeq*>(a.plan + KV_SEQ_AT);
  const int G = a.G, kvh = a.kv_heads, H = G * kvh, hd = a.hd, half = hd / 2, per = hd / 16;
  const int units = (H + 2 * kvh) * per;
  const size_t total = (size_t)a.rows * units;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
    const int row = (int)(i / units), u = (int)(i - (size_t)row * units);
    const int s = row / a.M, t = row - s * a.M;
    const int4 q4 = *reinterpret_cast<const int4*>(sq + s);  // the first fields, in one load
    const int n = q4.x, cnt = q4.y, row0 = q4.z, tab = q4.w, pos = n + t;
    if (t >= cnt) continue;
    const int head = u / per, c = u - head * per;
    const size_t src = (size_t)row * a.qkv_stride + (size_t)head * hd;
    const bool rot = head < H + kvh;
    float x[8], y[8];
    kv_load8<BF16, F32>(a.qkv, src + c * (rot ? 8 : 16), x);
    kv_load8<BF16, F32>(a.qkv, src + (rot ? half + c * 8 : c * 16 + 8), y);
    if (rot && a.rope) {
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
    const uint4 xv = kv_pack8<BF16>(x), yv = kv_pack8<BF16>(y);
    if (head < H) {
      const int g = head / G, j = head - g * G;
      uint16_t* d = a.q + ((size_t)g * h.R + row0 + (size_t)t * G + j) * hd + c * 8;
      *reinterpret_cast<uint4*>(d) = xv;
      *reinterpret_cast<uint4*>(d + half) = yv;
    } else {
      const bool is_v = head >= H + kvh;
      const int g = head - H - (is_v ? kvh : 0);
      const int page = a.tables[tab + (pos >> a.shift)];
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
    kv_attn_kernel(const KvArgs a, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap qhalf,
                   const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using SM = KvSmem<HD>;
  constexpr int NS = SM::kStages, CB = HD / 64;      // CB: 64-element column blocks of a row
  constexpr uint32_t QBLK = KV_TILE * 128, BLK = KV_CHUNK * 128;  // bytes of one column block of a Q tile, of a K or V chunk
  // Tensor memory of lane t: S of its even and odd half chunks at 128 t and 128 t + 64, P (two values a column)
  // over the first half of the S it comes from, O at 256 + HD t.
  constexpr uint32_t COL_O = 256;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t k_full[NS], k_empty[NS], v_full[NS], v_empty[NS];
  __shared__ uint64_t q_full[2][2], s_full[2][2], p_full[2][2], pv_done[2][2], o_free[2];
  __shared__ __align__(16) KvSeg s_segs[2][KV_SEGS_NEAR];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const uint32_t smem = (tc::su32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem_gen = smem_raw + (smem - tc::su32(smem_raw));

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const KvHdr& h = *reinterpret_cast<const KvHdr*>(a.plan);
  const KvProg pr = reinterpret_cast<const KvProg*>(a.plan + h.off_prog)[blockIdx.x];
  const KvSeg* const segs = reinterpret_cast<const KvSeg*>(a.plan + h.off_seg);
  if (pr.nseg[0] + pr.nseg[1] == 0) return pdl_wait();  // (when this grid has ended, the one before it has: in a step without rows too)

  constexpr int SEG16 = sizeof(KvSeg) / 16;
  static_assert(sizeof(KvSeg) % 16 == 0, "segments are copied in 16-byte pieces");
  for (int t = 0; t < 2; t++)
    for (int i = tid; i < min(pr.nseg[t], KV_SEGS_NEAR) * SEG16; i += KV_THREADS)
      reinterpret_cast<uint4*>(s_segs[t])[i] = reinterpret_cast<const uint4*>(segs + pr.seg[t])[i];
  auto seg_of = [&](int t, int i) -> const KvSeg& { return i < KV_SEGS_NEAR ? s_segs[t][i] : segs[pr.seg[t] + i]; };
  if (tid == 0) {
    for (int s = 0; s < NS; s++) {
      tc::mbar_init(&k_full[s], 1);
      tc::mbar_init(&v_full[s], 1);
      tc::mbar_init(&k_empty[s], 2);  // both lanes' MMAs, or one lane's and its issuer
      tc::mbar_init(&v_empty[s], 2);
    }
    for (int t = 0; t < 2; t++) {
      for (int e = 0; e < 2; e++) {
        tc::mbar_init(&q_full[t][e], 1);
        tc::mbar_init(&s_full[t][e], 1);
        tc::mbar_init(&p_full[t][e], 4);
        tc::mbar_init(&pv_done[t][e], 1);
      }
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
  // Only now: a kernel two launches on (the next product) takes tensor memory before it waits for this one. Were it
  // let onto the SM first, the allocation here could wait for it, and it for this kernel.
  pdl_trigger();
  const uint32_t tmem = s_tmem;
  // Ring use of lane t's chunk: pair chunk i is in stage i % NS of K and of V; chunk j of a lane's own
  // phase in stage (2 j + t) % NS, so that each lane's own stages advance with that lane alone. Its
  // phase is the number of uses the stage had before.
  auto ring = [&](int chunk, int t, int& stage, uint32_t& phase) {
    const uint32_t pairs = pr.pair_ch, c = chunk, v = c < pairs ? c : 2 * (c - pairs) + t;
    stage = v % NS;
    phase = v / NS + (c < pairs ? 0 : (pairs + NS - 1 - stage) / NS);
  };

  if (warp == 10) {
    // ---- producer: K and V chunks through the page tables, one box per page and column block ----
    const int page = 1 << a.shift, pg_rows = min(page, KV_CHUNK);
    struct Cursor {
      int seg, end, j, chunk;
    };
    Cursor c = {0, pr.nseg[0], 0, 0}, other = {pr.npair, pr.nseg[1], 0, pr.pair_ch};  // of lane t, of the other lane
    bool ok = true, waited = false;
    uint32_t issued = 0, parity = 0;  // per ring slot (K stages, then V stages): a copy was issued, its phase's parity
    int t = 0;
    auto swap = [&] {
      const Cursor x = c;
      c = other;
      other = x;
      t ^= 1;
    };
    while (ok && (c.seg < c.end || other.seg < other.end)) {
      if (c.seg >= c.end) swap();
      const KvSeg& s = seg_of(t, c.seg);
      if (!waited && s.causal != INT_MAX) {  // the block's own K/V rows; what was cached before is there already
        pdl_wait();
        waited = true;
      }
      const int pc = s.p0 + c.j * KV_CHUNK;
      const int npg = (min(KV_CHUNK, s.p1 - pc) + pg_rows - 1) / pg_rows;
      const int i = lane / CB, cb = lane - i * CB;
      const int pid = i < npg ? a.tables[s.tab + ((pc + i * pg_rows) >> a.shift)] : 0;
      const int y = ((s.kv_head * a.num_pages + pid) << a.shift) + (pc & (page - 1));
      int st;
      uint32_t ph;
      ring(c.chunk, t, st, ph);
      const uint32_t off = (uint32_t)st * SM::kChunk + cb * BLK + (uint32_t)(i * pg_rows) * 128u;
#pragma unroll
      for (int kv = 0; kv < 2; kv++) {
        uint64_t* full = kv ? &v_full[st] : &k_full[st];
        uint64_t* empty = kv ? &v_empty[st] : &k_empty[st];
        if (ph > 0) ok = ok && kv_wait(empty, (ph - 1) & 1, &s_abort);
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
      if (c.chunk > pr.pair_ch) swap();  // lane 0's pair chunks, then the lanes' own in turn
    }
    if (!ok) {  // copies in flight land before the CTA leaves
      int never = 0;
      for (int s = 0; s < 2 * NS; s++)
        if (issued >> s & 1) (void)kv_wait(s < NS ? &k_full[s] : &v_full[s - NS], parity >> s & 1, &never);
    }
  } else if (warp >= 8) {
    // ---- MMA issuer of lane t (the whole warp runs it, one lane issues) ----
    const int t = warp - 8, nseg = pr.nseg[t];
    pdl_wait();  // the query operand
    if (nseg > 0) {
      const uint32_t lead = kv_elect();
      const uint32_t sq = smem + SM::kQ + t * SM::kTile;
      const uint32_t t_s = tmem + t * 128, t_o = tmem + COL_O + t * HD;
      // Query tiles: segment i's may be loaded once the S products of the segment before it are done, or, when
      // both are short and in different halves of the tile, those of the one before that (the MMA reads
      // the other half's rows too, whatever they hold: no row's result depends on another row).
      int loaded = 0;
      auto load_ahead = [&](int i) {  // segments before i are done with their query tiles
#pragma unroll 1
        while (loaded < nseg && loaded <= i + 1) {
          const KvSeg& s = seg_of(t, loaded);
          const bool half = s.nrows <= KV_TILE / 2;
          if (loaded == i + 1) {
            const KvSeg& before = seg_of(t, i);
            if (!half || before.nrows > KV_TILE / 2 || before.shift == s.shift) break;
          }
          uint64_t* bar = &q_full[t][loaded & 1];
          if (lead) {
            tc::mbar_expect_tx(bar, half ? SM::kTile / 2 : SM::kTile);
#pragma unroll 1
            for (int cb = 0; cb < CB; cb++) kv_tma2d(sq + cb * QBLK + s.shift * 128u, half ? &qhalf : &qmap, cb * 64, s.qrow, bar);
          }
          __syncwarp();
          loaded++;
        }
      };
      // Half chunks in order, S of number sn, P V of number pn. S may run two ahead: into the buffer of number
      // sn - 2, once the P V that reads that one's P is done. A P V never waits for the operands of a later S:
      // these may be behind the stage that the P V frees. The softmax warps wait for this loop: what holds for
      // a chunk or a segment is kept in registers.
      int sn = 0, sseg = 0, schunk = 0, sleft = seg_of(t, 0).p1 - seg_of(t, 0).p0, sst, sh = 0;  // left: positions of the segment from here on
      int pn = 0, pseg = 0, pchunk = 0, pleft = sleft, pst, ph = 0;
      uint32_t sphase, pphase;
      bool snew = true, pnew = true, ready = false;  // at a segment's start; S's operands are there
      ring(0, t, sst, sphase);
      ring(0, t, pst, pphase);
      load_ahead(0);
      bool ok = true;
      uint32_t spins = 0;
#pragma unroll 1
      while (pseg < nseg) {
        if (sseg < nseg && sn < pn + 2) {
          uint64_t* const qb = &q_full[t][sseg & 1];
          if (!ready) {
            if (sn == pn) {
              ok = (!snew || kv_wait(qb, (sseg >> 1) & 1, &s_abort)) && kv_wait(&k_full[sst], sphase & 1, &s_abort);
              if (!__all_sync(0xffffffffu, ok)) break;
              ready = true;
            } else {
              ready = !snew || (loaded > sseg && tc::mbar_poll(qb, (sseg >> 1) & 1));
              ready = __all_sync(0xffffffffu, ready && tc::mbar_poll(&k_full[sst], sphase & 1));
            }
          }
          if (ready) {
            ok = sn < 2 || kv_wait(&pv_done[t][sn & 1], ((sn - 2) >> 1) & 1, &s_abort);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc::fence_after();
            const uint32_t a0 = kv_desc(sq, 16), b0 = kv_desc(smem + SM::kK + sst * SM::kChunk + sh * (KV_HALF * 128), 16);
            const uint32_t id = kv_idesc<BF16>(0, false) | (uint32_t)(min(KV_HALF, (sleft + 31) & ~31) >> 3) << 17;
#pragma unroll
            for (int k = 0; k < HD / 16; k++)
              kv_mma_ss(lead, t_s + (sn & 1) * KV_HALF, a0 + (((k >> 2) * QBLK + (k & 3) * 32u) >> 4),
                        b0 + (((k >> 2) * BLK + (k & 3) * 32u) >> 4), id, k > 0);
            kv_commit(lead, &s_full[t][sn & 1]);
            sn++;
            sleft -= KV_HALF;
            snew = sleft <= 0;
            if (snew || sh) {  // the chunk's last
              kv_commit(lead, &k_empty[sst]);
              if (schunk >= pr.pair_ch && lead) tc::mbar_arrive(&k_empty[sst]);
              sh = 0;
              ready = false;
              ring(++schunk, t, sst, sphase);
              if (snew && ++sseg < nseg) sleft = seg_of(t, sseg).p1 - seg_of(t, sseg).p0;
            } else {
              sh = 1;
            }
            spins = 0;
            continue;
          }
          // the S is still to come: take the P V if that is ready
          if (!__all_sync(0xffffffffu, tc::mbar_poll(&p_full[t][pn & 1], (pn >> 1) & 1))) {
            ok = ++spins < (1u << 24) && ((spins & 63) || !*(volatile int*)&s_abort);
            if (!__all_sync(0xffffffffu, ok)) {
              s_abort = 1;
              ok = false;
              break;
            }
            continue;
          }
        }
        ok = ph || kv_wait(&v_full[pst], pphase & 1, &s_abort);
        if (pnew && pseg > 0) ok = ok && kv_wait(&o_free[t], (pseg - 1) & 1, &s_abort);
        ok = ok && kv_wait(&p_full[t][pn & 1], (pn >> 1) & 1, &s_abort);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc::fence_after();
        const uint32_t b0 = kv_desc(smem + SM::kV + pst * SM::kChunk + ph * (KV_HALF * 128), BLK);
        const uint32_t tp = t_s + (pn & 1) * KV_HALF;
#pragma unroll
        for (int k = 0; k < KV_HALF / 16; k++)
          if (k < 2 || pleft > 32) kv_mma_ts(lead, t_o, tp + k * 8, b0 + k * (2048u >> 4), kv_idesc<BF16>(HD, true), !pnew || k > 0);
        kv_commit(lead, &pv_done[t][pn & 1]);
        pn++;
        pleft -= KV_HALF;
        pnew = pleft <= 0;
        if (pnew || ph) {
          kv_commit(lead, &v_empty[pst]);
          if (pchunk >= pr.pair_ch && lead) tc::mbar_arrive(&v_empty[pst]);
          ph = 0;
          ring(++pchunk, t, pst, pphase);
          if (pnew && ++pseg < nseg) {
            pleft = seg_of(t, pseg).p1 - seg_of(t, pseg).p0;
            load_ahead(pseg);
          }
        } else {
          ph = 1;
        }
        spins = 0;
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {  // the query tiles in flight land, the MMAs in flight end
        int never = 0;
        for (int i = max(0, loaded - 2); i < loaded; i++) (void)kv_wait(&q_full[t][i & 1], (i >> 1) & 1, &never);
        uint64_t* bar = &q_full[t][loaded & 1];
        kv_commit(lead, bar);
        (void)kv_wait(bar, (loaded >> 1) & 1, &never);
      }
    }
  } else {
    // ---- softmax of lane t: one query row per thread ----
    pdl_wait();  // the sequences' flags, cleared
    const int t = warp >> 2, quad = warp & 3;
    const uint32_t at = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t t_o = at + COL_O + t * HD;
    const float cs = 1.4426950408889634f / sqrtf((float)HD);
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      const bool done = __all_sync(0xffffffffu, kv_wait(bar, parity, &s_abort));
      tc::fence_after();
      return done;
    };
    auto arrive = [&](uint64_t* bar) {
      tc::fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(bar);
    };
    int chunk = 0, n = 0;  // n: the lane's half chunk
    bool ok = true;
#pragma unroll 1
    for (int i = 0; ok && i < pr.nseg[t]; i++) {
      const KvSeg& sg = seg_of(t, i);
      const int p0 = sg.p0, p1 = sg.p1, causal = sg.causal;
      const int row = quad * 32 + lane - sg.shift;
      const bool row_ok = row >= 0 && row < sg.nrows;
      const bool active = quad * 32 >= sg.shift && quad * 32 < sg.shift + sg.nrows;  // warp-uniform
      // last position the row sees, and the last that all of the warp's rows see
      int lim = p1 - 1, seen = p1 - 1;
      if (causal != INT_MAX) {
        if (row_ok) lim = min(lim, causal + (sg.trow0 + row) / a.G);
        seen = min(seen, causal + (sg.trow0 + max(0, quad * 32 - sg.shift)) / a.G);
      }
      float m_ref = -CUDART_INF_F, l = 0.f;
#pragma unroll 1
      for (int pc = p0; pc < p1; pc += KV_HALF, n++) {
        const int half = (pc - p0) & KV_HALF;
        const int ncol = min(KV_HALF, (p1 - pc + 31) & ~31);  // columns of S and P that the MMAs use
        const uint32_t t_s = at + t * 128 + (n & 1) * KV_HALF;
        ok = wait(&s_full[t][n & 1], (n >> 1) & 1);
        if (!ok) break;
        float x[KV_HALF];  // the row's scores
        float mb = 0.f;
        if (active) {
#pragma unroll
          for (int q = 0; q < 2; q++) kv_ld32(t_s + q * 32, x + q * 32);
#pragma unroll
          for (int q = 0; q < 2; q++) kv_wait32(x + q * 32);
          if (pc + KV_HALF - 1 > seen) {  // -inf into the columns that the row does not see
            const int vis = lim - pc;
#pragma unroll
            for (int c = 0; c < KV_HALF; c++) x[c] = c <= vis ? x[c] : -CUDART_INF_F;
          }
          float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
          for (int c = 0; c < KV_HALF; c += 2) mx[(c >> 1) & 3] = kv_max3_nan(mx[(c >> 1) & 3], x[c], x[c + 1]);
          const float m_new = kv_max_nan(kv_max_nan(mx[0], mx[1]), kv_max_nan(mx[2], mx[3])) * cs;  // NaN if one score is
          if (pc == p0) {
            m_ref = m_new;
          } else if (const bool grow = row_ok && !(m_new <= m_ref + KV_RESCALE); __any_sync(0xffffffffu, grow)) {
            // O and l to the new maximum, once the last P V has been added (of the rows that it has grown in
            // alone: what a row comes to does not depend on the others of its tile)
            ok = wait(&pv_done[t][(n - 1) & 1], ((n - 1) >> 1) & 1);
            if (!ok) break;
            const float m2 = grow ? kv_max_nan(m_ref, m_new) : m_ref;
            const float f = grow ? kv_ex2(m_ref - m2) : 1.f;
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
          // the exponents' base: 0 for a row that has seen nothing yet, NaN (and so the row's weights) for a
          // maximum that is infinite or NaN
          mb = m_ref == -CUDART_INF_F ? 0.f : m_ref + (m_ref - m_ref);
        }
        // V rows that nobody sees (past the range) are zeroed, and infinities and NaN of rows that
        // only some of the tile see; all four warps take part
        const bool tail = pc + ncol > p1;
        const bool fresh = causal != INT_MAX && p1 > causal + 1 && pc + KV_HALF > causal + 1;
        if (tail || fresh) {
          int st;
          uint32_t ph;
          ring(chunk, t, st, ph);
          ok = wait(&v_full[st], ph & 1);
          if (!ok) break;
          uint8_t* sv = smem_gen + SM::kV + st * SM::kChunk + half * 128;
          const int r1 = min(KV_HALF, p1 - pc);
          const int r0 = fresh ? max(0, causal + 1 - pc) : r1;
#pragma unroll 1
          for (int k = quad * 32 + lane; k < (ncol - r0) * CB * 8; k += 128) {
            const int r = r0 + k / (CB * 8), c = k % (CB * 8);
            uint4* p = reinterpret_cast<uint4*>(sv + (c >> 3) * BLK + r * 128 + (c & 7) * 16);
            if (r >= r1) {
              *p = make_uint4(0, 0, 0, 0);
            } else {
              uint4 v = *p;
              const uint4 n = make_uint4(kv_nonfinite<BF16>(v.x), kv_nonfinite<BF16>(v.y), kv_nonfinite<BF16>(v.z), kv_nonfinite<BF16>(v.w));
              if (n.x | n.y | n.z | n.w) {
                *p = make_uint4(v.x & ~n.x, v.y & ~n.y, v.z & ~n.z, v.w & ~n.w);
                a.flags[sg.flag] = 1;
              }
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        const uint64_t cs2 = kv_f2(cs, cs), mb2 = kv_f2(-mb, -mb);
        uint64_t ls[4] = {0, 0, 0, 0};
#pragma unroll
        for (int q = 0; q < 2; q++)
          if (active && q * 32 < ncol) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; e++) {
              const uint64_t z = kv_fma2(kv_f2(x[q * 32 + 2 * e], x[q * 32 + 2 * e + 1]), cs2, mb2);
              float2 w;
              if ((e & 3) == 2) {
                w = kv_ex2_fma<BF16>(z);
              } else {
                w = kv_un2(z);
                w.x = kv_ex2(w.x);
                w.y = kv_ex2(w.y);
              }
              ls[e & 3] = kv_add2(ls[e & 3], kv_f2(w.x, w.y));
              pk[e] = kv_pack<BF16>(w.x, w.y);
            }
            tc::st16(t_s + q * 16, pk);
          }
        if (active) tc::wait_st();
        const float2 lf = kv_un2(kv_add2(kv_add2(ls[0], ls[1]), kv_add2(ls[2], ls[3])));
        l += lf.x + lf.y;
        arrive(&p_full[t][n & 1]);
        if (half || pc + KV_HALF >= p1) chunk++;
      }
      if (!ok) break;
      ok = wait(&pv_done[t][(n - 1) & 1], ((n - 1) >> 1) & 1);
      if (!ok) break;
      if (active) {
        // A warp full of rows: four lanes write 128 bytes of a row together; each has its own row's, so they swap
        // first. (32 bytes a lane and row are whole sectors but no whole lines: 148 CTAs' tiles of 128 KB
        // take 6.2 instead of 4.2 us. With few rows the swaps cost more: two short samples 8.3 against 7.4.)
        const bool full = __all_sync(0xffffffffu, row_ok);
        float* po = a.part + ((size_t)sg.slot + (full ? row & ~3 : row)) * HD + (full ? (lane & 3) * 8 : 0);
        const int next = full ? HD : 8;  // from one 32-byte piece to the next
#pragma unroll 1
        for (int q = 0; q < HD / 32; q++) {
          float o[32];
          kv_ld32(t_o + q * 32, o);
          kv_wait32(o);
          if (full)
#pragma unroll
            for (int b = 1; b <= 2; b <<= 1)
#pragma unroll
              for (int c = 0; c < 4; c++)
                if (!(c & b))
#pragma unroll
                  for (int e = 0; e < 8; e++) {
                    float &lo = o[c * 8 + e], &hi = o[(c + b) * 8 + e];
                    const float got = __shfl_xor_sync(0xffffffffu, lane & b ? lo : hi, b);
                    if (lane & b)
                      lo = got;
                    else
                      hi = got;
                  }
          if (row_ok)
#pragma unroll
            for (int e = 0; e < 4; e++) kv_st8(po + q * 32 + e * next, o + 8 * e);
        }
        if (row_ok) reinterpret_cast<float2*>(a.part + (size_t)h.nslots * HD)[sg.slot + row] = make_float2(m_ref, l);
      }
      arrive(&o_free[t]);
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

// A query row's partials: their maximum, then their weighted sum, in plan order (the result does not
// depend on timing). A group of hd / 4 threads per row and head, 16 bytes of a partial each, or, when the plan
// says so (few rows, some with many partials), the block's groups together, each with every NG-th of them
// (SPLIT). Bound by L2's latency when there are few rows (sequence, units, then the maxima and four
// partials at once: three round trips, 3.7 us), by L2's bandwidth when there are many (4608 rows with 10
// partials of 512 bytes: 6.5 us). A whole warp per row at hd 64 too: 14.5 against 9.5 us for 64 x 32 rows
// of 14 heads. Eight partials in flight take registers, and so warps, away: 288 rows of 16 heads 9.0 against
// 8.2 us, 1024 rows of 14 heads 12.1 against 10.8; so does a kernel not held to 64 registers (22.1
// against 23.4 us for the three launches at 4608 rows). BT: f16 in the batched GEMM's operand layout.
template <int HD, bool BF16, bool BT, bool SPLIT>
__device__ __forceinline__ void kv_merge(const KvArgs& a, float (*s_acc)[HD], float2* s_ml) {
  constexpr int L = HD / 4, NG = 128 / L, PER = 32 / L, U = 4;  // lanes of a group, groups of a block and a warp; partials in flight
  const KvSeq* sqs = reinterpret_cast<const KvSeq*>(a.plan + KV_SEQ_AT);
  const KvHdr& h = *reinterpret_cast<const KvHdr*>(a.plan);
  const KvUnit* units = reinterpret_cast<const KvUnit*>(a.plan + h.off_unit);
  const int lane = threadIdx.x & (L - 1), grp = threadIdx.x / L, warp = threadIdx.x >> 5;
  const int G = a.G, kvh = a.kv_heads, H = G * kvh, M = a.M;
  const float2* pml = reinterpret_cast<const float2*>(a.part + (size_t)h.nslots * HD);
  constexpr int ks = SPLIT ? NG : 1;
  const int k0 = SPLIT ? grp : 0, sub = SPLIT ? 0 : grp % PER;
  const int items = a.rows * H, step = SPLIT ? gridDim.x : gridDim.x * NG;
  for (int it = SPLIT ? blockIdx.x : blockIdx.x * NG + warp * PER; it < items; it += step) {
    const int item = min(it + sub, items - 1);
    const int orow = item / H, head = item - orow * H, s = orow / M, t = orow - s * M;
    const KvSeq& q = sqs[s];
    const bool valid = it + sub < items && t < q.cnt;
    if ((SPLIT || PER == 1) && !valid) continue;  // (the groups of a warp stay together)
    const int g = head / G, row = q.row0 + t * G + (head - g * G);
    // the partials of the row's ranges in order: entry i's slot, and how many there are
    auto entry = [&](int i, int& n) {  // (not kept in registers for the few rows with more than L)
      int slot = 0;
      n = 0;
#pragma unroll
      for (int l = 0; l < KV_LEVELS; l++)
        if (l < q.nlev) {
          const int lr = row - q.lrow0[l];
          const KvUnit u = units[q.lunit[l] + g * q.ltile[l] + lr / KV_TILE];
          if (i >= n && i - n < u.nseg) slot = u.base + lr % KV_TILE + (i - n) * u.nrows;
          n += u.nseg;
        }
      return slot;
    };
    // the group's entries: k0, k0 + ks, .. ; lane i holds the weight of the i-th
    int n = 0, slot = 0, again;
    if (valid) {
      slot = entry(k0 + ks * lane, n);
      n = (n - k0 + ks - 1) / ks;
    }
    const int nmax = PER == 1 ? n : max(n, __shfl_xor_sync(0xffffffffu, n, 16));
    pdl_wait();
    const float2 none = make_float2(-CUDART_INF_F, 0.f);
    float2 ml = lane < n ? pml[slot] : none;
    const int flag = valid && t > 0 ? a.flags[s * kvh + g] : 0;
    float4 v[U];
    auto load = [&](int k) {  // entries k .. k + U of the L whose slots the lanes hold
#pragma unroll
      for (int e = 0; e < U; e++) {
        const int sl = __shfl_sync(0xffffffffu, slot, (k + e) & (L - 1), L);
        if (k + e < n) v[e] = *reinterpret_cast<const float4*>(a.part + (size_t)sl * HD + lane * 4);
      }
    };
    load(0);
    float m = ml.x;
#pragma unroll 1
    for (int i = L + lane; i < n; i += L) m = fmaxf(m, pml[entry(k0 + ks * i, again)].x);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int base = 0; base < nmax; base += L) {
      if (base > 0) {
        slot = base + lane < n ? entry(k0 + ks * (base + lane), again) : 0;
        ml = base + lane < n ? pml[slot] : none;
      }
      const float w = ml.x == -CUDART_INF_F ? 0.f : kv_ex2(ml.x - m);
      l += w * ml.y;
#pragma unroll 1
      for (int k = base; k < min(nmax, base + L); k += U) {
        if (k > 0) load(k);
#pragma unroll
        for (int e = 0; e < U; e++) {
          const float wk = __shfl_sync(0xffffffffu, w, (k + e) & (L - 1), L);
          if (k + e < n) {
            acc[0] += wk * v[e].x;
            acc[1] += wk * v[e].y;
            acc[2] += wk * v[e].z;
            acc[3] += wk * v[e].w;
          }
        }
      }
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if constexpr (SPLIT) {
      __syncthreads();  // (the last row's sums have been read)
      *reinterpret_cast<float4*>(&s_acc[grp][lane * 4]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (lane == 0) s_ml[grp] = make_float2(m, l);
      __syncthreads();
      if (warp != 0) continue;
      m = s_ml[0].x;
#pragma unroll
      for (int e = 1; e < NG; e++) m = fmaxf(m, s_ml[e].x);
      l = acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
#pragma unroll
      for (int e = 0; e < NG; e++) {
        const float w = s_ml[e].x == -CUDART_INF_F ? 0.f : kv_ex2(s_ml[e].x - m);
        l += w * s_ml[e].y;
#pragma unroll
        for (int x = 0; x < 4; x++) acc[x] += w * s_acc[e][lane * 4 + x];
      }
    }
    if (!valid || (SPLIT && grp != 0)) continue;
    const float inv = 1.0f / l;
#pragma unroll
    for (int e = 0; e < 4; e++) acc[e] *= inv;
    if (flag) {  // infinities and NaN of the block's own V rows that this row sees
#pragma unroll 1
      for (int tt = 1; tt <= t; tt++) {
        const int pos = q.n + tt;
        const size_t src = ((((size_t)g * a.num_pages + a.tables[q.tab + (pos >> a.shift)]) << a.shift) + (pos & ((1 << a.shift) - 1))) * HD + lane * 4;
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const uint32_t x = *reinterpret_cast<const uint32_t*>(a.v + src + e);
          const uint32_t nf = kv_nonfinite<BF16>(x);
          const float2 f = kv_unpack<BF16>(x);
          if (nf & 0xffffu) acc[e] += f.x;
          if (nf >> 16) acc[e + 1] += f.y;
        }
      }
    }
    uint16_t* out = BT ? a.out + bt_off(orow, head * HD + lane * 4, H * HD, a.out_bt_n) : a.out + (size_t)orow * a.out_stride + (size_t)head * HD + lane * 4;
    *reinterpret_cast<uint2*>(out) = make_uint2(kv_pack<BF16>(acc[0], acc[1]), kv_pack<BF16>(acc[2], acc[3]));
  }
}
template <int HD, bool BF16, bool BT>
__global__ void __launch_bounds__(128, 8) kv_merge_kernel(const KvArgs a) {
  __shared__ __align__(16) float s_acc[512 / HD][HD];
  __shared__ float2 s_ml[512 / HD];
  pdl_trigger();
  if (reinterpret_cast<const KvHdr*>(a.plan)->split_rows)
    kv_merge<HD, BF16, BT, true>(a, s_acc, s_ml);
  else
    kv_merge<HD, BF16, BT, false>(a, s_acc, s_ml);
  pdl_wait();  // (a warp without rows: the kernel after this one may rely on the one before it being done)
}

// ---- page copies ------------------------------------------------------------------------------------

// Copies of one launch (they travel in its parameters; few of them in a short list, since parameters cost the
// host time), grouped in runs that share source and rows: a run reads its source once.
constexpr int KV_COPIES = 1024, KV_FEW_COPIES = 64, KV_RUN = 8;
template <int N>
struct KvCopyList {
  int32_t src[N], rows[N];  // of run i
  int32_t first[N];         // its first destination, and (top 8 bits) how many it has
  int32_t dst[N];
};

// Tasks of 4 KB: (run, layer x head, K or V, piece of the page's rows). Every lane has its eight 16-byte loads
// in flight before the first store. Bound by HBM: a byte is read once for a run and written once a copy.
template <int N>
__global__ void __launch_bounds__(256) kv_copy_kernel(const __grid_constant__ KvCopyList<N> list, int n, uint4* __restrict__ k,
                                                      uint4* __restrict__ v, int blocks, int num_pages, int page16, int row16, int pieces) {
  pdl_trigger();
  pdl_wait();
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
    const int end = list.rows[i] * row16;
    const int at = piece * 256 + lane;
    if (piece * 256 >= end) continue;
    uint4* base = (kv ? v : k) + (size_t)b * num_pages * page16;
    const uint4* src = base + (size_t)list.src[i] * page16;
    uint4 r[8];
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (at + e * 32 < end) r[e] = __ldcs(src + at + e * 32);
    const int first = list.first[i] & 0xFFFFFF, last = first + (list.first[i] >> 24);
#pragma unroll 1
    for (int j = first; j < last; j++) {
      uint4* dst = base + (size_t)list.dst[j] * page16;
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (at + e * 32 < end) __stcs(dst + at + e * 32, r[e]);
    }
  }
}

template <int N>
static void launch_copies_t(void* k, void* v, int blocks, int hd, int page, int num_pages, const PageCopy* c, int m, int num_sms, cudaStream_t s) {
  const int row16 = hd / 8;
  KvCopyList<N> list;
  int runs = 0, rows = 0;
  for (int e = 0; e < m; e++) {
    list.dst[e] = c[e].dst;
    if (runs && c[e].src == list.src[runs - 1] && c[e].rows == list.rows[runs - 1] && (list.first[runs - 1] >> 24) < KV_RUN) {
      list.first[runs - 1] += 1 << 24;
      continue;
    }
    list.src[runs] = c[e].src;
    list.rows[runs] = c[e].rows;
    list.first[runs++] = e | 1 << 24;
    rows = std::max(rows, (int)c[e].rows);
  }
  if (rows == 0) return;
  const int pieces = (rows * row16 + 255) / 256;
  const long long tasks = (long long)runs * blocks * 2 * pieces;
  const int grid = (int)std::min<long long>((tasks + 7) / 8, (long long)num_sms * 8);
  launch_pdl(kv_copy_kernel<N>, dim3(grid), dim3(256), 0, s, list, runs, reinterpret_cast<uint4*>(k), reinterpret_cast<uint4*>(v), blocks,
             num_pages, page * row16, row16, pieces);
}

void launch_page_copies(void* k, void* v, int layers, int kv_heads, int hd, int page, int num_pages, const PageCopy* c, size_t n,
                        int num_sms, cudaStream_t s) {
  const int blocks = layers * kv_heads;
  if (n <= KV_FEW_COPIES) return launch_copies_t<KV_FEW_COPIES>(k, v, blocks, hd, page, num_pages, c, (int)n, num_sms, s);
  for (size_t i = 0; i < n; i += KV_COPIES)
    launch_copies_t<KV_COPIES>(k, v, blocks, hd, page, num_pages, c + i, (int)std::min<size_t>(KV_COPIES, n - i), num_sms, s);
}

// The staged parts of a step (host memory that the device reads): block i < n, a run of page-table entries; the
// others, the plan. What a thread moves first crosses the bus while the kernels before still run.
__global__ void __launch_bounds__(256) kv_stage_kernel(int32_t* __restrict__ table, const KvRange* __restrict__ ranges, int n,
                                                       uint4* __restrict__ plan, const uint4* __restrict__ staged, int plan16) {
  pdl_trigger();
  if (blockIdx.x < n) {
    const KvRange r = ranges[blockIdx.x];
    const int32_t* vals = reinterpret_cast<const int32_t*>(ranges + n) + r.from;
    int i = threadIdx.x;
    int32_t v = i < r.n ? vals[i] : 0;
    pdl_wait();
    for (; i < r.n; i += 256, v = i < r.n ? vals[i] : 0) table[r.at + i] = v;
  } else {
    const int step = (gridDim.x - n) * 256;
    int i = (blockIdx.x - n) * 256 + threadIdx.x;
    uint4 v = staged[min(i, plan16 - 1)];
    pdl_wait();
    for (; i < plan16; i += step, v = staged[min(i, plan16 - 1)]) plan[i] = v;
  }
}

void launch_stage(int32_t* table, const KvRange* ranges, int nranges, void* plan, const void* staged, size_t plan_bytes, cudaStream_t s) {
  const int plan16 = (int)(plan_bytes / 16);
  launch_pdl(kv_stage_kernel, dim3(nranges + std::min(64, (plan16 + 255) / 256)), dim3(256), 0, s, table, ranges, nranges,
             static_cast<uint4*>(plan), static_cast<const uint4*>(staged), plan16);
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

void KvWork::open(const KvGeom& geom, bool is_bf16, int* err_word, cudaStream_t s) {
  g = geom;
  bf16 = is_bf16;
  err = err_word;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const size_t qrows = g.rows_cap() * g.kv_heads;
  const size_t bp = up(g.plan_cap()), bq = up(qrows * g.hd * 2), bo = up(g.slots_cap() * (g.hd + 2) * 4), bf = up((size_t)g.nseq * g.kv_heads * 4);
  LS_CUDA(cudaMalloc(&mem, bp + bq + bo + bf));
  try {
    uint8_t* p = reinterpret_cast<uint8_t*>(mem);
    plan = p;
    q = p + bp;
    part = reinterpret_cast<float*>(p + bp + bq);
    flags = reinterpret_cast<int*>(p + bp + bq + bo);
    // the query operand's rows past the block's are read into tiles (and never used): finite from the start. In the
    // order of the stream that uses them first: cudaMemset's is the legacy stream, which a non-blocking one passes.
    LS_CUDA(cudaMemsetAsync(q, 0, bq, s));
    LS_CUDA(cudaMemsetAsync(flags, 0, bf, s));
    kv_encode_map(&qmap, q, qrows, g.hd, KV_TILE, bf16);
    kv_encode_map(&qmap_half, q, qrows, g.hd, KV_TILE / 2, bf16);
  } catch (...) {  // (mem says whether this is open)
    close();
    throw;
  }
}

void KvWork::close() {
  if (mem) cudaFree(mem);
  mem = nullptr;
}

template <int HD, bool BF16>
static void launch_kv_t(const KvWork& w, const KvAttn& a, const KvArgs& k, cudaStream_t s) {
  const int units = (w.g.heads + 2 * w.g.kv_heads) * (HD / 16);
  const size_t pieces = (size_t)a.rows * units;
  const int gp = (int)std::min<size_t>((pieces + 255) / 256, (size_t)w.g.nctas * 8);
  if (a.qkv_f32)
    launch_pdl(kv_prep_kernel<BF16, true>, dim3(gp), dim3(256), 0, s, k);
  else
    launch_pdl(kv_prep_kernel<BF16, false>, dim3(gp), dim3(256), 0, s, k);
  const size_t smem = KvSmem<HD>::kTotal;
  ensure_smem(kv_attn_kernel<HD, BF16>, smem);
  launch_pdl(kv_attn_kernel<HD, BF16>, dim3(w.g.nctas), dim3(KV_THREADS), smem, s, k, w.qmap, w.qmap_half, *a.kmap, *a.vmap);
  // hd / 4 threads per row and head, or a block for each of as many as the plan may split
  const size_t items = (size_t)a.rows * w.g.heads, per = 512 / HD;
  const int gm = (int)std::min(std::max((items + per - 1) / per, std::min(items, (size_t)w.g.nctas * KV_SPLIT_ITEMS)), (size_t)w.g.nctas * 16);
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
  k.rows = a.rows;
  k.M = a.M;
  if (w.g.hd == 64) return w.bf16 ? launch_kv_t<64, true>(w, a, k, s) : launch_kv_t<64, false>(w, a, k, s);
  return w.bf16 ? launch_kv_t<128, true>(w, a, k, s) : launch_kv_t<128, false>(w, a, k, s);
}

}  // namespace ls
