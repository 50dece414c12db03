// A paged K/V cache whose sequences share pages: page bookkeeping (counts, copy on write) and the
// host side of attention over shared pages (which rows read which positions, on which CTA).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include <string>
#include <utility>
#include <vector>

#include "ls_internal.h"

namespace ls {

// ---- page copies -------------------------------------------------------------------------------

struct PageCopy {
  int32_t src, dst, rows;  // rows [0, rows) of page src to page dst, in every layer and kv head
};
// Copies between pages of K and V pools [layers][kv_heads][num_pages][page][hd] of 2-byte elements.
// Destinations are distinct and no page is both a source and a destination (the caller has checked).
void launch_page_copies(void* k, void* v, int layers, int kv_heads, int hd, int page, int num_pages, const PageCopy* c, size_t n,
                        int num_sms, cudaStream_t s);

// Runs of page-table entries: table[at .. at + n) = values[from .. from + n), values behind the ranges.
struct KvRange {
  int32_t at, from, n, pad;
};
// The entries and the plan out of host memory that the device can read (plan_bytes a multiple of 16).
void launch_stage(int32_t* table, const KvRange* ranges, int nranges, void* plan, const void* staged, size_t plan_bytes, cudaStream_t s);

// ---- attention over shared pages: the plan ------------------------------------------------------
//
// The rows of one kv head's query operand are ordered (sequence in plan order, block row t, head of the
// group j). A NODE is a range of positions [a, b) that a run of consecutive rows reads through one
// page table: a prefix shared by several sequences, or one sequence's own positions. A UNIT is one
// 128-row tile of a node for one kv head; it is cut into SEGMENTS of whole 128-position chunks, each
// worked by one lane of one CTA and leaving (m, l, O) partials for its rows. Every CTA has two lanes
// (two tensor-memory tiles): first its pair segments, where the lanes hold two adjacent tiles that
// read the same chunks, then each lane's own.

constexpr int KV_TILE = 128;    // query rows of a tile
constexpr int KV_CHUNK = 128;   // positions of a chunk
constexpr int KV_SPLIT_ITEMS = 8;  // rows x heads per SM up to which the merge may take a block for each
constexpr int KV_LEVELS = 3;    // nodes on a row's path: two shared ranges at most, then its own

struct KvSeg {
  int32_t qrow;     // the tile's first row in the query operand
  int32_t nrows;    // its valid rows
  int32_t tab;      // offset of the page table its positions are read through
  int32_t kv_head;
  int32_t p0, p1;   // positions [p0, p1), p0 a multiple of the page or of the chunk inside one
  int32_t nch;
  int32_t causal;   // row r sees positions <= causal + (trow0 + r) / G; INT_MAX: all of them
  int32_t trow0;    // the tile's first row, counted from its sequence's first
  int32_t slot;     // partial row of the tile's first row
  int32_t flag;     // sequence * kv_heads + kv head (its own positions), -1 for a shared range
  int32_t shift;    // tensor-memory lane of the tile's first row: 0, or 64 for every other short tile of a lane
  int32_t unit;     // its unit
  int32_t pad[3];
};
struct KvProg {  // one CTA's program
  int32_t seg[2];   // first segment of each lane
  int32_t nseg[2];  // its segments, pair segments first
  int32_t npair;    // pair segments
  int32_t pair_ch;  // their chunks
  int32_t pad[2];
};
struct KvSeq {
  int32_t n, cnt;   // cached positions, rows of the block
  int32_t row0;     // first row in a kv head's query operand
  int32_t tab;      // offset of its page table
  int32_t nlev;     // nodes on its path; each one's first row, tiles, first unit:
  int32_t lrow0[KV_LEVELS], ltile[KV_LEVELS], lunit[KV_LEVELS];  // unit of (kv head g, tile i) = lunit + g * ltile + i
  int32_t pad[2];
};
struct KvUnit {     // a tile's partials: segment k's of its row r in partial row base + k * nrows + r
  int32_t base, nseg, nrows, pad;
};
struct KvHdr {
  int32_t M, nseq, R, max_pages;  // R: rows of a kv head's query operand
  int32_t off_prog, off_seg, off_unit;  // byte offsets in the plan (the sequences stand at KV_SEQ_AT)
  int32_t nslots, split_rows;  // split_rows: few rows, some with many partials (kv_merge_kernel)
  int32_t pad[3];
};
constexpr int KV_SEQ_AT = sizeof(KvHdr);  // where the plan's sequences stand: read without the header
static_assert(KV_SEQ_AT % 16 == 0, "plan sections start on 16 bytes");

struct KvGeom {
  int heads = 0, kv_heads = 0, hd = 0, shift = 6, num_pages = 0, max_pages = 0, nseq = 0, max_rows = 0, nctas = 148;
  int G() const { return heads / kv_heads; }
  int page() const { return 1 << shift; }
  size_t rows_cap() const { return (size_t)max_rows * G(); }  // rows of one kv head
  size_t units_cap() const { return (size_t)kv_heads * (KV_LEVELS * (rows_cap() / KV_TILE) + 2 * (size_t)nseq); }
  size_t segs_cap() const { return units_cap() + 4 * (size_t)nctas; }
  size_t slots_cap() const { return (size_t)kv_heads * KV_LEVELS * rows_cap() + 3 * (size_t)KV_TILE * nctas; }
  size_t plan_cap() const;
};

// One sequence as the planner sees it: n cached positions, cnt new rows, its page table.
struct KvSeqIn {
  int n = 0, cnt = 0;
  const int32_t* table = nullptr;
  int tab = 0;
};

class KvPlanner {
 public:
  KvGeom g;
  std::vector<uint8_t> bytes;  // the packed plan (KvHdr first)
  // version: changes whenever a page table changed other than by growing at its end (the sharing
  // tree of the last plan is kept while version and every sequence's class, by its rows, stay the same).
  void build(const std::vector<KvSeqIn>& seqs, int M, uint64_t version);
  // Throws unless the plan covers every row's positions exactly once, stays inside its bounds and loads the CTAs evenly.
  void check(const std::vector<KvSeqIn>& seqs) const;
  size_t shared_positions() const { return shared_pos_; }  // positions read for several sequences at once

 private:
  struct Node {
    int a, b;            // positions
    int first, last;     // sequences [first, last) in plan order
    int tab;
    bool own;
  };
  struct Job {
    int node, g, tile, ntiles, nch, p1;
  };
  static double start_of(const Job& j), chunk_of(const Job& j);  // costs (ls_kv_plan.cpp)
  struct Piece {
    int cta, job, c0, nch;
  };
  std::vector<int> order_;   // sequences with rows, in plan order
  std::vector<Node> shared_; // shared ranges
  enum Class : uint8_t { IDLE, GROUPED, ALONE };  // no rows; planned with those that share its pages; by itself
  std::vector<Class> class_;
  uint64_t version_ = ~0ull;
  size_t shared_pos_ = 0;
  std::vector<Node> nodes_;
  struct DNode {
    int row0, ntile, unit0;
  };
  std::vector<DNode> dnodes_;
  std::vector<KvSeq> dseqs_;
  std::vector<Job> jobs_;
  std::vector<Piece> pieces_;
  std::vector<KvSeg> segs_, lane_[2];
  std::vector<KvProg> progs_;
  std::vector<KvUnit> units_;
  Class class_of(int cnt) const;
  void tree(const std::vector<KvSeqIn>& seqs);
};

// ---- attention over shared pages: device state and launches ---------------------------------------

struct KvWork {
  KvGeom g;
  bool bf16 = false;
  uint8_t* plan = nullptr;     // device copy of the plan
  void* q = nullptr;           // query operand [kv_heads][R][hd], 16-bit
  float* part = nullptr;       // O partials [slots][hd], then (m, l) [slots][2]
  int* flags = nullptr;        // [nseq * kv_heads]: a new V row holds an infinity or a NaN
  int* err = nullptr;          // device-visible error word (1: a bounded wait gave up)
  CUtensorMap qmap{}, qmap_half{};  // boxes of a tile's rows, of half a tile's
  void* mem = nullptr;         // the allocation behind plan, q, part and flags
  void open(const KvGeom& geom, bool is_bf16, int* err_word, cudaStream_t s);  // on the current device; cleared in s's order
  void close();
};

struct KvAttn {
  const void* qkv = nullptr;  // rows q | k | v, row s * M + t
  size_t qkv_stride = 0;      // elements
  bool qkv_f32 = false;       // f32 rows, else the cache's type
  const float2* rope = nullptr;  // (cos, sin) [position][hd / 2], null: rows are rotated already
  void *k = nullptr, *v = nullptr;  // this layer's pools [kv_heads][num_pages][page][hd]
  const int32_t* tables = nullptr;  // device page tables
  const CUtensorMap *kmap = nullptr, *vmap = nullptr;
  void* out = nullptr;        // rows of the cache's type, row s * M + t
  size_t out_stride = 0;
  uint16_t* out_bt = nullptr; // instead of out: f16 in the batched GEMM's operand layout (groups of out_bt_n rows)
  int out_bt_n = 0;
  int rows = 0, M = 0;        // nseq * M, rows of a sequence
};
void launch_kv_attention(const KvWork& w, const KvAttn& a, cudaStream_t s);
// 2-D tensor map over rows of hd 16-bit elements (64 x box_rows boxes, 128-byte swizzle).
void kv_encode_map(CUtensorMap* m, const void* base, uint64_t rows, int hd, int box_rows, bool bf16);
inline int kv_box_rows(int page) { return page < KV_CHUNK ? page : KV_CHUNK; }

}  // namespace ls
