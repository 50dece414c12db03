// The paged K/V cache object behind ls_kv_*: pages with counts over pools that the caller owns, copies
// on write, and the plan and workspaces of attention over shared pages.
#include <algorithm>
#include <cstring>
#include <memory>
#include <unordered_map>

#include "layerstream.h"
#include "ls_kv.h"

using namespace ls;

namespace {

// Makes `device` current for a call and the caller's device again after it.
struct OnDevice {
  int before = -1;
  bool back = false;
  explicit OnDevice(int device) {
    if (device < 0) return;
    LS_CUDA(cudaGetDevice(&before));
    if (before != device) {
      LS_CUDA(cudaSetDevice(device));
      back = true;
    }
  }
  ~OnDevice() {
    if (back) cudaSetDevice(before);
  }
};

constexpr size_t kMaxSeqs = 4096, kMaxRows = 65536;

void check_pool(uint64_t layers, uint64_t kv_heads, uint64_t hd, uint64_t page, uint64_t num_pages) {
  if (layers == 0 || layers > 1024 || kv_heads == 0 || kv_heads > 1024) LS_THROW(LS_ERR_ARG, "layers and kv_heads must be in 1..1024");
  if (hd == 0 || hd % 8 || hd > 1024) LS_THROW(LS_ERR_ARG, "the head size must be a multiple of 8, at most 1024");
  if (page < 8 || page > 65536 || (page & (page - 1))) LS_THROW(LS_ERR_ARG, "the page must be a power of two in 8..65536");
  if (num_pages == 0 || num_pages > (1u << 30) || kv_heads * num_pages * page > 0x7fffffffull)
    LS_THROW(LS_ERR_ARG, "a layer's pool must hold 1..2^31-1 rows (kv_heads x num_pages x page)");
}

void check_aligned(const void* p, const char* what) {
  if (reinterpret_cast<uintptr_t>(p) & 15) LS_THROW(LS_ERR_ARG, std::string(what) + " must be 16-byte aligned");
}

bool capturing(cudaStream_t s) {
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  LS_CUDA(cudaStreamIsCapturing(s, &st));
  return st != cudaStreamCaptureStatusNone;
}

// The GPU whose memory p is.
int device_of(const void* p, const char* what) {
  cudaPointerAttributes a{};
  LS_CUDA(cudaPointerGetAttributes(&a, p));
  if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) LS_THROW(LS_ERR_ARG, std::string(what) + " is not device memory");
  return a.device;
}

int num_sms(int device) {
  int n = 148;
  if (device >= 0) LS_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device));
  return n;
}

}  // namespace

struct LsKv {
  int device = -1;  // -1: page bookkeeping alone, no GPU
  KvGeom g;
  size_t layers = 0, max_ctx = 0;
  bool bf16 = false;
  uint8_t *k = nullptr, *v = nullptr;  // the caller's pools
  size_t layer_bytes = 0;
  std::vector<CUtensorMap> maps;       // [layers] K, [layers] V
  KvWork work;
  KvPlanner planner;
  // pages
  std::vector<int32_t> ref;            // sequences holding each page
  int lowest = 0;                      // no page below this is free
  int nfree = 0;
  std::vector<int32_t> table;          // [nseq][max_pages]
  std::vector<int> held;               // logical pages of each sequence
  std::vector<int> len;                // cached positions
  std::vector<int> counts;             // rows of the begun step
  bool begun = false;
  uint64_t version = 0;
  // device tables, and the parts of them that changed since the last begin
  int32_t* d_table = nullptr;
  std::vector<std::pair<int, int>> dirty;  // [first, last) logical pages per sequence
  // staging: pinned buffers taken in turn, an event behind each upload
  struct Stage {
    uint8_t *p = nullptr, *d = nullptr;  // host and device address
    size_t cap = 0;
    cudaEvent_t done = nullptr;
  } stage[2];
  int turn = 0;
  int *h_err = nullptr, *d_err = nullptr;  // error word, mapped
  std::vector<PageCopy> copies;
  bool inject_fail = false;  // test hook: the next step's launches fail

  LsKv() = default;
  LsKv(const LsKv&) = delete;
  ~LsKv() {
    if (device < 0) return;
    int before = -1;
    if (cudaGetDevice(&before) != cudaSuccess) before = -1;
    cudaSetDevice(device);
    cudaDeviceSynchronize();  // the workspaces may still be in use
    work.close();
    if (d_table) cudaFree(d_table);
    for (Stage& s : stage) {
      if (s.p) cudaFreeHost(s.p);
      if (s.done) cudaEventDestroy(s.done);
    }
    if (h_err) cudaFreeHost(h_err);
    if (before >= 0 && before != device) cudaSetDevice(before);
  }

  int32_t* row(int s) { return table.data() + (size_t)s * g.max_pages; }
  const int32_t* row(int s) const { return table.data() + (size_t)s * g.max_pages; }
  int pages_of(size_t n) const { return (int)((n + g.page() - 1) >> g.shift); }
  void touch(int s, int first, int last) {
    if (first >= last) return;
    auto& d = dirty[s];
    d = d.first >= d.second ? std::make_pair(first, last) : std::make_pair(std::min(d.first, first), std::max(d.second, last));
  }
  int take() {
    while (ref[lowest]) lowest++;
    nfree--;
    ref[lowest] = 1;
    return lowest++;
  }
  void drop(int p) {
    if (--ref[p] == 0) {
      nfree++;
      lowest = std::min(lowest, p);
    }
  }
  void check_seq(uint64_t s) const {
    if (s >= (uint64_t)g.nseq) LS_THROW(LS_ERR_ARG, "sequence " + std::to_string(s) + " is outside the cache's " + std::to_string(g.nseq));
  }
  void check_err() {
    if (h_err && *reinterpret_cast<volatile int*>(h_err))
      LS_THROW(LS_ERR_DEVICE, "an attention kernel gave up waiting on an mbarrier (bounded wait)");
  }
  void changed() {  // the tables no longer are what the last plan was made for
    begun = false;
    version++;
  }
  void keep_pages(int s, int n) {
    while (held[s] > n) drop(row(s)[--held[s]]);
  }

  void open(int dev, uint64_t layers_, uint64_t heads, uint64_t kv_heads, uint64_t hd, int dtype, uint64_t page, uint64_t num_pages,
            uint64_t seqs, uint64_t ctx, uint64_t max_rows, void* k_pool, void* v_pool) {
    check_pool(layers_, kv_heads, hd, page, num_pages);
    if (hd != 64 && hd != 128) LS_THROW(LS_ERR_ARG, "attention over shared pages takes head sizes 64 and 128");
    if (heads == 0 || heads > 1024 || heads % kv_heads) LS_THROW(LS_ERR_ARG, "heads must be a multiple of kv_heads, at most 1024");
    if (dtype != LS_KV_F16 && dtype != LS_KV_BF16) LS_THROW(LS_ERR_ARG, "the cache's type must be LS_KV_F16 or LS_KV_BF16");
    if (seqs == 0 || seqs > kMaxSeqs) LS_THROW(LS_ERR_ARG, "seqs must be in 1..4096");
    if (ctx == 0 || ctx > (1u << 24)) LS_THROW(LS_ERR_ARG, "max_ctx must be in 1..2^24");
    if (max_rows == 0 || max_rows > kMaxRows) LS_THROW(LS_ERR_ARG, "max_rows must be in 1..65536");
    g.heads = (int)heads;
    g.kv_heads = (int)kv_heads;
    g.hd = (int)hd;
    while ((1u << g.shift) != page) g.shift = (1u << g.shift) < page ? g.shift + 1 : g.shift - 1;
    g.num_pages = (int)num_pages;
    g.nseq = (int)seqs;
    g.max_pages = pages_of(ctx);
    g.max_rows = (int)max_rows;
    if ((uint64_t)g.nseq * g.max_pages > 0x7fffffffull) LS_THROW(LS_ERR_ARG, "seqs x pages per sequence exceeds 2^31-1 table entries");
    if ((uint64_t)g.rows_cap() * kv_heads > 0x3fffffffull / KV_LEVELS) LS_THROW(LS_ERR_ARG, "max_rows x heads is too large");
    layers = layers_;
    max_ctx = ctx;
    bf16 = dtype == LS_KV_BF16;
    device = dev;
    g.nctas = num_sms(dev);
    planner.g = g;
    ref.assign(num_pages, 0);
    nfree = g.num_pages;
    table.assign((size_t)g.nseq * g.max_pages, -1);
    held.assign(g.nseq, 0);
    len.assign(g.nseq, 0);
    counts.assign(g.nseq, 0);
    dirty.assign(g.nseq, {0, 0});
    if (dev < 0) return;
    if (!k_pool || !v_pool) LS_THROW(LS_ERR_ARG, "the pools must not be NULL");
    check_aligned(k_pool, "k_pool");
    check_aligned(v_pool, "v_pool");
    if (device_of(k_pool, "k_pool") != dev || device_of(v_pool, "v_pool") != dev) LS_THROW(LS_ERR_ARG, "the pools lie on another device");
    k = static_cast<uint8_t*>(k_pool);
    v = static_cast<uint8_t*>(v_pool);
    layer_bytes = (size_t)kv_heads * num_pages * page * hd * 2;
    LS_CUDA(cudaHostAlloc(reinterpret_cast<void**>(&h_err), sizeof(int), cudaHostAllocMapped));
    *h_err = 0;
    LS_CUDA(cudaHostGetDevicePointer(reinterpret_cast<void**>(&d_err), h_err, 0));
    const size_t entries = (size_t)g.nseq * g.max_pages;
    LS_CUDA(cudaMalloc(&d_table, entries * 4));
    LS_CUDA(cudaMemset(d_table, 0, entries * 4));
    work.open(g, bf16, d_err, nullptr);  // (waited for below: steps may run on any stream)
    maps.resize(2 * layers);
    for (size_t l = 0; l < layers; l++)
      for (int i = 0; i < 2; i++)
        kv_encode_map(&maps[2 * l + i], (i ? v : k) + l * layer_bytes, (uint64_t)kv_heads * num_pages * page, g.hd, kv_box_rows(g.page()), bf16);
    for (Stage& s : stage) LS_CUDA(cudaEventCreateWithFlags(&s.done, cudaEventDisableTiming));
    LS_CUDA(cudaDeviceSynchronize());
  }

  // Sequence s holds exactly these pages, n positions of them cached.
  void set(uint64_t s, const int32_t* pages, uint64_t npages, uint64_t n) {
    check_seq(s);
    if (npages > (uint64_t)g.max_pages) LS_THROW(LS_ERR_ARG, "more pages than max_ctx positions need");
    if (n > max_ctx || n > npages << g.shift) LS_THROW(LS_ERR_ARG, "the pages hold fewer than n positions, or n exceeds max_ctx");
    std::vector<int32_t> p(pages, pages + npages);
    std::vector<int32_t> sorted = p;
    std::sort(sorted.begin(), sorted.end());
    if (npages && (sorted.front() < 0 || sorted.back() >= g.num_pages)) LS_THROW(LS_ERR_ARG, "a page is outside the pool");
    if (std::adjacent_find(sorted.begin(), sorted.end()) != sorted.end()) LS_THROW(LS_ERR_ARG, "a page is named twice");
    changed();
    for (int32_t x : p)
      if (ref[x]++ == 0) nfree--;
    keep_pages((int)s, 0);
    std::copy(p.begin(), p.end(), row((int)s));
    held[s] = (int)npages;
    len[s] = (int)n;
    touch((int)s, 0, (int)npages);
  }

  // Every dst holds the first n positions of src (in the same pages).
  void fork(uint64_t src, const uint64_t* dst, uint64_t ndst, uint64_t n) {
    check_seq(src);
    if (n > (uint64_t)len[src]) LS_THROW(LS_ERR_ARG, "sequence " + std::to_string(src) + " holds " + std::to_string(len[src]) + " positions");
    std::vector<uint8_t> seen(g.nseq, 0);
    for (uint64_t i = 0; i < ndst; i++) {
      check_seq(dst[i]);
      if (dst[i] == src) LS_THROW(LS_ERR_ARG, "a sequence cannot be forked onto itself");
      if (seen[dst[i]]++) LS_THROW(LS_ERR_ARG, "sequence " + std::to_string(dst[i]) + " is named twice");
    }
    changed();
    const int need = pages_of(n);
    for (uint64_t i = 0; i < ndst; i++) {
      const int d = (int)dst[i];
      for (int p = 0; p < need; p++) ref[row((int)src)[p]]++;
      keep_pages(d, 0);
      std::copy(row((int)src), row((int)src) + need, row(d));
      held[d] = need;
      len[d] = (int)n;
      touch(d, 0, need);
    }
  }

  void truncate(uint64_t s, uint64_t n) {
    check_seq(s);
    if (n > (uint64_t)len[s]) LS_THROW(LS_ERR_ARG, "cannot truncate " + std::to_string(len[s]) + " positions to " + std::to_string(n));
    changed();
    len[s] = (int)n;
    keep_pages((int)s, pages_of(n));
  }

  // Pages in use move to the lowest ids; every table follows.
  uint64_t compact(cudaStream_t st) {
    if (device >= 0) {
      check_err();
      if (capturing(st)) LS_THROW(LS_ERR_ARG, "the cache cannot be compacted while the stream is being captured");
    }
    const int used = g.num_pages - nfree;
    std::vector<int32_t> to(g.num_pages, -1);
    copies.clear();
    int low = 0;
    for (int p = used; p < g.num_pages; p++)
      if (ref[p]) {
        while (ref[low]) low++;
        to[p] = low;
        copies.push_back({p, low++, g.page()});
      }
    if (copies.empty()) return 0;
    if (device >= 0)
      launch_page_copies(k, v, (int)layers, g.kv_heads, g.hd, g.page(), g.num_pages, copies.data(), copies.size(), g.nctas, st);
    changed();
    for (const PageCopy& c : copies) {
      ref[c.dst] = ref[c.src];
      ref[c.src] = 0;
    }
    lowest = used;
    for (int s = 0; s < g.nseq; s++)
      for (int i = 0; i < held[s]; i++)
        if (to[row(s)[i]] >= 0) {
          row(s)[i] = to[row(s)[i]];
          touch(s, i, i + 1);
        }
    return copies.size();
  }

  std::vector<KvSeqIn> inputs() const {
    std::vector<KvSeqIn> in(g.nseq);
    for (int s = 0; s < g.nseq; s++) {
      in[s].n = len[s];
      in[s].cnt = counts[s];
      in[s].table = row(s);
      in[s].tab = (int)((size_t)s * g.max_pages);
    }
    return in;
  }

  // A step: sequence s is to get cnt[s] rows (0..M) behind its cached positions.
  void begin(const uint32_t* cnt, uint64_t M, cudaStream_t st) {
    if (M == 0 || M > (uint64_t)g.max_rows / g.nseq) LS_THROW(LS_ERR_ARG, "seqs x M must be in 1..max_rows");
    if (device >= 0) {
      check_err();
      if (capturing(st)) LS_THROW(LS_ERR_ARG, "a step cannot begin while the stream is being captured");
    }
    // what it takes: pages past the held ones, and copies of pages that others hold too (the last
    // holder of a page writes it in place)
    std::unordered_map<int32_t, int> writers;
    int64_t need = 0;
    for (int s = 0; s < g.nseq; s++) {
      if (cnt[s] > M) LS_THROW(LS_ERR_ARG, "sequence " + std::to_string(s) + " has more than M rows");
      if (cnt[s] == 0) continue;
      if ((uint64_t)len[s] + cnt[s] > max_ctx)
        LS_THROW(LS_ERR_ARG, "sequence " + std::to_string(s) + ": context is full (" + std::to_string(len[s]) + " + " + std::to_string(cnt[s]) +
                                 " > " + std::to_string(max_ctx) + ")");
      const int last = pages_of((size_t)len[s] + cnt[s]);
      need += std::max(0, last - held[s]);
      for (int i = len[s] >> g.shift; i < std::min(last, held[s]); i++)
        if (ref[row(s)[i]] > 1 && ++writers[row(s)[i]] < ref[row(s)[i]]) need++;
    }
    if (need > nfree) LS_THROW(LS_ERR_ARG, "the K/V page pool is exhausted: " + std::to_string(need) + " pages needed, " + std::to_string(nfree) + " free");
    begun = false;
    copies.clear();
    struct Entry {
      int s, i;
      int32_t before;  // -1: the sequence has grown by this page
    };
    std::vector<Entry> entries;  // table entries that the step changes
    try {
      for (int s = 0; s < g.nseq; s++) {
        counts[s] = (int)cnt[s];
        if (cnt[s] == 0) continue;
        const int last = pages_of((size_t)len[s] + cnt[s]);
        for (int i = len[s] >> g.shift; i < last; i++) {
          if (i >= held[s]) {
            entries.push_back({s, i, -1});
            row(s)[i] = take();
            held[s] = i + 1;
            touch(s, i, i + 1);
          } else if (ref[row(s)[i]] > 1) {
            const int old = row(s)[i], rows = std::max(0, len[s] - (i << g.shift));
            if (rows) copies.push_back({old, -1, rows});
            entries.push_back({s, i, old});
            row(s)[i] = take();
            drop(old);
            if (rows) copies.back().dst = row(s)[i];
            touch(s, i, i + 1);
            version++;
          }
        }
      }
      planner.build(inputs(), (int)M, version);
      if (inject_fail) LS_THROW(LS_ERR_CUDA, "the step's launches failed (test hook)");
      if (device >= 0) upload(st);
    } catch (...) {
      // the copies may not have been made: the tables are what they were, and go up whole with the next step
      inject_fail = false;
      for (size_t e = entries.size(); e-- > 0;) {
        const Entry& x = entries[e];
        drop(row(x.s)[x.i]);
        if (x.before < 0) {
          held[x.s] = x.i;
        } else {
          row(x.s)[x.i] = x.before;
          ref[x.before]++;
        }
      }
      for (int s = 0; s < g.nseq; s++) touch(s, 0, held[s]);
      changed();
      throw;
    }
    begun = true;
  }

  // The page copies, the changed table entries and the plan, in stream order.
  void upload(cudaStream_t st) {
    OnDevice on(device);
    if (!copies.empty()) launch_page_copies(k, v, (int)layers, g.kv_heads, g.hd, g.page(), g.num_pages, copies.data(), copies.size(), g.nctas, st);
    size_t nr = 0, entries = 0;
    for (const auto& d : dirty)
      if (d.first < d.second) {
        nr++;
        entries += d.second - d.first;
      }
    // staged as: plan | table ranges (KvRange each) | their entries
    const size_t plan = planner.bytes.size(), need = plan + nr * sizeof(KvRange) + entries * 4;
    Stage& sg = stage[turn ^= 1];
    LS_CUDA(cudaEventSynchronize(sg.done));  // its last upload has been read
    if (sg.cap < need) {
      if (sg.p) LS_CUDA(cudaFreeHost(sg.p));
      sg.p = nullptr;
      sg.cap = 0;
      const size_t cap = std::max<size_t>(2 * need, 1 << 16);
      LS_CUDA(cudaHostAlloc(reinterpret_cast<void**>(&sg.p), cap, cudaHostAllocMapped));
      LS_CUDA(cudaHostGetDevicePointer(reinterpret_cast<void**>(&sg.d), sg.p, 0));
      sg.cap = cap;
    }
    std::memcpy(sg.p, planner.bytes.data(), planner.bytes.size());
    auto* ranges = reinterpret_cast<KvRange*>(sg.p + plan);
    auto* vals = reinterpret_cast<int32_t*>(ranges + nr);
    size_t r = 0, at = 0;
    for (int s = 0; s < g.nseq; s++) {
      auto& d = dirty[s];
      if (d.first >= d.second) continue;
      const int n = d.second - d.first;
      ranges[r++] = {(int32_t)((size_t)s * g.max_pages + d.first), (int32_t)at, n, 0};
      std::copy(row(s) + d.first, row(s) + d.second, vals + at);
      at += n;
      d = {0, 0};
    }
    launch_stage(d_table, reinterpret_cast<const KvRange*>(sg.d + plan), (int)nr, work.plan, sg.d, plan, st);
    LS_CUDA(cudaEventRecord(sg.done, st));
  }

  void attention(uint64_t layer, const void* qkv, uint64_t qkv_stride, const float* rope, void* out, uint64_t out_stride, cudaStream_t st) {
    if (device < 0) LS_THROW(LS_ERR_ARG, "this cache keeps pages only (it was opened without a device)");
    if (!begun) LS_THROW(LS_ERR_ARG, "no step has begun (or the tables have changed since)");
    if (layer >= layers) LS_THROW(LS_ERR_ARG, "layer " + std::to_string(layer) + " is outside the cache's " + std::to_string(layers));
    if (!qkv || !out) LS_THROW(LS_ERR_ARG, "qkv and out must not be NULL");
    const uint64_t w = (uint64_t)(g.heads + 2 * g.kv_heads) * g.hd, H = (uint64_t)g.heads * g.hd;
    if (qkv_stride == 0) qkv_stride = w;
    if (out_stride == 0) out_stride = H;
    if (qkv_stride < w || qkv_stride % 8 || out_stride < H || out_stride % 8 || qkv_stride > (1ull << 32) || out_stride > (1ull << 32))
      LS_THROW(LS_ERR_ARG, "row strides must be multiples of 8 elements and hold a row");
    check_aligned(qkv, "qkv");
    check_aligned(out, "out");
    check_aligned(rope, "rope");
    check_err();
    OnDevice on(device);
    KvAttn a;
    a.qkv = qkv;
    a.qkv_stride = qkv_stride;
    a.rope = reinterpret_cast<const float2*>(rope);
    a.k = k + layer * layer_bytes;
    a.v = v + layer * layer_bytes;
    a.tables = d_table;
    a.kmap = &maps[2 * layer];
    a.vmap = &maps[2 * layer + 1];
    a.out = out;
    a.out_stride = out_stride;
    a.M = reinterpret_cast<const KvHdr*>(planner.bytes.data())->M;
    a.rows = a.M * g.nseq;
    launch_kv_attention(work, a, st);
  }

  // keep[s] of the step's rows stay (NULL: all of them); pages past them go back.
  void end(const uint32_t* keep) {
    if (!begun) LS_THROW(LS_ERR_ARG, "no step has begun (or the tables have changed since)");
    for (int s = 0; keep && s < g.nseq; s++)
      if (keep[s] > (uint32_t)counts[s]) LS_THROW(LS_ERR_ARG, "sequence " + std::to_string(s) + " cannot keep more rows than it got");
    for (int s = 0; s < g.nseq; s++) {
      if (counts[s] == 0) continue;
      len[s] += keep ? (int)keep[s] : counts[s];
      keep_pages(s, pages_of(len[s]));
    }
    begun = false;
  }

  void inject(int code) {
    if (code < 0 || code > 2 || (code == 2 && device < 0)) LS_THROW(LS_ERR_ARG, "the injected error must be 0, 1 or (with a GPU) 2");
    inject_fail = code == 1;
    if (code == 2) *reinterpret_cast<volatile int*>(h_err) = 1;
  }

  // Throws unless the pages' counts, the free count and the plan agree with the tables.
  void self_check() const {
    std::vector<int32_t> count(g.num_pages, 0);
    for (int s = 0; s < g.nseq; s++) {
      if (held[s] < pages_of(len[s]) || held[s] > g.max_pages) LS_THROW(LS_ERR_ARG, "a sequence holds too few or too many pages");
      for (int i = 0; i < held[s]; i++) {
        const int p = row(s)[i];
        if (p < 0 || p >= g.num_pages) LS_THROW(LS_ERR_ARG, "a table names a page outside the pool");
        count[p]++;
      }
    }
    int free = 0;
    for (int p = 0; p < g.num_pages; p++) {
      if (count[p] != ref[p]) LS_THROW(LS_ERR_ARG, "a page's count is not the number of tables that name it");
      free += count[p] == 0;
      if (count[p] == 0 && p < lowest) LS_THROW(LS_ERR_ARG, "a free page lies below the lowest");
    }
    if (free != nfree) LS_THROW(LS_ERR_ARG, "the free count is wrong");
    if (!begun) return;
    for (int s = 0; s < g.nseq; s++)
      for (int i = len[s] >> g.shift; counts[s] && i < pages_of((size_t)len[s] + counts[s]); i++)
        if (ref[row(s)[i]] != 1) LS_THROW(LS_ERR_ARG, "a page to be written is shared");
    planner.check(inputs());
  }
};

namespace ls {

LsKv* kv_open(int device, uint64_t layers, uint64_t heads, uint64_t kv_heads, uint64_t hd, int dtype, uint64_t page, uint64_t num_pages,
              uint64_t seqs, uint64_t max_ctx, uint64_t max_rows, void* k_pool, void* v_pool) {
  OnDevice on(device);
  std::unique_ptr<LsKv> kv(new LsKv);
  kv->open(device, layers, heads, kv_heads, hd, dtype, page, num_pages, seqs, max_ctx, max_rows, k_pool, v_pool);
  return kv.release();
}
void kv_free(LsKv* kv) { delete kv; }
void kv_set(LsKv* kv, uint64_t s, const int32_t* pages, uint64_t npages, uint64_t n) { kv->set(s, pages, npages, n); }
void kv_fork(LsKv* kv, uint64_t src, const uint64_t* dst, uint64_t ndst, uint64_t n) { kv->fork(src, dst, ndst, n); }
void kv_truncate(LsKv* kv, uint64_t s, uint64_t n) { kv->truncate(s, n); }
uint64_t kv_compact(LsKv* kv, cudaStream_t st) {
  OnDevice on(kv->device);
  return kv->compact(st);
}
void kv_begin(LsKv* kv, const uint32_t* counts, uint64_t M, cudaStream_t st) {
  OnDevice on(kv->device);
  kv->begin(counts, M, st);
}
void kv_attention(LsKv* kv, uint64_t layer, const void* qkv, uint64_t qkv_stride, const float* rope, void* out, uint64_t out_stride,
                  cudaStream_t st) {
  kv->attention(layer, qkv, qkv_stride, rope, out, out_stride, st);
}
void kv_end(LsKv* kv, const uint32_t* keep) { kv->end(keep); }
void kv_self_check(const LsKv* kv) { kv->self_check(); }
void kv_inject(LsKv* kv, int code) { kv->inject(code); }
void kv_info(const LsKv* kv, LsKvInfo* o) {
  o->seqs = kv->g.nseq;
  o->max_pages = kv->g.max_pages;
  o->num_pages = kv->g.num_pages;
  o->pages_used = kv->g.num_pages - kv->nfree;
  o->pages_shared = 0;
  for (int32_t r : kv->ref) o->pages_shared += r > 1;
  o->shared_positions = kv->begun ? kv->planner.shared_positions() : 0;
}
uint64_t kv_len(const LsKv* kv, uint64_t s) {
  kv->check_seq(s);
  return kv->len[s];
}
void kv_tables(const LsKv* kv, int32_t* out) {
  for (int s = 0; s < kv->g.nseq; s++)
    for (int i = 0; i < kv->g.max_pages; i++) out[(size_t)s * kv->g.max_pages + i] = i < kv->held[s] ? kv->row(s)[i] : -1;
}

void kv_copy_pages(void* k, void* v, uint64_t layers, uint64_t kv_heads, uint64_t hd, uint64_t page, uint64_t num_pages, const int32_t* src,
                   const int32_t* dst, const int32_t* rows, uint64_t n, cudaStream_t st) {
  check_pool(layers, kv_heads, hd, page, num_pages);
  if (!k || !v) LS_THROW(LS_ERR_ARG, "the pools must not be NULL");
  check_aligned(k, "k_pool");
  check_aligned(v, "v_pool");
  if (n == 0) return;
  if (!src || !dst) LS_THROW(LS_ERR_ARG, "src and dst must not be NULL");
  if (n > num_pages) LS_THROW(LS_ERR_ARG, "more copies than pages");
  std::vector<PageCopy> c(n);
  std::vector<uint8_t> role(num_pages, 0);  // 1: read, 2: written
  for (uint64_t i = 0; i < n; i++) {
    if (src[i] < 0 || (uint64_t)src[i] >= num_pages || dst[i] < 0 || (uint64_t)dst[i] >= num_pages)
      LS_THROW(LS_ERR_ARG, "a page is outside the pool");
    const int r = rows ? rows[i] : (int)page;
    if (r < 0 || (uint64_t)r > page) LS_THROW(LS_ERR_ARG, "rows must be in 0..page");
    if (role[dst[i]]) LS_THROW(LS_ERR_ARG, "page " + std::to_string(dst[i]) + " is written twice, or also read");
    role[dst[i]] = 2;
    c[i] = {src[i], dst[i], r};
    if (role[src[i]] == 2) LS_THROW(LS_ERR_ARG, "page " + std::to_string(src[i]) + " is both read and written");
    role[src[i]] = 1;
  }
  const int dev = device_of(k, "k_pool");
  if (device_of(v, "v_pool") != dev) LS_THROW(LS_ERR_ARG, "the pools lie on different devices");
  OnDevice on(dev);
  launch_page_copies(k, v, (int)layers, (int)kv_heads, (int)hd, (int)page, (int)num_pages, c.data(), n, num_sms(dev), st);
}

}  // namespace ls
