// Host side of attention over shared pages: finds the ranges of positions that several sequences
// hold in the same pages, and cuts the work into the CTAs' programs. No GPU is needed here.
#include <algorithm>
#include <cstring>
#include <unordered_map>

#include "layerstream.h"
#include "ls_kv.h"

namespace ls {

// A range is read for its sequences at once when that saves at least this many position reads over
// the sequences reading it one by one: below it, the extra partial that every row then leaves and
// joins costs about as much as the reads. Calls in a graph, single rows of 2 to 64 sequences, 14/2 heads of 64, 16/2
// and 32/8 of 128, read at once against one by one: 3 to 7 % slower where 32 to 200 reads are saved (two
// sequences under 64 positions 7.66 against 7.31 us), within 4 % either way from 256 to 1500, then up to 8 % faster with
// 2 kv heads (64 under 512: 10.4 against 11.3) and up to 51 % with 8 (14.5 against 29.6). It stays slower, by up to
// 13 %, for 16 to 64 sequences under at most 256 positions at hd 128 with 2 kv heads (64 under 128: 11.8 against 10.4).
constexpr long long kMinSaved = 256;

// Time of a CTA's work in units of one pair chunk: a chunk for two tiles, for one tile (the two lanes work on
// different ones), and what a piece costs before its first chunk and after its last. From timelines of the CTAs
// (hd 64 and 128, 2 to 64 readers of 2k to 64k positions): a pair chunk takes about 3400 cycles. Without the starts
// of pieces that a CTA's end cuts, the CTAs of single tiles ended 40 % after those of pairs; with them
// all end within 15 % of the mean (four prompts of 8k with 16 samples each 61.8 against 54.8 us, a prefill of
// eight chunks 52.8 against 46.5). A single chunk at 0.55 instead: 64 readers of 32k 68.6 against 65.4 us.
// Dealt by shares of what is left instead of by the least time that is enough, the last CTA was left with whatever
// the estimate of the cuts had missed: 8 sequences x 5 rows under 8192 (14/2 heads x 64) 71.5 against 13.3 us, 32 x 1
// 36.2 against 13.2, 4 x 12 (16/2 x 128) 101 against 17.5; at most 7 % faster (4 x 48, 26.1 against 27.9).
constexpr double kPairChunk = 1.0, kSingleChunk = 0.62, kPairStart = 1.5, kSingleStart = 0.4;
constexpr double kDealSlack = 2 * kPairStart + kPairChunk;

// A row with more partials than this is merged by a whole block instead of hd / 4 of its threads when rows and
// heads are few (KV_SPLIT_ITEMS). 16 rows of 14 heads, 40 partials: hd / 4 threads 10.4 us, a block 5.0; 288
// rows of 16 heads, 10 partials: 7.0 and 13.3.
constexpr int kSplitRows = 8;

static size_t align16(size_t n) { return (n + 15) / 16 * 16; }

size_t KvGeom::plan_cap() const {
  return align16(sizeof(KvHdr)) + align16(nctas * sizeof(KvProg)) + align16(segs_cap() * sizeof(KvSeg)) +
         align16(nseq * sizeof(KvSeq)) + align16(units_cap() * sizeof(KvUnit));
}

// Groups the sequences with rows by their first page, then each group by the page after its common
// prefix: two levels of shared ranges at most (a system prompt, then a prompt under it); what
// deeper forks share is read by each sequence on its own. Only pages whose every position is cached
// in all of the group (none of them is written by this step) are shared.
void KvPlanner::tree(const std::vector<KvSeqIn>& seqs) {
  order_.clear();
  shared_.clear();
  std::vector<int> act, alone;
  for (size_t i = 0; i < seqs.size(); i++)
    if (class_[i] != IDLE) (class_[i] == ALONE ? alone : act).push_back((int)i);
  auto full = [&](int i) { return seqs[i].n >> g.shift; };
  // runs of `ids` that agree on the page at depth d, in order of first appearance; sequences without a
  // full page there come last, one by one
  auto split = [&](const std::vector<int>& ids, int d) {
    std::vector<std::vector<int>> runs;
    std::unordered_map<int, size_t> at;
    for (int i : ids)
      if (full(i) > d) {
        auto it = at.find(seqs[i].table[d]);
        if (it == at.end()) {
          at[seqs[i].table[d]] = runs.size();
          runs.push_back({i});
        } else {
          runs[it->second].push_back(i);
        }
      }
    for (int i : ids)
      if (full(i) <= d) runs.push_back({i});
    return runs;
  };
  auto common = [&](const std::vector<int>& ids, int d) {  // pages [0, c) equal in all, c >= d
    int c = full(ids[0]);
    for (int i : ids) c = std::min(c, full(i));
    for (size_t k = 1; k < ids.size(); k++) {
      int e = d;
      while (e < c && seqs[ids[k]].table[e] == seqs[ids[0]].table[e]) e++;
      c = std::min(c, e);
    }
    return std::max(c, d);
  };
  auto worth = [&](size_t members, int a_pages, int b_pages) {
    return members >= 2 && (long long)(b_pages - a_pages) * g.page() * (long long)(members - 1) >= kMinSaved;
  };
  for (const auto& grp : split(act, 0)) {
    int base = 0;  // pages covered by shared ranges so far
    const int c = grp.size() >= 2 ? common(grp, 0) : 0;
    const size_t at1 = shared_.size();
    if (worth(grp.size(), 0, c)) {
      shared_.push_back({0, c << g.shift, (int)order_.size(), 0, seqs[grp[0]].tab, false});
      base = c;
    }
    for (const auto& sub : split(grp, c)) {
      const int c2 = sub.size() >= 2 ? common(sub, c) : 0;
      if (sub.size() < grp.size() && worth(sub.size(), base, c2))
        shared_.push_back({base << g.shift, c2 << g.shift, (int)order_.size(), (int)(order_.size() + sub.size()), seqs[sub[0]].tab, false});
      order_.insert(order_.end(), sub.begin(), sub.end());
    }
    if (base) shared_[at1].last = (int)order_.size();
  }
  order_.insert(order_.end(), alone.begin(), alone.end());
}

KvPlanner::Class KvPlanner::class_of(int cnt) const {
  if (cnt == 0) return IDLE;
  // rows that fill tiles of their own read the prefix once per pair of tiles either way: as one range with
  // their own positions they leave one partial less
  // (2 to 8 sequences of 16 to 128 rows under 1k to 8k: blocks that fill their pairs to 0.9 and more take up to 31 %
  // longer in a group, 8 x 128 rows of 16/2 heads of 128 under 8k 100.9 against 77.1 us; blocks that fill them to 0.5 to
  // 0.7 take up to 16 % longer alone, 8 x 20 rows of 14/2 heads of 64 under 8k 24.2 against 20.4)
  const int rows = cnt * g.G(), pairs = (rows + 2 * KV_TILE - 1) / (2 * KV_TILE);
  return rows * 5 >= pairs * 2 * KV_TILE * 4 ? ALONE : GROUPED;
}

double KvPlanner::start_of(const Job& j) { return j.ntiles == 2 ? kPairStart : kSingleStart; }
double KvPlanner::chunk_of(const Job& j) { return j.ntiles == 2 ? kPairChunk : kSingleChunk; }

void KvPlanner::build(const std::vector<KvSeqIn>& seqs, int M, uint64_t version) {
  std::vector<Class> now(seqs.size());
  for (size_t i = 0; i < seqs.size(); i++) now[i] = class_of(seqs[i].cnt);
  if (version != version_ || now != class_) {
    class_ = now;
    version_ = ~0ull;  // (kept if tree throws: the next build makes it anew)
    tree(seqs);
    version_ = version;
  }
  const int G = g.G(), kvh = g.kv_heads;
  // rows, nodes
  dseqs_.assign(seqs.size(), KvSeq{});
  for (size_t i = 0; i < seqs.size(); i++) {
    dseqs_[i].n = seqs[i].n;
    dseqs_[i].cnt = seqs[i].cnt;
    dseqs_[i].tab = seqs[i].tab;
  }
  int R = 0;
  for (int i : order_) {
    dseqs_[i].row0 = R;
    R += seqs[i].cnt * G;
  }
  nodes_ = shared_;
  shared_pos_ = 0;
  std::vector<int> from(seqs.size(), 0);
  for (size_t k = 0; k < shared_.size(); k++) {
    const Node& nd = shared_[k];
    shared_pos_ += nd.b - nd.a;
    for (int o = nd.first; o < nd.last; o++) {
      KvSeq& d = dseqs_[order_[o]];
      d.lunit[d.nlev++] = (int)k;  // the node, until its unit is known
      from[order_[o]] = nd.b;
    }
  }
  for (size_t o = 0; o < order_.size(); o++) {
    const int i = order_[o];
    KvSeq& d = dseqs_[i];
    d.lunit[d.nlev++] = (int)nodes_.size();
    nodes_.push_back({from[i], seqs[i].n + seqs[i].cnt, (int)o, (int)o + 1, seqs[i].tab, true});
  }
  // units, jobs: pairs of tiles of one kv head first, then single tiles
  dnodes_.clear();
  jobs_.clear();
  int units = 0;
  auto rows_of = [&](const Node& nd) {
    const KvSeq &f = dseqs_[order_[nd.first]], &l = dseqs_[order_[nd.last - 1]];
    return std::make_pair((int)f.row0, (int)(l.row0 + l.cnt * G - f.row0));
  };
  auto end_of = [&](const Node& nd, int tile, int nrows) {  // positions past what the tile's last row sees are left out
    if (!nd.own) return nd.b;
    const int last = std::min((tile + 1) * KV_TILE, nrows) - 1;
    return std::min(nd.b, seqs[order_[nd.first]].n + last / G + 1);
  };
  for (size_t k = 0; k < nodes_.size(); k++) {
    const auto [row0, nrows] = rows_of(nodes_[k]);
    const int nt = (nrows + KV_TILE - 1) / KV_TILE;
    dnodes_.push_back({row0, nt, units});
    units += nt * kvh;
  }
  for (int i : order_)
    for (int l = 0; l < dseqs_[i].nlev; l++) {
      const DNode& d = dnodes_[dseqs_[i].lunit[l]];
      dseqs_[i].lrow0[l] = d.row0;
      dseqs_[i].ltile[l] = d.ntile;
      dseqs_[i].lunit[l] = d.unit0;
    }
  for (int pass = 0; pass < 2; pass++)
    for (size_t k = 0; k < nodes_.size(); k++) {
      const auto [row0, nrows] = rows_of(nodes_[k]);
      (void)row0;
      const int nt = dnodes_[k].ntile;
      for (int h = 0; h < kvh; h++) {
        if (pass == 0)
          for (int t = 0; t + 1 < nt; t += 2) {
            const int p1 = end_of(nodes_[k], t + 1, nrows);
            jobs_.push_back({(int)k, h, t, 2, (p1 - nodes_[k].a + KV_CHUNK - 1) / KV_CHUNK, p1});
          }
        else if (nt & 1) {
          const int p1 = end_of(nodes_[k], nt - 1, nrows);
          jobs_.push_back({(int)k, h, nt - 1, 1, (p1 - nodes_[k].a + KV_CHUNK - 1) / KV_CHUNK, p1});
        }
      }
    }
  // The jobs' chunks in order, dealt to the CTAs: each takes what fits into its time, at least one chunk; the least time
  // for which the CTAs are enough is searched for, to 2 %. A CTA wastes less than a start and a chunk and pays one
  // start that a cut added, so kDealSlack above the mean is always enough.
  double work = 0, least = 0;
  for (const Job& j : jobs_) {
    work += start_of(j) + j.nch * chunk_of(j);
    least = std::max(least, start_of(j) + chunk_of(j));
  }
  auto deal = [&](double time, bool keep) {  // CTAs that it takes
    int cta = 0;
    double room = time;
    for (size_t k = 0; k < jobs_.size(); k++) {
      const double q = chunk_of(jobs_[k]), o = start_of(jobs_[k]);
      for (int c = 0; c < jobs_[k].nch;) {
        const double fit = (room - o) / q;
        if (fit < 1) {  // (never in a CTA that has nothing yet)
          cta++;
          room = time;
          continue;
        }
        const int take = fit < jobs_[k].nch - c ? (int)fit : jobs_[k].nch - c;
        if (keep) pieces_.push_back({cta, (int)k, c, take});
        room -= o + take * q;
        c += take;
      }
    }
    return cta + 1;
  };
  pieces_.clear();
  if (!jobs_.empty()) {
    double low = std::max(work / g.nctas, least * (1 + 1e-9)), high = low + kDealSlack;
    if (deal(low, false) <= g.nctas) high = low;
    while (high - low > 0.02 * low) {
      const double mid = (low + high) / 2;
      (deal(mid, false) <= g.nctas ? high : low) = mid;
    }
    if (deal(high, true) > g.nctas) LS_THROW(LS_ERR_ARG, "internal: an attention plan needs more CTAs than there are");
  }
  // segments
  segs_.clear();
  progs_.assign(g.nctas, KvProg{});
  units_.assign(units, KvUnit{});
  auto emit = [&](std::vector<KvSeg>& to, const Job& j, int tile, int c0, int nch) {
    const Node& nd = nodes_[j.node];
    const auto [row0, nrows] = rows_of(nd);
    KvSeg s{};
    s.qrow = j.g * R + row0 + tile * KV_TILE;
    s.nrows = std::min(KV_TILE, nrows - tile * KV_TILE);
    s.tab = nd.tab;
    s.kv_head = j.g;
    s.p0 = nd.a + c0 * KV_CHUNK;
    s.p1 = std::min(j.p1, nd.a + (c0 + nch) * KV_CHUNK);
    s.nch = nch;
    s.causal = nd.own ? seqs[order_[nd.first]].n : INT_MAX;
    s.trow0 = tile * KV_TILE;
    s.flag = nd.own ? order_[nd.first] * kvh + j.g : -1;
    s.unit = dnodes_[j.node].unit0 + j.g * dnodes_[j.node].ntile + tile;
    s.slot = units_[s.unit].nseg++;  // which of the unit's segments, until its partials have a place
    units_[s.unit].nrows = s.nrows;
    to.push_back(s);
  };
  for (size_t k = 0; k < pieces_.size();) {
    const int cta = pieces_[k].cta;
    lane_[0].clear();
    lane_[1].clear();
    KvProg& pr = progs_[cta];
    for (; k < pieces_.size() && pieces_[k].cta == cta && jobs_[pieces_[k].job].ntiles == 2; k++) {
      const Piece& p = pieces_[k];
      for (int t = 0; t < 2; t++) emit(lane_[t], jobs_[p.job], jobs_[p.job].tile + t, p.c0, p.nch);
      pr.npair++;
      pr.pair_ch += p.nch;
    }
    int single = 0;
    for (size_t e = k; e < pieces_.size() && pieces_[e].cta == cta; e++) single += pieces_[e].nch;
    // single tiles: the first half of their chunks to lane 0, the rest to lane 1
    int left0 = (single + 1) / 2;
    for (; k < pieces_.size() && pieces_[k].cta == cta; k++) {
      const Piece& p = pieces_[k];
      const Job& j = jobs_[p.job];
      const int n0 = std::min(left0, p.nch);
      if (n0) emit(lane_[0], j, j.tile, p.c0, n0);
      if (p.nch > n0) emit(lane_[1], j, j.tile, p.c0 + n0, p.nch - n0);
      left0 -= n0;
    }
    // short tiles of a lane's own phase alternate between the halves of its tensor-memory lanes (the other
    // lane starts with the other half: their warps then sit on different schedulers)
    for (int t = 0; t < 2; t++)
      for (size_t i = pr.npair; i < lane_[t].size(); i++)
        if (lane_[t][i].nrows <= KV_TILE / 2) lane_[t][i].shift = ((int)i - pr.npair + t) % 2 * (KV_TILE / 2);
    for (int t = 0; t < 2; t++) {
      pr.seg[t] = (int)segs_.size();
      pr.nseg[t] = (int)lane_[t].size();
      segs_.insert(segs_.end(), lane_[t].begin(), lane_[t].end());
    }
  }
  int slots = 0, most = 0;  // most: partials of one row
  for (KvUnit& u : units_) {
    u.base = slots;
    slots += u.nseg * u.nrows;
  }
  for (KvSeg& s : segs_) s.slot = units_[s.unit].base + s.slot * s.nrows;
  for (int i : order_)
    for (int kh = 0; kh < kvh; kh++) {
      int n = 0;
      for (int l = 0; l < dseqs_[i].nlev; l++)
        n += units_[dseqs_[i].lunit[l] + kh * dseqs_[i].ltile[l] + (dseqs_[i].row0 - dseqs_[i].lrow0[l]) / KV_TILE].nseg;
      most = std::max(most, n);
    }
  if ((size_t)R > g.rows_cap() || (size_t)units > g.units_cap() || segs_.size() > g.segs_cap() || (size_t)slots > g.slots_cap())
    LS_THROW(LS_ERR_ARG, "internal: an attention plan outgrew its workspace");
  // pack
  KvHdr h{};
  h.M = M;
  h.nseq = (int)seqs.size();
  h.R = R;
  h.max_pages = g.max_pages;
  h.nslots = slots;
  h.split_rows = most > kSplitRows && (long long)R * kvh <= (long long)g.nctas * KV_SPLIT_ITEMS;
  size_t at = KV_SEQ_AT + align16(dseqs_.size() * sizeof(KvSeq));
  auto place = [&](int32_t& off, size_t n) {
    off = (int32_t)at;
    at += align16(n);
  };
  place(h.off_prog, progs_.size() * sizeof(KvProg));
  place(h.off_seg, segs_.size() * sizeof(KvSeg));
  place(h.off_unit, units_.size() * sizeof(KvUnit));
  bytes.resize(at);
  auto put = [&](int32_t off, const void* p, size_t n) {
    if (n) std::memcpy(bytes.data() + off, p, n);
  };
  put(0, &h, sizeof h);
  put(h.off_prog, progs_.data(), progs_.size() * sizeof(KvProg));
  put(h.off_seg, segs_.data(), segs_.size() * sizeof(KvSeg));
  put(KV_SEQ_AT, dseqs_.data(), dseqs_.size() * sizeof(KvSeq));
  put(h.off_unit, units_.data(), units_.size() * sizeof(KvUnit));
  if (at > g.plan_cap()) LS_THROW(LS_ERR_ARG, "internal: an attention plan outgrew its workspace");
}

// Reads the packed plan as the kernels do (the jobs' costs are the last build's).
void KvPlanner::check(const std::vector<KvSeqIn>& seqs) const {
  auto need = [](bool ok, const char* what) {
    if (!ok) LS_THROW(LS_ERR_ARG, std::string("attention plan: ") + what);
  };
  need(bytes.size() >= sizeof(KvHdr) && bytes.size() <= g.plan_cap(), "size");
  const KvHdr& h = *reinterpret_cast<const KvHdr*>(bytes.data());
  const auto* prog = reinterpret_cast<const KvProg*>(bytes.data() + h.off_prog);
  const auto* seg = reinterpret_cast<const KvSeg*>(bytes.data() + h.off_seg);
  const auto* sq = reinterpret_cast<const KvSeq*>(bytes.data() + KV_SEQ_AT);
  const auto* unit = reinterpret_cast<const KvUnit*>(bytes.data() + h.off_unit);
  const int G = g.G();
  need((size_t)h.R <= g.rows_cap() && (size_t)h.nslots <= g.slots_cap() && h.nseq == (int)seqs.size(), "header");
  // every program's segments: in bounds, pairs aligned, slots written once
  std::unordered_map<int, const KvSeg*> at;
  size_t nseg = 0;
  std::vector<uint8_t> written(h.nslots, 0);
  double work = 0, least = 0;
  for (const Job& j : jobs_) {
    work += start_of(j) + j.nch * chunk_of(j);
    least = std::max(least, start_of(j) + chunk_of(j));
  }
  const double longest = std::max(work / g.nctas, least) + kDealSlack;
  for (int c = 0; c < g.nctas; c++) {
    const KvProg& p = prog[c];
    int pair_ch = 0, own[2] = {0, 0};
    for (int t = 0; t < 2; t++) {
      need(p.nseg[t] >= p.npair, "pair segments");
      for (int i = 0; i < p.nseg[t]; i++) {
        const KvSeg& s = seg[p.seg[t] + i];
        nseg++;
        need(s.nrows >= 1 && s.nrows <= KV_TILE && s.kv_head >= 0 && s.kv_head < g.kv_heads, "rows");
        need(s.qrow >= s.kv_head * h.R && s.qrow + s.nrows <= (s.kv_head + 1) * h.R, "query rows");
        need(s.nch >= 1 && s.p0 >= 0 && s.p1 > s.p0 + (s.nch - 1) * KV_CHUNK && s.p1 <= s.p0 + s.nch * KV_CHUNK, "positions");
        need(s.shift == 0 || (s.shift == KV_TILE / 2 && s.nrows <= KV_TILE / 2 && i >= p.npair), "lane half");
        need(s.p0 % std::min(g.page(), KV_CHUNK) == 0, "page alignment");
        need(s.slot >= 0 && s.slot + s.nrows <= h.nslots, "partial rows");
        for (int r = 0; r < s.nrows; r++) {
          need(!written[s.slot + r], "a partial row is written twice");
          written[s.slot + r] = 1;
        }
        at[s.slot] = &s;
        if (i < p.npair) {
          const KvSeg& a = seg[p.seg[0] + i];
          need(s.tab == a.tab && s.p0 == a.p0 && s.p1 == a.p1 && s.nch == a.nch && s.kv_head == a.kv_head, "pair");
          if (t == 0) pair_ch += s.nch;
        } else {
          own[t] += s.nch;
        }
        // its page-table entries exist
        int seqi = -1;
        for (size_t q = 0; q < seqs.size(); q++)
          if (seqs[q].cnt > 0 && seqs[q].tab == s.tab) seqi = (int)q;
        need(seqi >= 0 && s.p1 <= seqs[seqi].n + seqs[seqi].cnt, "page table");
        for (int p = s.p0 >> g.shift; p <= (s.p1 - 1) >> g.shift; p++)
          need(seqs[seqi].table[p] >= 0 && seqs[seqi].table[p] < g.num_pages, "page id");
      }
    }
    need(pair_ch == p.pair_ch && (own[0] == own[1] || own[0] == own[1] + 1), "lane balance");
    need(p.npair * kPairStart + pair_ch * kPairChunk + (own[0] + own[1]) * kSingleChunk <= longest, "a CTA's share of the work");
  }
  need(nseg == at.size(), "segments");
  // every row's path: positions covered once, through pages equal to its own
  for (int i = 0; i < h.nseq; i++) {
    need(sq[i].cnt == seqs[i].cnt && sq[i].n == seqs[i].n && sq[i].tab == seqs[i].tab, "sequence");
    for (int t = 0; t < sq[i].cnt; t++)
      for (int j = 0; j < G; j++)
        for (int kh = 0; kh < g.kv_heads; kh++) {
          if (t > 2 && t < sq[i].cnt - 1 && (t % 29) != 0) continue;  // long blocks: a sample of the rows
          const int row = sq[i].row0 + t * G + j;
          std::vector<std::pair<int, int>> cover;
          for (int l = 0; l < sq[i].nlev; l++) {
            const int lr = row - sq[i].lrow0[l], tile = lr / KV_TILE;
            need(lr >= 0 && tile < sq[i].ltile[l], "tile");
            const KvUnit& u = unit[sq[i].lunit[l] + kh * sq[i].ltile[l] + tile];
            need(u.nseg > 0, "a unit without segments");
            for (int k = 0; k < u.nseg; k++) {
              auto it = at.find(u.base + k * u.nrows);
              need(it != at.end(), "slot of a segment");
              const KvSeg& s = *it->second;
              need(s.nrows == u.nrows, "rows of a unit");
              need(s.kv_head == kh && s.qrow + lr % KV_TILE == kh * h.R + row && lr % KV_TILE < s.nrows, "row of a segment");
              if (s.causal != INT_MAX) need(s.causal == seqs[i].n && (s.trow0 + lr % KV_TILE) / G == t && s.flag == i * g.kv_heads + kh, "causal limit");
              else need(s.p1 <= seqs[i].n, "a shared range ends inside the cached positions");
              cover.push_back({s.p0, s.p1});
              for (int p = s.p0 >> g.shift; p <= (s.p1 - 1) >> g.shift && s.tab != seqs[i].tab; p++) {
                int other = -1;
                for (size_t q = 0; q < seqs.size(); q++)
                  if (seqs[q].cnt > 0 && seqs[q].tab == s.tab) other = (int)q;
                need(seqs[other].table[p] == seqs[i].table[p], "a shared range names another page");
              }
            }
          }
          std::sort(cover.begin(), cover.end());
          int p = 0;
          for (const auto& c : cover) {
            need(c.first == p, "positions are covered once, in order");
            p = c.second;
          }
          need(p >= seqs[i].n + t + 1, "positions up to the row's own");
        }
  }
}

}  // namespace ls
