// Fragment attention: the plan (work lists of both passes, made once per fragment layout) and the entry points.
#include <algorithm>
#include <utility>
#include <vector>

#include "attention.h"
#include "attention_host.h"

struct vsn_attn {
  struct Side {
    vsn::AttnWork *small_work = nullptr, *pair_work = nullptr, *lone_work = nullptr, *coop_work = nullptr;
    vsn::AttnJoin* join = nullptr;
    vsn::AttnBlock* block = nullptr;
    int small = 0, pair = 0, lone = 0, coop = 0, joins = 0, few = 0, blocks = 0, slots = 0, long_rows = 0;
    vsn::AttnPlanView view() const {
      return {small_work, pair_work, lone_work, coop_work, small, pair, lone, coop, long_rows, block, blocks, join, joins, few};
    }
  };
  int device = 0, heads = 0, kv_heads = 0, dim = 0, reach = 0, n_rel = 0, n_buckets = 0;
  int64_t used_q = 0, used_k = 0;
  bool same_rows = true;  // a fragment's queries are its keys' rows
  Side fwd, by_query, by_key;
  int* lut = nullptr;
  char* lists = nullptr;  // what all of these point into
};

namespace vsn {
namespace {

// A workgroup of four waves reads each tile of rows once for 128 columns, a lone wave once for 32.  Sharing pays from a few
// workgroups on, which pieces multiply, and narrow heads sooner.  Forward + backward with a table, 8 heads, shared and alone:
//   dim 32    104 workgroups (1600 atoms) bf16 224 and 242 us, f32 362 and 342; 192 (3000 atoms) bf16 401 and 455, f32 equal
//   dim 64    104 workgroups bf16 345 and 325 us, f16 345 and 331, f32 622 and 601; 152 (2400 atoms) bf16 467 and 463, f16 479
//             and 482, f32 equal; 192 bf16 587 and 615, f16 609 and 640, f32 1395 and 1474
//   dim 128   104 workgroups bf16 721 and 696 us, f32 1273 and 1226; 192 bf16 1221 and 1245, f32 2849 and 3034
constexpr int kCoopCols = kTile * kCoopWaves;
inline int64_t coop_min(int dim) { return dim <= 32 ? 64 : 160; }
// A run of rows is split into pieces where the items alone are too few waves for the 1024 SIMDs to be filled evenly
// (12 rounds of one wave each); a piece keeps at least 2 tiles.  Whole calls with pieces of 1, 2 and 4 tiles: one protein of
// 175 atoms f32, forward, 18.1, 17.9 and 18.1 us; four proteins of up to 746 atoms f32, forward, 38.3 and 34.4 us, both
// directions 229, 185 and 204 us; 8 read-out rows over up to 17 882 atoms bf16, forward, 42.6, 34.7 and 32.4 us.
constexpr int64_t kPieceWaves = 12288;
constexpr int kPieceTiles = 2;

constexpr int kSmallSums = 4096;  // floats of table sums per wave

struct Lists {
  std::vector<AttnWork> small, pair, lone, coop;
  std::vector<AttnJoin> join;
  std::vector<AttnBlock> block;
  int slots = 0, few = 0;
  bool long_rows = false;
};

Lists make_lists(int64_t n, const int64_t* col_start, const int64_t* col_end, const int64_t* row_start,
                 const int64_t* row_end, int heads, int dim, bool small, bool pair) {
  Lists out;
  int64_t groups = 0;
  for (int64_t f = 0; f < n; ++f) {
    const int64_t cols = col_end[f] - col_start[f];
    if (cols > 2 * kTile) groups += (cols + kCoopCols - 1) / kCoopCols * heads;
  }
  const bool share = groups >= coop_min(dim);
  std::vector<AttnWork> all;
  int64_t waves = 0, tiles = 0;  // of 32 columns; tiles of 32 x 32
  for (int64_t f = 0; f < n; ++f) {
    const int64_t cols = col_end[f] - col_start[f], rows = row_end[f] - row_start[f];
    AttnWork w = {};
    w.slot = -1;
    w.row0 = (int)row_start[f], w.row1 = (int)row_end[f];
    if (small && cols && rows && cols <= kTile && rows <= kTile) {
      w.col0 = (int)col_start[f], w.cols = (int)cols;
      out.small.push_back(w);
      continue;
    }
    if (pair && cols && rows && cols <= 2 * kTile && rows <= 2 * kTile) {
      w.col0 = (int)col_start[f], w.cols = (int)cols;
      out.pair.push_back(w);
      continue;
    }
    const int64_t step = share && cols > 2 * kTile ? kCoopCols : kTile;
    for (int64_t c = 0; c < cols; c += step) {
      w.col0 = (int)(col_start[f] + c), w.cols = (int)std::min<int64_t>(step, cols - c);
      w.step = (int)(step / kTile);
      all.push_back(w);
      out.block.push_back({w.col0, w.cols});
      const int64_t each = (w.cols + kTile - 1) / kTile;
      waves += each * heads, tiles += each * heads * ((rows + kTile - 1) / kTile);
    }
  }
  const bool split = waves < kPieceWaves;
  const int64_t least = std::max<int64_t>(kPieceTiles, (tiles + kPieceWaves - 1) / kPieceWaves);
  for (const AttnWork& w : all) {
    std::vector<AttnWork>& to = w.step > 1 ? out.coop : out.lone;
    const int64_t have = ((int64_t)w.row1 - w.row0 + kTile - 1) / kTile;
    const int64_t per = std::max<int64_t>(least, (have + kMaxSlots - 1) / kMaxSlots);
    out.long_rows |= have > 1;
    if (!split || have < 2 * per) {
      to.push_back(w);
      continue;
    }
    AttnWork piece = w;
    piece.slots = (int)((have + per - 1) / per), piece.slot0 = out.slots;
    for (int i = 0; i < piece.slots; ++i) {
      piece.row0 = (int)(w.row0 + i * per * kTile);
      piece.row1 = (int)std::min<int64_t>(w.row1, w.row0 + (i + 1) * per * kTile);
      piece.slot = out.slots;
      out.slots += w.step;
      to.push_back(piece);
    }
    for (int k = 0; k * kTile < w.cols; ++k)
      out.join.push_back({w.col0 + k * kTile, std::min(kTile, w.cols - k * kTile), piece.slot0 + k, piece.slots, w.step});
  }
  // One launch joins all where there are few blocks; else those of a few pieces go first, by a launch of their own.
  const bool one = out.join.size() <= 64;
  const auto few = std::stable_partition(out.join.begin(), out.join.end(), [](const AttnJoin& j) { return j.slots <= kFewSlots; });
  out.few = one && few != out.join.end() ? 0 : (int)(few - out.join.begin());
  return out;
}

// All lists of a plan in one device allocation: packed on the host, copied once, pointers set afterwards.
struct Packed {
  std::vector<char> host;
  std::vector<std::pair<void**, size_t>> at;
  template <typename E>
  void add(const std::vector<E>& v, E** dev) {
    if (v.empty()) return;
    at.push_back({(void**)dev, host.size()});
    const size_t bytes = (v.size() * sizeof(E) + 63) & ~(size_t)63;
    host.resize(host.size() + bytes);
    memcpy(host.data() + at.back().second, v.data(), v.size() * sizeof(E));
  }
  void add(const Lists& l, vsn_attn::Side& s) {
    s.small = (int)l.small.size(), s.pair = (int)l.pair.size(), s.lone = (int)l.lone.size(), s.coop = (int)l.coop.size();
    s.joins = (int)l.join.size(), s.few = l.few, s.slots = l.slots;
    s.blocks = (int)l.block.size(), s.long_rows = l.long_rows;
    add(l.small, &s.small_work);
    add(l.pair, &s.pair_work);
    add(l.lone, &s.lone_work);
    add(l.coop, &s.coop_work);
    add(l.join, &s.join);
    add(l.block, &s.block);
  }
  bool upload(char** dev) {
    if (host.empty()) return true;
    if (hipMalloc((void**)dev, host.size()) != hipSuccess) return false;
    if (hipMemcpy(*dev, host.data(), host.size(), hipMemcpyHostToDevice) != hipSuccess) return false;
    for (auto& a : at) *a.first = *dev + a.second;
    return true;
  }
};

bool ranges_ok(int64_t n, const int64_t* start, const int64_t* end) {
  if (!start || !end) return false;
  for (int64_t f = 0; f < n; ++f)
    if (end[f] < start[f] || start[f] != (f ? end[f - 1] : 0)) return false;
  return end[n - 1] <= (int64_t)1 << 30;
}

// Workers per head of the dq pass: each adds up the slope's and the table's gradient over its items and leaves one
// partial sum, so their number is bounded, and more tightly where a partial sum is a large table.
int workers(int items, int heads, int n_rel, int most) {
  int64_t cap = std::max(1, most / heads);
  if (n_rel) cap = std::min<int64_t>(cap, std::max<int64_t>(32, ((int64_t)1 << 24) / ((int64_t)n_rel * heads)));
  return (int)std::min<int64_t>(items, cap);
}

constexpr int64_t kMaxRowStep = (int64_t)1 << 25;

// A launch has fewer than 2^32 threads along an axis: whole workgroups of four waves here.  (Joins have fewer: there are
// none from kPieceWaves waves on; the backward passes' workers are bounded by workers().)
constexpr int64_t kMostGroups = ((int64_t)1 << 24) - 1;
bool countable(const Lists& l, int heads, int kv_heads) {
  const int64_t small = l.small.size(), lone = l.lone.size(), coop = l.coop.size();
  const int64_t waves = std::max(lone * heads, small * small_groups((int)small, kv_heads));
  return (waves + 3) / 4 <= kMostGroups && coop * heads <= kMostGroups;
}
// workgroups of the backward pass's last launch (join_launch): positions by block and fragment, slopes, table
bool joinable(const vsn_attn& a, const vsn_attn_grads& g) {
  int64_t n = g.dslope ? a.heads : 0;
  if (g.dtable) n += (int64_t)a.heads * a.n_buckets;
  const int64_t small = small_groups(a.by_query.small, a.kv_heads) > 1 ? a.by_query.small : 0;
  if (g.dpos) n += a.by_key.blocks + a.by_query.pair + small;
  if (g.dquery_pos) n += a.by_query.blocks + a.by_query.pair + small;
  return n <= kMostGroups;
}

struct Workspace {
  int64_t size = 0;
  int64_t take(int64_t bytes) {
    const int64_t at = size;
    size += (bytes + 255) & ~(int64_t)255;
    return at;
  }
};

struct BackwardSpace {
  int64_t delta, pos_q, pos_k, slope, hist, ml, o, o2, g, size;
  AttnWorkers workers;
  int parts;
};

BackwardSpace backward_space(const vsn_attn& a, int64_t rows_q, int64_t rows_k, bool pos, bool table) {
  BackwardSpace s;
  s.workers.lone = workers(a.by_query.lone, a.heads, a.n_rel, a.n_rel ? 2048 : 4096);
  s.workers.coop = workers(a.by_query.coop, a.heads, a.n_rel, 2048);
  s.workers.small = workers(a.by_query.small, 1, a.n_rel * a.heads, 4096);
  s.workers.pair = workers(a.by_query.pair, a.heads, a.n_rel, 4096);
  s.parts = s.workers.lone + s.workers.coop + s.workers.small + s.workers.pair;
  Workspace w;
  s.delta = w.take(rows_q * a.heads * 8);
  s.pos_q = w.take(pos ? rows_q * a.heads * 12 : 0);
  s.pos_k = w.take(pos ? rows_k * a.kv_heads * 12 : 0);
  s.slope = w.take((int64_t)s.parts * a.heads * kCoopWaves * 4);
  s.hist = w.take(table ? (int64_t)s.parts * a.heads * a.n_rel * 4 : 0);
  // pieces: the dq pass and the dk / dv pass use the same space one after the other
  const int64_t q_cols = (int64_t)a.by_query.slots * a.heads * kTile, k_cols = (int64_t)a.by_key.slots * a.kv_heads * kTile;
  s.ml = w.take(q_cols * 8);
  s.o = w.take(std::max(q_cols, k_cols) * a.dim * 4);
  s.o2 = w.take(k_cols * a.dim * 4);
  s.g = w.take(pos ? std::max(q_cols, k_cols) * 16 : 0);
  s.size = w.size;
  return s;
}

int64_t forward_space(const vsn_attn& a, int64_t* ml) {
  Workspace w;
  const int64_t rows = (int64_t)a.fwd.slots * a.heads * kTile;
  w.take(rows * a.dim * 4);
  const int64_t at = w.take(rows * 8);
  if (ml) *ml = at;
  return w.size;
}

bool lines_up(const void* p, int64_t row, int64_t head, int heads, int dim, int size) {
  const int64_t step = 16 / size;
  // (rows further apart than kMaxRowStep elements would overflow a lane's 32-bit offset within a tile)
  return p && (uintptr_t)p % 16 == 0 && row % step == 0 && head % step == 0 && row >= 0 && row <= kMaxRowStep &&
         head >= 0 && (heads == 1 || head >= dim);
}

// rows and heads of an output that do not run into one another
bool apart(int64_t rows, int64_t row, int heads, int64_t head, int dim) {
  if (rows > 1 && row < dim) return false;
  if (heads > 1 && head < dim) return false;
  return rows <= 1 || heads <= 1 || row >= (heads - 1) * head + dim || head >= (rows - 1) * row + dim;
}

bool io_ok(const vsn_attn& a, const vsn_attn_io& io) {
  if (io.dtype < VSN_F32 || io.dtype > VSN_F16) return false;
  const int size = io.dtype == VSN_F32 ? 4 : 2;
  if (io.rows_q < a.used_q || io.rows_k < a.used_k || io.rows_q > (int64_t)1 << 30 || io.rows_k > (int64_t)1 << 30)
    return false;
  if (a.used_q && !lines_up(io.q, io.q_row, io.q_head, a.heads, a.dim, size)) return false;
  if (a.used_k && (!lines_up(io.k, io.k_row, io.k_head, a.kv_heads, a.dim, size) ||
                   !lines_up(io.v, io.v_row, io.v_head, a.kv_heads, a.dim, size)))
    return false;
  if (io.slope && ((a.used_q && !io.q_pos) || (a.used_k && !io.k_pos))) return false;
  if (io.table && (!a.n_rel || (a.used_q && !io.q_res) || (a.used_k && !io.k_res))) return false;
  return true;
}

AttnParams params(const vsn_attn& a, const vsn_attn_io& io) {
  AttnParams p = {};
  p.heads = a.heads, p.kv_heads = a.kv_heads, p.dim = a.dim;
  p.reach = a.reach, p.n_rel = a.n_rel, p.n_buckets = a.n_buckets, p.lut = a.lut;
  p.q = io.q, p.k = io.k, p.v = io.v;
  p.q_row = io.q_row, p.q_head = io.q_head, p.k_row = io.k_row, p.k_head = io.k_head, p.v_row = io.v_row,
  p.v_head = io.v_head;
  p.q_pos = io.q_pos, p.k_pos = io.k_pos, p.slope = io.slope;
  p.q_res = io.q_res, p.k_res = io.k_res, p.table = io.table;
  p.scale = io.scale;
  p.rows_q = io.rows_q, p.rows_k = io.rows_k;
  p.out = io.out, p.out_row = io.out_row, p.out_head = io.out_head;
  p.stats = (float2*)io.stats;
  return p;
}

}  // namespace
}  // namespace vsn

extern "C" int vsn_attn_create(vsn_attn_handle* out, int device_id, int64_t n, const int64_t* host_start,
                               const int64_t* host_end, const int64_t* host_query_start, const int64_t* host_query_end,
                               int heads, int kv_heads, int head_dim, int reach, const int32_t* host_buckets,
                               int n_buckets) {
  using namespace vsn;
  if (!out) return -22;
  *out = nullptr;
  if (n <= 0 || n > (int64_t)1 << 30 || !ranges_ok(n, host_start, host_end)) return -22;
  if ((host_query_start != nullptr) != (host_query_end != nullptr)) return -22;
  if (host_query_start && !ranges_ok(n, host_query_start, host_query_end)) return -22;
  if (heads < 1 || heads > 1024 || kv_heads < 1 || heads % kv_heads || head_dim < 8 || head_dim > 128 || head_dim % 8)
    return -22;
  if (n_buckets < 0 || (n_buckets && !host_buckets) || reach < 0 || reach > kMaxReach) return -22;
  if (n_buckets > 4096) return -22;
  if (n_buckets)
    for (int i = 0; i < 2 * reach + 1; ++i)
      if (host_buckets[i] < 0 || host_buckets[i] >= n_buckets) return -22;
  const int64_t* qs = host_query_start ? host_query_start : host_start;
  const int64_t* qe = host_query_start ? host_query_end : host_end;
  vsn_attn* a = nullptr;
  bool ok = false;
  try {
    a = new vsn_attn();
    a->device = device_id, a->heads = heads, a->kv_heads = kv_heads, a->dim = head_dim;
    a->used_q = qe[n - 1], a->used_k = host_end[n - 1];
    a->same_rows = std::equal(qe, qe + n, host_end);
    std::vector<int> lut;
    if (n_buckets) {
      a->reach = reach, a->n_rel = 2 * reach + 1, a->n_buckets = n_buckets;
      lut.assign(host_buckets, host_buckets + a->n_rel);
    }
    // One-tile fragments go by a kernel of their own where a wave's per-head sums fit its share of LDS - and where there
    // are enough of them, or nothing else: a launch for a few next to others costs more than the tiles it saves (8 read-out
    // rows, one of them over one tile: 33.5 us with a launch of its own, 29.1 without; a protein of 175 atoms and two fragments,
    // forward, 21.0 and 18.1).  4096 fragments gain by it, from 34 to 256 (a thirtieth of them of two tiles) the other kernels
    // take 0.78 ... 1.0 of its time, at 512 both directions f32 1.17 and bf16 0.99: the border is on the low side.
    int64_t tiles = 0;
    for (int64_t f = 0; f < n; ++f) tiles += host_end[f] - host_start[f] <= kTile && qe[f] - qs[f] <= kTile;
    const bool small = heads <= 64 && (int64_t)heads * a->n_rel <= kSmallSums && (tiles >= 32 || tiles == n);
    const bool pair = heads == kv_heads && head_dim <= 64;  // (wider or shared heads would not fit its registers)
    const Lists fwd = make_lists(n, qs, qe, host_start, host_end, heads, head_dim, small, false);
    const Lists by_query = make_lists(n, qs, qe, host_start, host_end, heads, head_dim, small, pair);
    const Lists by_key = make_lists(n, host_start, host_end, qs, qe, kv_heads, head_dim, small, pair);
    if (!countable(fwd, heads, kv_heads) || !countable(by_query, heads, kv_heads) || !countable(by_key, kv_heads, kv_heads)) {
      delete a;
      return -22;
    }
    DeviceScope scope(device_id);
    if (!scope.ok) {
      delete a;
      return -19;
    }
    Packed all;
    all.add(fwd, a->fwd);
    all.add(by_query, a->by_query);
    all.add(by_key, a->by_key);
    all.add(lut, &a->lut);
    ok = all.upload(&a->lists);
  } catch (...) {  // out of host memory
    ok = false;
  }
  if (!ok) {
    (void)hipGetLastError();
    vsn_attn_destroy(a);
    return -12;
  }
  *out = a;
  return 0;
}

extern "C" void vsn_attn_destroy(vsn_attn_handle a) {
  if (!a) return;
  vsn::DeviceScope scope(a->device);
  hipFree(a->lists);
  delete a;
}

extern "C" int64_t vsn_attn_workspace(vsn_attn_handle a, int64_t rows_q, int64_t rows_k, int backward) {
  if (!a || rows_q < a->used_q || rows_k < a->used_k || backward < 0 || backward > 7) return -22;
  if (!(backward & VSN_ATTN_BACKWARD)) return vsn::forward_space(*a, nullptr);
  return vsn::backward_space(*a, rows_q, rows_k, !(backward & VSN_ATTN_NO_POS), !(backward & VSN_ATTN_NO_TABLE)).size;
}

extern "C" int vsn_attn_forward(vsn_attn_handle a, const vsn_attn_io* io, void* dev_workspace, int64_t workspace_bytes,
                                void* stream) {
  using namespace vsn;
  if (!a || !io || !io_ok(*a, *io)) return -22;
  if (a->used_q && (!lines_up(io->out, io->out_row, io->out_head, a->heads, a->dim, io->dtype == VSN_F32 ? 4 : 2) ||
                    !apart(io->rows_q, io->out_row, a->heads, io->out_head, a->dim)))
    return -22;
  int64_t ml = 0;
  const int64_t need = forward_space(*a, &ml);
  if (need && (!dev_workspace || (uintptr_t)dev_workspace % 16 || workspace_bytes < need)) return -22;
  DeviceScope scope(a->device);
  if (!scope.ok) return -19;
  AttnParams p = params(*a, *io);
  p.part_o = (float*)dev_workspace;
  p.part_ml = (float2*)((char*)dev_workspace + ml);
  return attn_forward(io->dtype, a->fwd.view(), p, (hipStream_t)stream);
}

extern "C" int vsn_attn_backward(vsn_attn_handle a, const vsn_attn_io* io, const vsn_attn_grads* g,
                                 void* dev_workspace, int64_t workspace_bytes, void* stream) {
  using namespace vsn;
  if (!a || !io || !g || !io_ok(*a, *io)) return -22;
  const int size = io->dtype == VSN_F32 ? 4 : 2;
  if (a->used_q && (!io->stats || !lines_up(g->dout, g->dout_row, g->dout_head, a->heads, a->dim, size) || !g->dq))
    return -22;
  if (a->used_k && (!g->dk || !g->dv)) return -22;
  if ((uintptr_t)g->dq % 16 || (uintptr_t)g->dk % 16 || (uintptr_t)g->dv % 16) return -22;
  if ((g->dpos || g->dquery_pos || g->dslope) && !io->slope) return -22;
  if (g->dquery_pos && !g->dpos) return -22;
  // one gradient for both ends of a pair: they have to be the same atoms
  if (g->dpos && !g->dquery_pos && (!a->same_rows || io->rows_q != io->rows_k || io->q_pos != io->k_pos)) return -22;
  if (g->dtable && !io->table) return -22;
  if (!joinable(*a, *g)) return -22;
  const BackwardSpace s = backward_space(*a, io->rows_q, io->rows_k, g->dpos != nullptr, g->dtable != nullptr);
  if (s.size && (!dev_workspace || (uintptr_t)dev_workspace % 16 || workspace_bytes < s.size)) return -22;
  DeviceScope scope(a->device);
  if (!scope.ok) return -19;
  char* base = (char*)dev_workspace;
  AttnParams p = params(*a, *io);
  p.dout = g->dout, p.do_row = g->dout_row, p.do_head = g->dout_head;
  p.delta = (float2*)(base + s.delta);
  p.dq = g->dq, p.dk = g->dk, p.dv = g->dv;
  p.parts = s.parts;
  if (g->dpos) {
    p.part_pos_q = (float*)(base + s.pos_q);
    p.part_pos_k = (float*)(base + s.pos_k);
  }
  p.part_ml = (float2*)(base + s.ml);
  p.part_o = (float*)(base + s.o), p.part_o2 = (float*)(base + s.o2), p.part_g = (float*)(base + s.g);
  if (g->dslope) p.part_slope = (float*)(base + s.slope);
  if (g->dtable) p.part_hist = (float*)(base + s.hist);
  p.dpos = g->dpos, p.dq_pos = g->dquery_pos, p.dslope = g->dslope, p.dtable = g->dtable;
  return attn_backward(io->dtype, a->by_query.view(), a->by_key.view(), p, s.workers, (hipStream_t)stream);
}
