// What the kernels of the branch attention share: the parameters, and how its work is laid out in
// a line of units and cut into one part per worker. Every kernel computes that from the lengths on
// the device, a warp at a time, so all of them agree on it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>
#include <type_traits>

#include "h3sa_div.cuh"
#include "h3sa_host.h"
#include "h3sa_ptx.cuh"

namespace h3sa {

constexpr int kD = 128;    // head dimension
constexpr int kBlk = 128;  // KV rows of a block (a page)
constexpr int kSpan = 256;     // query rows of an item of the tensor line: two tiles
constexpr int kRowSpan = 16;   // query rows of an item of the warp line
constexpr int kRowUnit = 32;   // keys of a unit of the warp line
constexpr int kRowWarpsPerBlock = 4;
// P = 2^(x - m + boost). m follows a row's maximum only when that grows past it by more than kGrowth, so P is
// at most 2^(kGrowth + boost) and O is seldom rescaled. bf16 caches take P in bf16, which holds any of these,
// with no boost; e4m3 caches take it in f16, 11 bits from 2^-14 to 2^16: the boost puts a fresh maximum at
// 2^7, so that weights of 2^-21 of it have all bits and the last step is 2^-31 of it.
constexpr float kGrowth = 8.0f;
constexpr float kBoostF8 = 7.0f;

// A line: items of up to `span` query rows, first those against the shared blocks and then those
// of each branch against its own, KV head by KV head; an item has a unit for every `unit` keys, each
// weighs `few` or, in an item of more than 128 rows, `many`, and the item `pad` more, which is about what starting and
// ending it costs.
struct Line {
  int span, unit, pad, few, many;
  int shared_tiles;  // items per KV head against the shared blocks (0: the other line has them)
  int own_tiles;     // items per KV head and branch against its own (0: the other line has them)
  int workers;
  int least;  // a worker's part is at least this
};

struct BranchParams {
  const __nv_bfloat16* q;
  long long q_sb, q_sn, q_sh;  // element strides of [batch, rows, heads, 128]
  __nv_bfloat16* out;          // contiguous [batch, rows, heads, 128]
  float* lse;                  // contiguous [batch, rows, heads] or null
  const int* table;            // [batch, width]
  const int* lengths;          // [batch]
  int width, batch, rows, heads, kv_heads, group;
  Divisor rows_div, group_div, own_div, stacked_div;  // of rows, group, rows * group, batch * rows * group
  int shared_keys;             // leading keys of the shared items (0: there are none), whole blocks
  int causal, joint;
  int whole;                   // the warp line takes whole items
  int pool_pages;
  float scale_log2;
  const float* k_scale;        // e4m3: [kv_heads]
  const float* v_scale;
  const void* key_pool;        // [kv_heads, pool_pages * 128, 128]
  const void* value_pool;
  Line tensor, warp;           // workers: CTAs, warps
  int shared_slot_rows, own_slot_rows;
  long long own_row0;          // first workspace row of the own items' slots
  float* part_o;               // [workspace rows, 128]
  float2* part_ml;             // [workspace rows]: (maximum, sum)
  int* plan;                   // for the merge: [3 + batch] of the tensor line, then of the warp line
  int* err;
};

// New rows that are the nodes of a drafted tree: they lie behind the first lengths[b] rows, and row i sees
// those and the nodes of its mask.
struct TreeParams : BranchParams {
  const uint32_t* masks;  // [batch, rows, words]: bit n of row i: node n is node i or above it
  const int* counts;      // [batch] nodes, or null: `rows` of each
  int words;
  int compact;            // shared items are stacked of rows that there are (up to kMaxStack sequences)
};
constexpr int kMaxStack = 256;
// Header of a line's schedule as the merge reads it; own offsets [batch] and, of the line with the shared items, the
// stacked rows in front of each sequence [batch] follow.
constexpr int kPlanHead = 4;
template <class P>
constexpr bool is_tree = std::is_same_v<P, TreeParams>;

// Rows of a sequence: all keys, and those that each of its new rows may see; `rows`: of its stacked query rows, those
// that there are (of a tree the nodes', the rest of its rows come out zero).
struct Extent {
  int all, clean, rows;
};
__device__ __forceinline__ int clean_rows(const BranchParams& p, int b) {
  const int n = __ldg(p.lengths + b);
  return max(0, min(n, p.width * kBlk));
}
__device__ __forceinline__ Extent extent_of(const BranchParams& p, int b) {
  const int n = clean_rows(p, b);
  return Extent{n, n, p.rows * p.group};
}
__device__ __forceinline__ Extent extent_of(const TreeParams& p, int b) {
  const int n = clean_rows(p, b);
  const int nodes = p.counts ? max(0, min(__ldg(p.counts + b), p.rows)) : p.rows;
  const int all = min(n + nodes, p.width * kBlk);
  return Extent{all, n, (all - n) * p.group};
}

// A sequence that ends inside the shared blocks has no part in their items, where rows behind its end that
// others see would meet its zeros of P, and NaN or infinities among them its output: its own items
// have all its keys.
__device__ __forceinline__ bool takes_shared(const BranchParams& p, const Extent& x) { return x.clean >= p.shared_keys; }
// The first key outside the shared items, and the units behind it of the rows of tile t of a
// sequence.
__device__ __forceinline__ int own_lo(const BranchParams& p, const Extent& x) { return takes_shared(p, x) ? p.shared_keys : 0; }
__device__ __forceinline__ int own_limit(const BranchParams& p, const Line& ln, const Extent& x, int t) {
  if (!p.causal) return x.all;
  const int last = min((t + 1) * ln.span, p.rows * p.group) - 1;
  return x.all - (p.rows - 1 - static_cast<int>(quotient(last, p.group_div)));
}
template <class P>
__device__ __forceinline__ int own_units(const P& p, const Line& ln, const Extent& x, int t) {
  if (is_tree<P> && t * ln.span >= x.rows) return 0;
  return over_pow2(max(0, own_limit(p, ln, x, t) - own_lo(p, x) + ln.unit - 1), ln.unit);
}
// What a unit of an item of `rows` rows weighs: 1, or of the tensor line in a tree's call one of the two below (of
// chains all weigh the same). Blocks of up to 128 and of more rows take a CTA 1.5 to 1.75 and 2.6 us (e4m3 1.1 and 2.1), and
// an item 4 to 6 us (8 to 12) from its last scores to the next one's first. Weight of an item, 12 / 16 / 20 (us): 24 trees of 96
// rows over 9000 keys 113.4 / 111.5 / 112.1, 12 trees of up to 240 over shared and own keys 74.2 / 72.6 / 73.6; e4m3, 16 / 24 / 40: wide
// trees 188.7 / 188 / 186, 24 trees of 64 rows over 16000 keys 163 / 160 / 158.
constexpr int kFewCost = 5, kManyCost = 8, kTreePad = 16, kTreePadF8 = 40;
template <class P>
__device__ __forceinline__ int cost_of(const P&, const Line& ln, int rows) {
  return is_tree<P> ? (rows > kBlk ? ln.many : ln.few) : 1;
}
template <class P>
__device__ __forceinline__ int own_cost(const P& p, const Line& ln, const Extent& x, int t) { return cost_of(p, ln, x.rows - t * ln.span); }
__device__ __forceinline__ int weight_of(const Line& ln, int units, int cost) { return units > 0 ? units * cost + ln.pad : 0; }
template <class P>
__device__ __forceinline__ int own_weight(const P& p, const Line& ln, const Extent& x, int t) {
  return weight_of(ln, own_units(p, ln, x, t), own_cost(p, ln, x, t));
}
template <class P>
__device__ __forceinline__ int own_weight_all(const P& p, const Line& ln, const Extent& x) {
  if constexpr (is_tree<P>) {  // all live tiles but the last are full
    const int tiles = min(ln.own_tiles, over_pow2(x.rows + ln.span - 1, ln.span));
    return tiles == 0 ? 0 : own_weight(p, ln, x, 0) * (tiles - 1) + own_weight(p, ln, x, tiles - 1);
  }
  if (!p.causal) return own_weight(p, ln, x, 0) * ln.own_tiles;
  int n = 0;
  for (int t = 0; t < ln.own_tiles; ++t) n += own_weight(p, ln, x, t);
  return n;
}

// Rows of a sequence among those stacked for the shared items.
template <class P>
__device__ __forceinline__ int stacked_of(const P& p, const Extent& x) {
  if constexpr (is_tree<P>) return p.compact ? (takes_shared(p, x) ? x.rows : 0) : p.rows * p.group;
  return p.rows * p.group;
}
template <class P>
__device__ __forceinline__ int live_tiles(const P&, const Line& ln, int live) {
  if constexpr (is_tree<P>) return min(ln.shared_tiles, over_pow2(live + ln.span - 1, ln.span));
  return ln.shared_tiles;
}

// What a KV head's shared items weigh, from the units of one; all but the last one of a tree's call weigh the same.
template <class P>
__device__ __forceinline__ int shared_cost(const P& p, const Line& ln, int live, int t) { return cost_of(p, ln, live - t * ln.span); }
template <class P>
__device__ __forceinline__ int shared_weight_all(const P& p, const Line& ln, int units, int live, int tiles) {
  return tiles == 0 ? 0 : weight_of(ln, units, shared_cost(p, ln, live, 0)) * (tiles - 1) +
                              weight_of(ln, units, shared_cost(p, ln, live, tiles - 1));
}

struct Plan {
  int shared_blocks;  // of the shared items: 0 if no sequence has all of them
  int shared_units;   // units of one shared item
  int live;           // stacked rows
  int shared_tiles;   // shared items a KV head
  int shared_weight;  // of one of them, but perhaps the last
  int shared_all;     // of all of them
  int head_weight;    // one KV head's part of the line
  int cut;            // one worker's part
  int longest;        // sequence whose table row gives the shared pages
};

template <class P>
__device__ __forceinline__ Plan make_plan(const P& p, const Line& ln, int lane) {
  int own = 0, best = -1, at = 0, live = 0;
  for (int b = lane; b < p.batch; b += 32) {
    const Extent x = extent_of(p, b);
    own += own_weight_all(p, ln, x);
    live += stacked_of(p, x);
    if (x.clean > best) {
      best = x.clean;
      at = b;
    }
  }
  own = __reduce_add_sync(0xffffffffu, own);
  if constexpr (is_tree<P>) live = __reduce_add_sync(0xffffffffu, live);
  else live = p.batch * p.rows * p.group;
  const int top = __reduce_max_sync(0xffffffffu, best);
  at = __reduce_min_sync(0xffffffffu, best == top ? at : INT_MAX);
  Plan pl;
  pl.longest = at;
  pl.shared_blocks = own_lo(p, Extent{top, top, 0}) / kBlk;
  pl.shared_units = pl.shared_blocks * over_pow2(kBlk, ln.unit);
  pl.live = live;
  pl.shared_tiles = live_tiles(p, ln, live);
  pl.shared_weight = weight_of(ln, pl.shared_units, shared_cost(p, ln, live, 0));
  pl.shared_all = shared_weight_all(p, ln, pl.shared_units, live, pl.shared_tiles);
  pl.head_weight = pl.shared_all + own;
  const int all = pl.head_weight * p.kv_heads;
  pl.cut = max(ln.least, (all + ln.workers - 1) / ln.workers);
  return pl;
}

// A worker's place in the line: the item (a shared tile, b < 0, or tile t of branch b) and the
// offset in it.
struct Place {
  int head, b, t, off;
};

// The place of position `u` of the line (warp-collective).
template <class P>
__device__ __forceinline__ Place locate(const P& p, const Line& ln, const Plan& pl, int u, int lane) {
  Place at;
  at.head = u / pl.head_weight;
  at.b = -1;
  at.t = 0;
  int x = u - at.head * pl.head_weight;
  const int w = pl.shared_weight;
  if (x < pl.shared_all) {
    at.t = x / w;
    at.off = x - at.t * w;
    return at;
  }
  x -= pl.shared_all;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + lane;
    const int n = b < p.batch ? own_weight_all(p, ln, extent_of(p, b)) : 0;
    int cum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, cum, d);
      if (lane >= d) cum += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, cum > x);
    if (past) {
      const int f = __ffs(past) - 1;
      at.b = b0 + f;
      x -= __shfl_sync(0xffffffffu, cum - n, f);
      break;
    }
    x -= __shfl_sync(0xffffffffu, cum, 31);
  }
  const Extent ext = extent_of(p, at.b);
  for (int v; x >= (v = own_weight(p, ln, ext, at.t)); ++at.t) x -= v;
  at.off = x;
  return at;
}

// To the next item that has units; there must be one.
template <class P>
__device__ __forceinline__ void step_item(const P& p, const Line& ln, const Plan& pl, Place& at) {
  const bool shared = pl.shared_tiles > 0 && pl.shared_units > 0;
  at.off = 0;
  if (at.b < 0) {
    if (++at.t < pl.shared_tiles) return;
    at.b = 0;
    at.t = -1;
  }
  while (true) {
    if (++at.t >= ln.own_tiles) {
      at.t = 0;
      if (++at.b >= p.batch || ln.own_tiles == 0) {
        ++at.head;
        at.b = shared ? -1 : 0;
        if (shared) return;
      }
    }
    if (ln.own_tiles > 0 && own_units(p, ln, extent_of(p, at.b), at.t) > 0) return;
  }
}
// The item at a place: its units, and what each weighs.
struct PlaceUnits {
  int units, cost;
};
template <class P>
__device__ __forceinline__ PlaceUnits place_units(const P& p, const Line& ln, const Plan& pl, const Place& at) {
  if (at.b < 0) return PlaceUnits{pl.shared_units, shared_cost(p, ln, pl.live, at.t)};
  const Extent x = extent_of(p, at.b);
  return PlaceUnits{own_units(p, ln, x, at.t), own_cost(p, ln, x, at.t)};
}
// Its units that begin in [off, off + part) of it; part: what is left of the item or of the worker's own part.
struct UnitRange {
  int part, first, count;
};
__device__ __forceinline__ UnitRange units_in(const Line& ln, const PlaceUnits& it, int off, int left) {
  UnitRange r;
  r.part = min(weight_of(ln, it.units, it.cost) - off, left);
  const auto up = [&](int x) { return it.cost == 1 ? x : it.cost == kManyCost ? (x + kManyCost - 1) / kManyCost : (x + kFewCost - 1) / kFewCost; };
  r.first = up(off);
  r.count = min(it.units, up(off + r.part)) - r.first;
  return r;
}

// Stacked rows in front of each sequence's (warp-collective).
__device__ __forceinline__ void stack_rows(const TreeParams& p, int* before, int lane) {
  int sum = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + lane, n = b < p.batch ? stacked_of(p, extent_of(p, b)) : 0;
    int cum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, cum, d);
      if (lane >= d) cum += v;
    }
    if (b < p.batch) before[b] = sum + cum - n;
    sum += __shfl_sync(0xffffffffu, cum, 31);
  }
}

// Writes a line's schedule down for the merge: the shared units, a head's and a worker's part, the stacked rows, and
// what lies in front of each sequence's own items.
template <class P>
__device__ __forceinline__ void write_plan(const P& p, const Line& ln, const Plan& pl, int* out, int lane) {
  if (lane == 0) {
    out[0] = pl.shared_blocks;
    out[1] = pl.head_weight;
    out[2] = pl.cut;
    out[3] = pl.live;
  }
  if constexpr (is_tree<P>) {
    if (p.compact && ln.shared_tiles > 0) stack_rows(p, out + kPlanHead + p.batch, lane);
  }
  int before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + lane;
    const int n = b < p.batch ? own_weight_all(p, ln, extent_of(p, b)) : 0;
    int cum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, cum, d);
      if (lane >= d) cum += v;
    }
    if (b < p.batch) out[kPlanHead + b] = before + cum - n;
    before += __shfl_sync(0xffffffffu, cum, 31);
  }
}

__device__ __forceinline__ void flag_lengths(const BranchParams& p, int lane) {
  for (int b = lane; b < p.batch; b += 32) {
    const int n = __ldg(p.lengths + b);
    if ((n < 0 || n > p.width * kBlk) && p.err) atomicOr(p.err, kErrBadIndex);
  }
}
__device__ __forceinline__ void flag_lengths(const TreeParams& p, int lane) {
  for (int b = lane; b < p.batch; b += 32) {
    const int n = __ldg(p.lengths + b), nodes = p.counts ? __ldg(p.counts + b) : p.rows;
    const bool fits = n >= 0 && n <= p.width * kBlk && nodes >= 0 && nodes <= p.rows && n + nodes <= p.width * kBlk;
    if (!fits && p.err) atomicOr(p.err, kErrBadIndex);
  }
}

// A stacked row (branch, row, query head of the KV head's group).
struct RowAt {
  int b, i, h;
};
__device__ __forceinline__ RowAt row_at(const BranchParams& p, int head, int r) {
  const int bi = quotient(r, p.group_div);
  RowAt a;
  a.h = head * p.group + (r - bi * p.group);
  a.b = quotient(bi, p.rows_div);
  a.i = bi - a.b * p.rows;
  return a;
}

// What a node sees: all keys in front of `base`, and key base + n, n < count, if bit n of its mask says so. A row that
// has no part in an item (one behind the nodes, one without the shared blocks) is `hidden`: it goes through the item as if it
// saw everything, which costs least (hiding keys of such rows one by one took 111 us for 94), and what it
// has then is dropped.
struct Sight {
  int base, count, row;  // row of the masks
  __device__ __forceinline__ bool hidden() const { return base == INT_MAX; }
  __device__ __forceinline__ uint32_t word(const TreeParams& p, int w) const {
    const int rest = count - 32 * w;
    if (w < 0 || rest <= 0) return 0u;
    const uint32_t bits = __ldg(p.masks + static_cast<size_t>(row) * p.words + w);
    return rest >= 32 ? bits : bits & ((1u << rest) - 1u);
  }
  // bit j: whether it sees key + j
  __device__ __forceinline__ uint32_t seen32(const TreeParams& p, int key) const {
    const int x = key - base;
    if (x <= -32) return 0xffffffffu;
    if (x < 0) return (0xffffffffu >> (32 + x)) | (word(p, 0) << -x);
    return __funnelshift_r(word(p, x >> 5), word(p, (x >> 5) + 1), x & 31);
  }
};
__device__ __forceinline__ Sight sight_of(const TreeParams& p, const RowAt& ra, bool shared) {
  const Extent x = extent_of(p, ra.b);
  const int count = x.all - x.clean;
  if (ra.i >= count || (shared && !takes_shared(p, x))) return Sight{INT_MAX, 0, 0};
  return Sight{x.clean, count, ra.b * p.rows + ra.i};
}

// The r-th of the rows that there are, from what lies in front of each sequence's: it is in the last one that
// begins at or before it.
__device__ __forceinline__ RowAt live_row_at(const TreeParams& p, const int* before, int head, int r) {
  int lo = 0, hi = p.batch;  // before[lo] <= r < before[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (before[mid] <= r) lo = mid;
    else hi = mid;
  }
  r -= before[lo];
  RowAt a;
  a.b = lo;
  a.i = quotient(r, p.group_div);
  a.h = head * p.group + r - a.i * p.group;
  return a;
}

// Of a chain, only a limit.
struct Limit {
  int base;
};
__device__ __forceinline__ Limit sight_of(const BranchParams& p, const RowAt& ra, bool shared) {
  const Extent x = extent_of(p, ra.b);
  return Limit{shared && !takes_shared(p, x) ? 0 : x.all - (p.causal ? p.rows - 1 - ra.i : 0)};
}

// Infinities and NaN in V of a node must not reach rows that do not see it, whose P is zero there: they are
// taken out of V's tile in shared memory, and a row that does see such a node gets them back in the end.
// Two values of a word at a time; `top` are the exponent bits of one.
template <uint32_t kTop>
__device__ __forceinline__ uint32_t non_finite(uint32_t w) {  // 0xffff in each half that is an infinity or NaN
  constexpr uint32_t kLow = kTop & (0u - kTop);               // the exponent's lowest bit: all ones and it carry out
  const uint32_t carry = ((w & (kTop | kTop << 16)) + (kLow | kLow << 16)) & 0x80008000u;
  return (carry >> 15) * 0xffffu;
}

// V of the nodes of sequence b in a KV head, read from the pool again.
template <bool kFp8>
struct NodeValues {
  const uint8_t* pool;  // of the head
  const int* table;
  __device__ __forceinline__ NodeValues(const TreeParams& p, int b, int head)
      : pool(static_cast<const uint8_t*>(p.value_pool) +
             static_cast<size_t>(head) * p.pool_pages * kBlk * (kD * (kFp8 ? 1 : 2))),
        table(p.table + static_cast<size_t>(b) * p.width) {}
  // The infinities and NaN of column `col` in the nodes that a row sees, added up; 0 if there are none. Only of keys in
  // [from, to), and of every step-th (1 or 2) block there: those of other pieces are added to them, and here, where
  // this piece's weight may vanish, they would make NaN.
  __device__ __forceinline__ float non_finite_sum(const TreeParams& p, const Sight& sight, int col, int from, int to, int step) const {
    float sum = 0.f;
    if (sight.hidden()) return sum;
    for (int n = max(0, from - sight.base), end = min(sight.count, to - sight.base); n < end; ++n) {
      if (!(sight.word(p, n >> 5) >> (n & 31) & 1u) || (((sight.base + n - from) / kBlk) & (step - 1))) continue;
      const int key = sight.base + n, page = __ldg(table + key / kBlk);
      if (page < 0 || page >= p.pool_pages) continue;
      const size_t at = (static_cast<size_t>(page) * kBlk + key % kBlk) * kD + col;
      if constexpr (kFp8) {
        if ((pool[at] & 0x7fu) == 0x7fu) sum = __int_as_float(0x7fffffff);
      } else {
        const uint32_t v = reinterpret_cast<const uint16_t*>(pool)[at];
        if ((v & 0x7f80u) == 0x7f80u) sum += __uint_as_float(v << 16);
      }
    }
    return sum;
  }
};

__device__ __forceinline__ uint32_t f16x2_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t f16x2_of_e4m3x2(uint32_t e) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(e)));
  return r;
}

// The power of two that brings a bf16 row's largest magnitude (given as its bits) into [128, 256),
// as an exponent; rows of tiny numbers keep their products within fp32, rows of zeros are left alone.
__device__ __forceinline__ int row_exponent(uint32_t top) {
  return top == 0u ? 0 : max(-120, min(7 - (static_cast<int>(top >> 7) - 127), 120));
}
// The factor of e4m3 scores. Hidden ones are -inf before they are scaled, and -inf times a factor that is
// zero (a k_scale of zero) or came out as zero (tiny queries over tiny keys) would be NaN. With the
// smallest normal number instead, visible scores, at most 2^24, still come out as nothing.
__device__ __forceinline__ float score_factor(float f) { return f == 0.f ? 1.17549435e-38f : f; }
__device__ __forceinline__ float exp2_int(int k) { return __uint_as_float(static_cast<uint32_t>(k + 127) << 23); }

// A tile load that marks its lines as the first to go from L2. Keys that one worker alone reads would
// push everything else out of it, the kernels' own code and queries among it, whose next reads then
// queue behind them for memory: 109 -> 99 us for 60 rows over 98304 e4m3 keys of 8 heads.
__device__ __forceinline__ void tma_load_3d_once(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1,
                                                 int c2, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
      : "memory");
}

// Launches the warp line's kernel (h3sa_branch_rows.cu); `after`: along with another kernel, whose end
// the line then waits for as well. Returns an H3SA_* status.
int launch_branch_rows(const BranchParams& p, bool e4m3, bool after, cudaLaunchConfig_t cfg);
int launch_branch_rows(const TreeParams& p, bool e4m3, bool after, cudaLaunchConfig_t cfg);

// Tensor map of a pool with boxes of `rows` rows of 128 bytes, 128-byte swizzle.
int encode_pool(CUtensorMap* map, const BranchParams& p, const void* pool, bool e4m3, int rows);

}  // namespace h3sa
