// What the kernels of the branch attention share: the parameters, and how its work is laid out in
// a line of units and cut into one part per worker. Every kernel computes that from the lengths on
// the device, a warp at a time, so all of them agree on it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>

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
// of each branch against its own, KV head by KV head; an item has a unit for every `unit` keys and
// weighs `pad` more, which is about what starting and ending it costs.
struct Line {
  int span, unit, pad;
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

__device__ __forceinline__ int seq_length(const BranchParams& p, int b) {
  const int n = __ldg(p.lengths + b);
  return max(0, min(n, p.width * kBlk));
}

// A sequence that ends inside the shared blocks has no part in their items, where rows behind its end that
// others see would meet its zeros of P, and NaN or infinities among them its output: its own items
// have all its keys.
__device__ __forceinline__ bool takes_shared(const BranchParams& p, int len) { return len >= p.shared_keys; }
// The first key outside the shared items, and the units behind it of the rows of tile t of a
// sequence of length `len`.
__device__ __forceinline__ int own_lo(const BranchParams& p, int len) { return takes_shared(p, len) ? p.shared_keys : 0; }
__device__ __forceinline__ int own_limit(const BranchParams& p, const Line& ln, int len, int t) {
  if (!p.causal) return len;
  const int last = min((t + 1) * ln.span, p.rows * p.group) - 1;
  return len - (p.rows - 1 - last / p.group);
}
__device__ __forceinline__ int own_units(const BranchParams& p, const Line& ln, int len, int t) {
  return max(0, own_limit(p, ln, len, t) - own_lo(p, len) + ln.unit - 1) / ln.unit;
}
__device__ __forceinline__ int weight_of(const Line& ln, int units) { return units > 0 ? units + ln.pad : 0; }
__device__ __forceinline__ int own_weight_all(const BranchParams& p, const Line& ln, int len) {
  if (!p.causal) return weight_of(ln, own_units(p, ln, len, 0)) * ln.own_tiles;
  int n = 0;
  for (int t = 0; t < ln.own_tiles; ++t) n += weight_of(ln, own_units(p, ln, len, t));
  return n;
}

struct Plan {
  int shared_blocks;  // of the shared items: 0 if no sequence has all of them
  int shared_units;   // units of one shared item
  int head_weight;    // one KV head's part of the line
  int cut;            // one worker's part
  int longest;        // sequence whose table row gives the shared pages
};

__device__ __forceinline__ Plan make_plan(const BranchParams& p, const Line& ln, int lane) {
  int own = 0, best = -1, at = 0;
  for (int b = lane; b < p.batch; b += 32) {
    const int len = seq_length(p, b);
    own += own_weight_all(p, ln, len);
    if (len > best) {
      best = len;
      at = b;
    }
  }
  own = __reduce_add_sync(0xffffffffu, own);
  const int top = __reduce_max_sync(0xffffffffu, best);
  at = __reduce_min_sync(0xffffffffu, best == top ? at : INT_MAX);
  Plan pl;
  pl.longest = at;
  pl.shared_blocks = own_lo(p, top) / kBlk;
  pl.shared_units = pl.shared_blocks * (kBlk / ln.unit);
  pl.head_weight = ln.shared_tiles * weight_of(ln, pl.shared_units) + own;
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
__device__ __forceinline__ Place locate(const BranchParams& p, const Line& ln, const Plan& pl, int u, int lane) {
  Place at;
  at.head = u / pl.head_weight;
  at.b = -1;
  at.t = 0;
  int x = u - at.head * pl.head_weight;
  const int w = weight_of(ln, pl.shared_units);
  if (x < ln.shared_tiles * w) {
    at.t = x / w;
    at.off = x - at.t * w;
    return at;
  }
  x -= ln.shared_tiles * w;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + lane;
    const int n = b < p.batch ? own_weight_all(p, ln, seq_length(p, b)) : 0;
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
  const int len = seq_length(p, at.b);
  for (int v; x >= (v = weight_of(ln, own_units(p, ln, len, at.t))); ++at.t) x -= v;
  at.off = x;
  return at;
}

// To the next item that has units; there must be one.
__device__ __forceinline__ void step_item(const BranchParams& p, const Line& ln, const Plan& pl, Place& at) {
  const bool shared = ln.shared_tiles > 0 && pl.shared_units > 0;
  at.off = 0;
  if (at.b < 0) {
    if (++at.t < ln.shared_tiles) return;
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
    if (ln.own_tiles > 0 && own_units(p, ln, seq_length(p, at.b), at.t) > 0) return;
  }
}
__device__ __forceinline__ int place_units(const BranchParams& p, const Line& ln, const Plan& pl, const Place& at) {
  return at.b < 0 ? pl.shared_units : own_units(p, ln, seq_length(p, at.b), at.t);
}

// Writes a line's schedule down for the merge: the shared units, a head's and a worker's part, and
// what lies in front of each sequence's own items.
__device__ __forceinline__ void write_plan(const BranchParams& p, const Line& ln, const Plan& pl, int* out, int lane) {
  if (lane == 0) {
    out[0] = pl.shared_blocks;
    out[1] = pl.head_weight;
    out[2] = pl.cut;
  }
  int before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + lane;
    const int n = b < p.batch ? own_weight_all(p, ln, seq_length(p, b)) : 0;
    int cum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, cum, d);
      if (lane >= d) cum += v;
    }
    if (b < p.batch) out[3 + b] = before + cum - n;
    before += __shfl_sync(0xffffffffu, cum, 31);
  }
}

__device__ __forceinline__ void flag_lengths(const BranchParams& p, int lane) {
  for (int b = lane; b < p.batch; b += 32) {
    const int n = __ldg(p.lengths + b);
    if ((n < 0 || n > p.width * kBlk) && p.err) atomicOr(p.err, kErrBadIndex);
  }
}

// A stacked row (branch, row, query head of the KV head's group).
struct RowAt {
  int b, i, h;
};
__device__ __forceinline__ RowAt row_at(const BranchParams& p, int head, int r) {
  const int bi = r / p.group;
  RowAt a;
  a.h = head * p.group + (r - bi * p.group);
  a.b = bi / p.rows;
  a.i = bi - a.b * p.rows;
  return a;
}

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

// Tensor map of a pool with boxes of `rows` rows of 128 bytes, 128-byte swizzle.
int encode_pool(CUtensorMap* map, const BranchParams& p, const void* pool, bool e4m3, int rows);

}  // namespace h3sa
