// Branch attention for few query rows: the items of the warp line (h3sa_branch.cuh), up to 16 rows
// each against the shared blocks or a branch's own.
//
//   x_j = scale * q . k_j,   O = sum_j 2^(x_j' - m) v_j,   l = sum_j 2^(x_j' - m),   x' = x log2 e
//
// Sixteen rows use a key 2 * 16 * 2 * 128 flops for its 512 bytes: the kernel is bound by reading K
// and V, and for a branch's own few blocks by latency. So a warp works alone, with another that
// starts its copies: 48 KB of keys and values, three units of 32 keys or six in e4m3, are on their
// way from memory by TMA, across the ends of its items, and the four pairs of an SM have 192 KB in
// flight. A unit takes a warp 1200 cycles, 350 for S, 360 for the softmax and 440 for P V; when it
// started its copies itself, 1800. Reading straight into registers, which hold one unit, took 40.1 us
// where this takes 32.4 (60 rows of 8 KV heads over 4096 shared keys and up to 1000 of their own). One
// row of 24 heads over 16384 keys, 201 MB: 41.2 us, 0.75 of the measured copy rate with launch and merge.
//
// mma.m16n8k16 leaves the order of the contracted index open as long as both operands agree, and so
// the column order of the result, and the orders are chosen for the 128-byte swizzle of the tiles:
//   S = Q K^T: lane 4r + c takes, of key r of each group of eight, 32 bytes (two 16-byte chunks) of every
//      128; step s contracts four elements of them;
//   O += P V: lane 4r + c takes keys 2c, 2c + 1, 2c + 8, 2c + 9 of sixteen and chunk r of every 128 bytes of
//      each; two keys' words are woven into the operand's pairs by byte permutes.
// Either way the eight lanes of a phase read eight different chunks: no bank conflicts. e4m3 caches
// become f16 pairs, exactly, on the way; the query row is scaled by a power of two and taken as
// f16 (11 bits to bf16's 8), and P is f16 too.
#include <mutex>

#include "h3sa_branch.cuh"

namespace h3sa {
namespace {

constexpr int kRowWarps = kRowWarpsPerBlock;
constexpr int kRowRing = 48 * 1024;  // bytes a warp
constexpr int kMaxRowStages = 6;
template <bool kFp8>
struct RowCfg {
  static constexpr int kTileBytes = kRowUnit * kD * (kFp8 ? 1 : 2);  // K or V of a unit
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = kRowRing / kStageBytes;  // 3, and 6 for e4m3
};
constexpr size_t kRowSmem = static_cast<size_t>(kRowWarps) * kRowRing + 1024;

__device__ __forceinline__ void load16(const void* at, uint32_t* r) {
  const uint4 v = __ldg(static_cast<const uint4*>(at));
  r[0] = v.x;
  r[1] = v.y;
  r[2] = v.z;
  r[3] = v.w;
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}

template <bool kF16>
__device__ __forceinline__ void mma16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  if constexpr (kF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

// P of two groups of eight keys as operands of bf16 and of what that leaves off, 16 bits in all. P in
// bf16 adds as much to the error as the output's own rounding (0.0024 against 0.0017 relative). The
// second product is taken where it costs least, for few rows (6 over 1152 keys 9.9 -> 10.0 us, 126 rows
// 11.0 -> 11.5) and short tables (384 keys 10.4 -> 12.5); 2400 rows over 4096 keys would take 22.0 for 20.7.
__device__ __forceinline__ void split_bf16(const float (&p)[4], const float (&q)[4], uint4& hi, uint4& lo) {
  const auto rest = [](uint32_t h, float a, float b) {
    return pack_bf16x2(a - __uint_as_float(h << 16), b - __uint_as_float(h & 0xffff0000u));
  };
  hi = make_uint4(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(q[0], q[1]), pack_bf16x2(q[2], q[3]));
  lo = make_uint4(rest(hi.x, p[0], p[1]), rest(hi.y, p[2], p[3]), rest(hi.z, q[0], q[1]), rest(hi.w, q[2], q[3]));
}

// Takes infinities and NaN out of 16 bytes of V; returns whether there were any.
template <bool kFp8>
__device__ __forceinline__ bool take_out(uint4& v) {
  uint32_t* const w = &v.x;
  uint32_t met = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t bad = kFp8 ? __vcmpeq4(w[i] & 0x7f7f7f7fu, 0x7f7f7f7fu) : non_finite<0x7f80u>(w[i]);
    w[i] &= ~bad;
    met |= bad;
  }
  return met != 0u;
}

// The column of o[j][e] and o[j][2 + e] in lane 4r + c: eight neighbouring columns are o[8h + i][e], i < 8, of one h and e.
template <bool kFp8>
__device__ __forceinline__ int column_of(int c, int j, int e) {
  const int h = j >> 3, i = j & 7;
  return kFp8 ? 32 * c + 8 * (2 * e + h) + i : 64 * h + 16 * c + 8 * e + i;
}

// What a warp knows of a segment: rows row0 .. of KV head `head` against `units` units of keys from key0.
struct RowSegment {
  int units, head, seq, shared, row0, n_rows, key0, kv_end, clean, direct;
  long long slot;
};

// kWhole: no line; a warp takes whole items, a branch's rows against all its keys, and nothing is left
// to merge. kFine: bf16 P in two terms.
template <bool kFp8, bool kWhole, bool kFine, class P>
__global__ void __launch_bounds__(2 * 32 * kRowWarps, 1)
    branch_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                       const P p, const bool after) {
  constexpr bool kTree = is_tree<P>;
  constexpr int kTileBytes = RowCfg<kFp8>::kTileBytes, kStageBytes = RowCfg<kFp8>::kStageBytes;
  constexpr int kRowStages = RowCfg<kFp8>::kStages;
  constexpr float kBoost = kFp8 ? kBoostF8 : 0.0f;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kRowWarps][kMaxRowStages], empty[kRowWarps][kMaxRowStages];
  __shared__ int abort_word;
  __shared__ int before[kTree ? kMaxStack : 1];  // see live_row_at
  volatile int* abort_flag = &abort_word;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = (threadIdx.x >> 5) & (kRowWarps - 1), lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const bool loader = threadIdx.x >= 32 * kRowWarps;
  const uint32_t ring = ((smem_u32(smem_raw) + 1023u) & ~1023u) + warp * kRowRing;
  if (threadIdx.x == 0) {
    for (int w = 0; w < kRowWarps; ++w)
      for (int s = 0; s < kRowStages; ++s) {
        mbar_init(smem_u32(&full[w][s]), 1);
        mbar_init(smem_u32(&empty[w][s]), 1);
      }
    abort_word = 0;
    fence_mbar_init();
  }
  if (threadIdx.x == 32) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  const Line& ln = p.warp;
  const int worker = blockIdx.x * kRowWarps + warp;
  const int own_all = p.rows * p.group;
  Plan pl;
  int u, u_end;  // this warp's part of the line; kWhole: its next item, and how many there are
  Place at = {0, -1, 0, 0};
  if constexpr (kWhole) {
    u = warp * gridDim.x + blockIdx.x;  // few items: one an SM
    u_end = p.kv_heads * p.batch * ln.own_tiles;
  } else {
    pl = make_plan(p, ln, lane);
    if constexpr (kTree) {
      if (p.compact && ln.shared_tiles > 0 && threadIdx.x < 32) stack_rows(p, before, lane);
    }
    const int all = pl.head_weight * p.kv_heads;
    u = min(all, worker * pl.cut);
    u_end = min(all, u + pl.cut);
    if (u < u_end) at = locate(p, ln, pl, u, lane);
  }
  __syncthreads();

  // The next segment of this pair of warps' part (units 0: there is none).
  const auto next_segment = [&]() {
    RowSegment g;
    g.units = 0;
    if constexpr (kWhole) {
      for (; u < u_end && g.units == 0; u += gridDim.x * kRowWarps) {
        const int bh = u / ln.own_tiles, t = u - bh * ln.own_tiles;
        g.head = bh / p.batch;
        g.seq = bh - g.head * p.batch;
        g.shared = 0;
        g.row0 = g.seq * own_all + t * kRowSpan;
        g.key0 = 0;
        const Extent x = extent_of(p, g.seq);
        g.n_rows = min(kRowSpan, x.rows - t * kRowSpan);
        g.kv_end = x.all;
        g.clean = x.clean;
        g.direct = 1;
        g.slot = 0;
        g.units = own_units(p, ln, x, t);
        if (!kTree && g.units > 0) continue;
        // rows that see nothing, or come behind the nodes
        const int none = g.units > 0 ? g.n_rows : 0, all = min(kRowSpan, own_all - t * kRowSpan);
        for (int i = none * 16 + lane; !loader && i < all * 16; i += 32) {
          const RowAt ra = row_at(p, g.head, g.row0 + (i >> 4));
          const long long id = (static_cast<long long>(ra.b) * p.rows + ra.i) * p.heads + ra.h;
          reinterpret_cast<uint4*>(p.out + id * kD)[i & 15] = make_uint4(0u, 0u, 0u, 0u);
          if (p.lse && (i & 15) == 0) p.lse[id] = -INFINITY;
        }
      }
      return g;
    }
    while (u < u_end && g.units == 0) {
      const PlaceUnits it = place_units(p, ln, pl, at);
      const UnitRange in = units_in(ln, it, at.off, u_end - u);
      if (in.count > 0) {
        g.units = in.count;
        g.head = at.head;
        g.shared = at.b < 0;
        g.seq = g.shared ? pl.longest : at.b;
        g.row0 = (g.shared ? 0 : at.b * own_all) + at.t * kRowSpan;
        const Extent x = extent_of(p, g.seq);
        g.n_rows = min(kRowSpan, g.shared ? pl.live - g.row0 : x.rows - at.t * kRowSpan);
        g.key0 = (g.shared ? 0 : own_lo(p, x)) + in.first * kRowUnit;
        g.kv_end = x.all;
        g.clean = x.clean;
        g.direct = pl.shared_blocks == 0 && in.count == it.units;
        const long long item = g.shared ? static_cast<long long>(at.head) * ln.shared_tiles + at.t
                                        : (static_cast<long long>(at.head) * p.batch + at.b) * ln.own_tiles + at.t;
        g.slot = (g.shared ? 0 : p.own_row0) + (item + worker) * (g.shared ? p.shared_slot_rows : p.own_slot_rows);
      }
      u += in.part;
      if (u < u_end) step_item(p, ln, pl, at);
    }
    return g;
  };
  // The pages of a segment's keys from block `first` (of the segment) on, one a lane.
  const auto pages_of = [&](const RowSegment& g, int first) {
    const int block = (g.key0 >> 7) + first + lane, last = (g.key0 + g.units * kRowUnit - 1) >> 7;
    int page = block <= last ? __ldg(p.table + static_cast<size_t>(g.seq) * p.width + block) : 0;
    if (page < 0 || page >= p.pool_pages) {  // flagged, and read as page 0
      if (p.err) atomicOr(p.err, kErrBadPage);
      page = 0;
    }
    return page;
  };
  bool ok = true;
  int stage = 0, phase = 0;
  const auto advance = [&]() {
    if (++stage == kRowStages) {
      stage = 0;
      phase ^= 1;
    }
  };
  if (loader) {
    // ================================================================ copies
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    const bool once = !kWhole && ln.shared_tiles <= 1 && ln.own_tiles <= 1;  // keys that only one warp reads
    int issued = 0;
    for (RowSegment g = next_segment(); ok && g.units > 0; g = next_segment()) {
      int pages = 0, pages_from = -32;  // the block (of the segment) whose page lane 0 holds
      for (int i = 0; i < g.units; ++i) {
        const int key = g.key0 + i * kRowUnit, block = (key >> 7) - (g.key0 >> 7);
        if (block - pages_from >= 32) {
          pages_from = block;
          pages = pages_of(g, block);
        }
        const int row = __shfl_sync(0xffffffffu, pages, block - pages_from) * kBlk + (key & (kBlk - 1));
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&empty[warp][stage]), phase ^ 1, abort_flag, p.err));
        if (!ok) break;
        if (lane == 0) {
          const uint32_t bar = smem_u32(&full[warp][stage]);
          mbar_expect_tx(bar, kStageBytes);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int a = 0; a < (kFp8 ? 1 : 2); ++a) {
              const uint32_t dst = ring + stage * kStageBytes + kv * kTileBytes + a * (kTileBytes / 2);
              if (once) tma_load_3d_once(dst, kv ? &tmV : &tmK, bar, a * 64, row, g.head, policy);
              else tma_load_3d(dst, kv ? &tmV : &tmK, bar, a * 64, row, g.head);
            }
        }
        ++issued;
        advance();
      }
    }
    if (!ok) {
      // leaving early: no copy may still be in flight when the block ends
      for (int k = min(issued, kRowStages); k > 0; --k) {
        if (--stage < 0) {
          stage = kRowStages - 1;
          phase ^= 1;
        }
        const unsigned long long t0 = global_ns();
        while (!mbar_try_wait(smem_u32(&full[warp][stage]), phase) && global_ns() - t0 < kWaitTimeoutNs) {
        }
      }
    }
    return;
  }
  // ================================================================ products and softmax
  for (RowSegment g = next_segment(); g.units > 0; g = next_segment()) {
    // this lane's rows, r and r + 8 of the item
    const auto at_row = [&](int k) {
      const int row = g.row0 + min(k, g.n_rows - 1);
      if constexpr (kTree) {
        if (g.shared && p.compact) return live_row_at(p, before, g.head, row);
      }
      return row_at(p, g.head, row);
    };
    const RowAt at0 = at_row(r), at1 = at_row(r + 8);
    uint32_t qa[16], qb[16];
    {
      const __nv_bfloat16* a = p.q + at0.b * p.q_sb + at0.i * p.q_sn + at0.h * p.q_sh;
      const __nv_bfloat16* b = p.q + at1.b * p.q_sb + at1.i * p.q_sn + at1.h * p.q_sh;
      // the elements that this lane's chunks of a key hold
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int from = kFp8 ? 32 * c + 8 * k : 64 * (k >> 1) + 16 * c + 8 * (k & 1);
        load16(a + from, qa + 4 * k);
        load16(b + from, qb + 4 * k);
      }
    }
    const auto sight0 = sight_of(p, at0, g.shared != 0), sight1 = sight_of(p, at1, g.shared != 0);
    const int lim0 = sight0.base, lim1 = sight1.base;
    if constexpr (kTree) {  // read at the end of the item, mostly the first words
      asm volatile("prefetch.global.L1 [%0];" ::"l"(p.masks + static_cast<size_t>(sight0.row) * p.words));
      asm volatile("prefetch.global.L1 [%0];" ::"l"(p.masks + static_cast<size_t>(sight1.row) * p.words));
    }
    bool taken_out = false;  // whether a node's V held an infinity or NaN
    float sl2 = p.scale_log2, sl2b = p.scale_log2;  // of row r and row r + 8
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      if (r >= g.n_rows) qa[k] = 0u;
      if (r + 8 >= g.n_rows) qb[k] = 0u;
    }
    if constexpr (kFp8) {
      sl2 = sl2b = p.scale_log2 * __ldg(p.k_scale + g.head);
      uint32_t ta = 0u, tb = 0u;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        ta = __vmaxu2(ta, qa[k] & 0x7fff7fffu);
        tb = __vmaxu2(tb, qb[k] & 0x7fff7fffu);
      }
      ta = max(ta >> 16, ta & 0xffffu);
      tb = max(tb >> 16, tb & 0xffffu);
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        ta = max(ta, __shfl_xor_sync(0xffffffffu, ta, d));
        tb = max(tb, __shfl_xor_sync(0xffffffffu, tb, d));
      }
      const int ka = row_exponent(ta), kb = row_exponent(tb);
      const float ua = exp2_int(ka), ub = exp2_int(kb);
#pragma unroll
      for (int k = 0; k < 16; ++k) {  // infinities and NaN stay what they are
        qa[k] = f16x2_of(__uint_as_float(qa[k] << 16) * ua, __uint_as_float(qa[k] & 0xffff0000u) * ua);
        qb[k] = f16x2_of(__uint_as_float(qb[k] << 16) * ub, __uint_as_float(qb[k] & 0xffff0000u) * ub);
      }
      sl2 = score_factor(sl2 * exp2_int(-ka));
      sl2b = score_factor(sl2b * exp2_int(-kb));
    }
    float o[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll 1
    for (int i = 0; i < g.units; ++i) {
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[warp][stage]), phase, abort_flag, p.err));
      if (!ok) break;
      const uint32_t kt = ring + stage * kStageBytes, vt = kt + kTileBytes;
      const int key = g.key0 + i * kRowUnit;
      float s[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
        const uint32_t row = kt + (8 * j + r) * 128;
#pragma unroll
        for (int a = 0; a < (kFp8 ? 1 : 2); ++a) {
          const uint4 x = lds16(row + a * (kTileBytes / 2) + (((2 * c) ^ r) << 4));
          const uint4 y = lds16(row + a * (kTileBytes / 2) + (((2 * c + 1) ^ r) << 4));
          const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
          if constexpr (kFp8) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              mma16<true>(s[j], make_uint4(qa[2 * k], qb[2 * k], qa[2 * k + 1], qb[2 * k + 1]), f16x2_of_e4m3x2(w[k]),
                          f16x2_of_e4m3x2(w[k] >> 16));
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma16<false>(s[j], make_uint4(qa[8 * a + 2 * k], qb[8 * a + 2 * k], qa[8 * a + 2 * k + 1], qb[8 * a + 2 * k + 1]),
                           w[2 * k], w[2 * k + 1]);
          }
        }
      }
      // keys at or past a row's limit are hidden from it
      if (__any_sync(0xffffffffu, key + 32 > min(lim0, lim1))) {
        if constexpr (kTree) {  // but for nodes that it sees
          const uint32_t seen0 = sight0.seen32(p, key), seen1 = sight1.seen32(p, key);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              if (!(seen0 >> (8 * j + 2 * c + k) & 1u)) s[j][k] = -INFINITY;
              if (!(seen1 >> (8 * j + 2 * c + k) & 1u)) s[j][2 + k] = -INFINITY;
            }
        } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int at_key = key + 8 * j + 2 * c + k;
            if (at_key >= lim0) s[j][k] = -INFINITY;
            if (at_key >= lim1) s[j][2 + k] = -INFINITY;
          }
        }
      }
      float t0 = fmaxf(fmax3(fmaxf(s[0][0], s[0][1]), s[1][0], s[1][1]), fmax3(fmaxf(s[2][0], s[2][1]), s[3][0], s[3][1]));
      float t1 = fmaxf(fmax3(fmaxf(s[0][2], s[0][3]), s[1][2], s[1][3]), fmax3(fmaxf(s[2][2], s[2][3]), s[3][2], s[3][3]));
      t0 = quad_max(t0) * sl2;
      t1 = quad_max(t1) * sl2b;
      const bool need0 = t0 > m0 + kGrowth, need1 = t1 > m1 + kGrowth;
      if (__any_sync(0xffffffffu, need0 || need1)) {
        const float a0 = need0 ? fast_exp2(m0 - t0) : 1.f, a1 = need1 ? fast_exp2(m1 - t1) : 1.f;
        m0 = need0 ? t0 : m0;
        m1 = need1 ? t1 : m1;
        l0 *= a0;
        l1 *= a1;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          o[j][0] *= a0;
          o[j][1] *= a0;
          o[j][2] *= a1;
          o[j][3] *= a1;
        }
      }
      // a row that has seen nothing yet keeps m = -inf: x - m would be NaN
      const float b0 = kBoost - (m0 == -INFINITY ? 0.f : m0), b1 = kBoost - (m1 == -INFINITY ? 0.f : m1);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j][0] = fast_exp2(fmaf(s[j][0], sl2, b0));
        s[j][1] = fast_exp2(fmaf(s[j][1], sl2, b0));
        s[j][2] = fast_exp2(fmaf(s[j][2], sl2b, b1));
        s[j][3] = fast_exp2(fmaf(s[j][3], sl2b, b1));
        l0 += s[j][0] + s[j][1];
        l1 += s[j][2] + s[j][3];
      }
      const bool tail = key + 32 > g.kv_end;
      if constexpr (kTree) {
        if (key + 32 > g.clean) {  // the unit has nodes
          bool met = false;
          for (int i = lane; i < kTileBytes / 16; i += 32) {  // 16 bytes of a row
            const int row = (i >> 3) & 31;
            if (key + row < g.clean || key + row >= g.kv_end) continue;
            const uint32_t at = vt + (i >> 8) * (kTileBytes / 2) + row * 128 + (i & 7) * 16;
            uint4 v = lds16(at);
            if (take_out<kFp8>(v)) {
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                           : "memory");
              met = true;
            }
          }
          if (__any_sync(0xffffffffu, met)) {
            taken_out = true;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the stage is filled again by TMA
          }
          __syncwarp();
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // sixteen keys
        uint4 a, rest;
        if constexpr (kFp8)
          a = make_uint4(f16x2_of(s[2 * h][0], s[2 * h][1]), f16x2_of(s[2 * h][2], s[2 * h][3]),
                         f16x2_of(s[2 * h + 1][0], s[2 * h + 1][1]), f16x2_of(s[2 * h + 1][2], s[2 * h + 1][3]));
        else
          split_bf16(s[2 * h], s[2 * h + 1], a, rest);
#pragma unroll
        for (int atom = 0; atom < (kFp8 ? 1 : 2); ++atom) {
          uint4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = h * 16 + 2 * c + (k >> 1) * 8 + (k & 1);
            v[k] = lds16(vt + atom * (kTileBytes / 2) + row * 128 + ((r ^ (row & 7)) << 4));
            // values past the sequence's end may be anything, NaN too, and P's zeros do not undo that
            if (tail && key + row >= g.kv_end) v[k] = make_uint4(0u, 0u, 0u, 0u);
          }
          const uint32_t x[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, y[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
          const uint32_t z[4] = {v[2].x, v[2].y, v[2].z, v[2].w}, t[4] = {v[3].x, v[3].y, v[3].z, v[3].w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            if constexpr (kFp8) {  // four columns a word
              const uint32_t xy = __byte_perm(x[w], y[w], 0x5140), zt = __byte_perm(z[w], t[w], 0x5140);
              const uint32_t xy2 = __byte_perm(x[w], y[w], 0x7362), zt2 = __byte_perm(z[w], t[w], 0x7362);
              mma16<true>(o[4 * w], a, f16x2_of_e4m3x2(xy), f16x2_of_e4m3x2(zt));
              mma16<true>(o[4 * w + 1], a, f16x2_of_e4m3x2(xy >> 16), f16x2_of_e4m3x2(zt >> 16));
              mma16<true>(o[4 * w + 2], a, f16x2_of_e4m3x2(xy2), f16x2_of_e4m3x2(zt2));
              mma16<true>(o[4 * w + 3], a, f16x2_of_e4m3x2(xy2 >> 16), f16x2_of_e4m3x2(zt2 >> 16));
            } else {  // two
              const int n = 8 * atom + 2 * w;
              const uint32_t b0 = __byte_perm(x[w], y[w], 0x5410), b1 = __byte_perm(z[w], t[w], 0x5410);
              const uint32_t b2 = __byte_perm(x[w], y[w], 0x7632), b3 = __byte_perm(z[w], t[w], 0x7632);
              mma16<false>(o[n], a, b0, b1);
              mma16<false>(o[n + 1], a, b2, b3);
              if constexpr (kFine) {
                mma16<false>(o[n], rest, b0, b1);
                mma16<false>(o[n + 1], rest, b2, b3);
              }
            }
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      if (lane == 0) mbar_arrive(smem_u32(&empty[warp][stage]));
      advance();
    }
    if (!ok) break;
    if constexpr (kTree) {
      if (sight0.hidden()) {
        m0 = -INFINITY;
        l0 = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = 0.f;
      }
      if (sight1.hidden()) {
        m1 = -INFINITY;
        l1 = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j][2] = o[j][3] = 0.f;
      }
      // what was taken out of V, to the rows that see it
      if (__any_sync(0xffffffffu, taken_out)) {
        const NodeValues<kFp8> nodes(p, g.seq, g.head);
#pragma unroll 1
        for (int k = 0; k < 32; ++k) {  // one column's code: it is seldom needed
          const int col = column_of<kFp8>(c, k >> 1, k & 1);
          const int end = g.key0 + g.units * kRowUnit;
          const float lost0 = nodes.non_finite_sum(p, sight0, col, g.key0, end, 1);
          const float lost1 = nodes.non_finite_sum(p, sight1, col, g.key0, end, 1);
#pragma unroll
          for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (k == 2 * j + e) {
                o[j][e] += lost0;
                o[j][2 + e] += lost1;
              }
        }
      }
    }
    l0 = quad_sum(l0);
    l1 = quad_sum(l1);
    // ---- this lane's columns: e4m3 32c .. + 31, bf16 16c .. + 15 and 64 + 16c .. + 15; eight at a time
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row_in = r + 8 * half;
      if (row_in >= g.n_rows) continue;
      const float l = half ? l1 : l0, m = (half ? m1 : m0) - kBoost;
      const RowAt& ra = half ? at1 : at0;
      const long long id = (static_cast<long long>(ra.b) * p.rows + ra.i) * p.heads + ra.h;
      float w = l == 0.f ? 0.f : 1.0f / l;
      if constexpr (kFp8) w *= __ldg(p.v_scale + g.head);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // o[j][e], o[j + 1][e] ..: eight neighbouring columns from `col` on
        const int j = kFp8 ? (k & 1) * 8 : (k >> 1) * 8, e = 2 * half + (kFp8 ? k >> 1 : k & 1);
        const int col = kFp8 ? 32 * c + 8 * k : 64 * (k >> 1) + 16 * c + 8 * (k & 1);
        if (g.direct) {
          *reinterpret_cast<uint4*>(p.out + id * kD + col) =
              make_uint4(pack_bf16x2(o[j][e] * w, o[j + 1][e] * w), pack_bf16x2(o[j + 2][e] * w, o[j + 3][e] * w),
                         pack_bf16x2(o[j + 4][e] * w, o[j + 5][e] * w), pack_bf16x2(o[j + 6][e] * w, o[j + 7][e] * w));
        } else {
          float4* dst = reinterpret_cast<float4*>(p.part_o + (g.slot + row_in) * kD + col);
          dst[0] = make_float4(o[j][e], o[j + 1][e], o[j + 2][e], o[j + 3][e]);
          dst[1] = make_float4(o[j + 4][e], o[j + 5][e], o[j + 6][e], o[j + 7][e]);
        }
      }
      if (c == 0) {
        if (!g.direct) p.part_ml[g.slot + row_in] = make_float2(m, l);
        else if (p.lse) p.lse[id] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      }
    }
  }
  if (worker == 0) {
    flag_lengths(p, lane);
    if constexpr (!kWhole) write_plan(p, ln, pl, p.plan + kPlanHead + 2 * p.batch, lane);
  }
  // what follows this kernel needs the other line's too; one block's wait holds it, and the others make
  // room for it
  if (after && blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <bool kFp8, bool kWhole, bool kFine, class P>
int launch_rows(const P& p, bool after, cudaLaunchConfig_t cfg) {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (dev >= 64 || !done[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(branch_rows_kernel<kFp8, kWhole, kFine, P>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(kRowSmem));
      if (e != cudaSuccess) return set_cuda_error("cudaFuncSetAttribute(branch rows)", e);
      if (dev < 64) done[dev] = true;
    }
  }
  CUtensorMap tmK, tmV;
  int rc = encode_pool(&tmK, p, p.key_pool, kFp8, kRowUnit);
  if (!rc) rc = encode_pool(&tmV, p, p.value_pool, kFp8, kRowUnit);
  if (rc) return rc;
  const int sms = p.warp.workers / kRowWarps;
  cfg.gridDim = dim3(kWhole ? min(sms, p.kv_heads * p.batch * p.warp.own_tiles) : sms);
  cfg.blockDim = dim3(2 * 32 * kRowWarps);
  cfg.dynamicSmemBytes = kRowSmem;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, branch_rows_kernel<kFp8, kWhole, kFine, P>, tmK, tmV, p, after);
  return e == cudaSuccess ? H3SA_OK : set_cuda_error("branch_rows_kernel launch", e);
}

template <class P>
int launch_lines(const P& p, bool e4m3, bool after, cudaLaunchConfig_t cfg) {
  if (e4m3)
    return p.whole ? launch_rows<true, true, false, P>(p, after, cfg) : launch_rows<true, false, false, P>(p, after, cfg);
  if (p.whole) return launch_rows<false, true, true, P>(p, after, cfg);
  const long long stacked = static_cast<long long>(p.batch) * p.rows * p.heads;
  return kRowWarps * stacked <= p.warp.workers ? launch_rows<false, false, true, P>(p, after, cfg)
                                               : launch_rows<false, false, false, P>(p, after, cfg);
}

}  // namespace

int launch_branch_rows(const BranchParams& p, bool e4m3, bool after, cudaLaunchConfig_t cfg) {
  return launch_lines(p, e4m3, after, cfg);
}
int launch_branch_rows(const TreeParams& p, bool e4m3, bool after, cudaLaunchConfig_t cfg) {
  return launch_lines(p, e4m3, after, cfg);
}

int encode_pool(CUtensorMap* map, const BranchParams& p, const void* pool, bool e4m3, int rows) {
  const uint64_t pool_rows = static_cast<uint64_t>(p.pool_pages) * kBlk, row_bytes = kD * (e4m3 ? 1 : 2);
  const uint64_t dims[3] = {kD, pool_rows, static_cast<uint64_t>(p.kv_heads)};
  const uint64_t strides[2] = {row_bytes, pool_rows * row_bytes};
  const uint32_t box[3] = {e4m3 ? 128u : 64u, static_cast<uint32_t>(rows), 1};
  return encode_tiled_3d(map, e4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, pool, dims,
                         strides, box);
}

}  // namespace h3sa
