// Attention of several branches of one stream over their shared history and their own rows.
//
// A branch (sequence) b of a paged, head-major KV pool is one row of a page table and a length;
// the first `shared` pages of every row are the same pages. Row (b, i) of query head h sees the
// keys j < limit(b, i) = length(b) - (causal ? n - 1 - i : 0) of its own sequence:
//
//   x_j = scale * q . k_j,   out = sum_j 2^(x_j' - m) v_j / sum_j 2^(x_j' - m),  x' = x log2 e
//
// In the split form an item is either a span of all branches' rows stacked (b, i, and the query
// heads of the KV head's group) against the shared blocks, which are so read once for all, or the
// rows of one branch against its own blocks; in the joint form (see joint_form) an
// item is a span of one branch's rows against all its blocks. There are two kernels for them, the
// tensor line here (items of up to 256 rows, tcgen05) and the warp line in h3sa_branch_rows.cu
// (items of 16 rows, each warp by itself); shape_of says which takes what. Either one's units,
// a step of keys of one KV head against one item, lie in one line (KV head, shared items, own items)
// that is cut into equal ranges, one per CTA or warp, whatever the lengths are; lengths are read on
// the device. An item that no cut divides and that nothing else contributes to is written out
// directly; the pieces of all others go to a workspace as unnormalised fp32 O, running maximum and
// sum, and branch_merge_kernel joins them in a fixed order, so results do not depend on timing.
//
// Warp roles of branch_attn_kernel (one persistent CTA per SM, 384 threads):
//   warp 0      walks the CTA's units: publishes each item segment in a small descriptor ring and
//               loads its K and V blocks by TMA into one ring of tiles.
//   warp 1, 2   issue the MMAs of query tile 0 and 1: S_t = Q_t K^T, then O_t += P_t V, one elected
//               lane per tcgen05 instruction (warp 1 also owns TMEM).
//   warp 3      e4m3: widens V to f16.
//   warps 4-7, 8-11: softmax and epilogue of query tile 0 and 1, one thread per TMEM lane.
// An item of more than 128 rows takes both tiles, each block being used by both; smaller items
// take one tile per block in turn, so two blocks are in flight. Items of up to 32 (64) rows of
// chains are held 4 (2) times, once per 32-lane (64-lane) part of the tile: each copy takes the exponentials
// of its own quarter (half) of the block's columns and writes zeros elsewhere, which spreads the
// softmax of few rows over all four warps; the copies are joined in the epilogue. Trees' rows are held once:
// what bounds the kernel beside the softmax is its own code, streaming past the instruction caches, and the two other
// forms in between cost trees more than they bring (wide e4m3 trees 237 -> 206 us without them, 64 rows over 16000
// keys 203 -> 199, e4m3 239 -> 214). Measured, trees, with the merge: 24 of 96 rows over up to 9000 keys each 98 to 102 us
// (4.7 TB/s of 472 MB; 5.9 while blocks stream), 20 small ones over 8192 shared keys 61 to 63, e4m3, four of 635 rows over up to
// 24001 keys 179 to 193 (600 to 650 TFLOP/s, by power).
// TMEM columns: S0 [0,128), S1 [128,256), O0 [256,384), O1 [384,512); P of a tile overwrites the
// first half of its S. A tile's MMAs are issued in order by one warp, so the barrier of a QK^T also
// says that the tile's previous P V is complete.
//
// e4m3 caches: K goes to the tensor cores as it is (kind::f8f6f4), and each query row, scaled by a
// power of two to a maximum in [128, 256), as a sum of two e4m3 terms, whose products add up in fp32. Two
// terms hold a bf16 number exactly from 2^-2 on, and a smaller one to within 2^-10, 2^-17 of the row's
// maximum. P cannot go that way: the terms' last step would be 2^-15 of the largest weight, and the tail
// behind a key that dominates, thousands of keys each below that, would count in the sum and not in O. So P
// is f16 (11 bits down to 2^-21 of a fresh maximum, steps of 2^-31 of it below), and warp 3 widens each
// V block to f16 in shared memory, where kind::f16 takes it: one f16 product costs what two of e4m3 do, and
// the softmax has no terms to split. Against two e4m3 terms (us): 3 x 1211 rows of 24 heads to 15.7 K keys 721 /
// 821, 60 stacked rows of 8 KV heads over 98304 keys 97.6 / 92.2 (91 since the widening loop is half as long): a block's 1850
// cycles in warp 3 take issue slots from the softmax warps beside it.
// P of bf16 caches is bf16, 8 bits of each weight however small, as the output has.
//
// Measured: 3 branches of 1211 rows, 24 heads, to 15.7 K keys, bf16, joint: 640 to 750 us (0.86 to
// 1.0 PFLOP/s, by power), the tensor pipe 53 % active; what bounds it is the softmax's latency, 2000 cycles
// a half block of both tiles in step, 1024 of them 2^x. 60 stacked rows of 8 KV heads over 98304 e4m3 keys, with own rows and
// merge: 91 us (2.5 TB/s of 227 MB), bound by the round trips of half blocks; 9 us go by before the first scores (all
// CTAs' first loads and queries at once) and 5 in the epilogue.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstring>
#include <mutex>

#include "h3sa_branch.cuh"

namespace h3sa {
namespace {

constexpr int kBrThreads = 384;
constexpr int kBrRegsControl = 88;
constexpr int kBrRegsSoftmax = 208;
constexpr int kBrRegSplit = 128 * kBrRegsControl + 256 * kBrRegsSoftmax;
constexpr int kDescRing = 4;
constexpr int kAtom = kBlk * 128;  // 128 rows of one 128-byte swizzle atom

// One item segment of a CTA, as warp 0 publishes it.
struct Segment {
  int live;      // 0: the CTA's last descriptor; 2: against the shared blocks
  int number;    // of the CTA's segments, from 1
  int head;      // KV head
  int row0;      // first stacked query row of the item
  int n_rows;    // rows of the item (1..256)
  int block0;    // first logical block
  int blocks;
  int kv_end;    // rows at or past it hold nothing
  int clean;     // rows at or past it are nodes of a tree
  int direct;    // the segment is its rows' whole result
  long long slot_row[2];  // workspace row of each tile's partial
};

template <bool kFp8>
struct BrCfg {
  static constexpr int kElem = kFp8 ? 1 : 2;
  static constexpr int kTile = kBlk * kD * kElem;
  static constexpr int kStages = kFp8 ? 6 : 5;  // even for e4m3: K in the even slots, V in the odd ones
  static constexpr int kSteps = kFp8 ? 4 : 8;   // MMA K steps of S
  // Order of a segment's loads: K0 K1 V0 K2 V1 ..., each V behind the next K, which is wanted first (V waits for a
  // softmax, in a slot of the ring). In turn / as it is, us: 24 trees of 96 rows over 9000 keys 118.6 / 101.8, of 64 over 16000
  // 179 / 150; 24 chains of 96 rows over 9000 keys 101.3 / 89.7, of 4 x 32 over 8192 shared keys 46.8 / 46.1; e4m3: K0 V0 K1
  // V1 ..., as V is widened on its way.
  static constexpr bool kSkew = !kFp8;
  static constexpr uint32_t kIdescQK = kFp8 ? idesc_e4m3(kBlk, kBlk / 2, false) : idesc_bf16(kBlk, kBlk / 2, false);
  static constexpr uint32_t kIdescPV = kFp8 ? idesc_f16(kBlk, kD, true) : idesc_bf16(kBlk, kD, true);
};

constexpr int kQBytes = 2 * kAtom;  // a query tile: 128 x 128 bf16, or two e4m3 terms

// V of e4m3 caches in f16, blocks in turn, and the barriers between the warp that widens them and the
// MMA warps: [tile][buffer], of the tiles as those of the ring. With a third buffer for two slots of the ring
// 60 rows over 98304 keys take 100.7 us instead of 97.6.
constexpr int kWide = 2;
constexpr int kWideTile = 2 * kAtom;
template <bool kFp8>
struct BrWide {};
template <>
struct BrWide<true> {  // begins at a multiple of 1024 bytes, as the tiles in front of it are multiples
  uint8_t v[kWide][kWideTile];
  uint64_t full[2][kWide], empty[2][kWide];
};

// The numbers of the segments in whose V a node had an infinity or NaN. A tile's epilogue reads the one of its segment when
// its warps have taken one of the next two, and no warp can be more than the descriptors' ring in front of that: places of
// twice the ring are not taken again before they are read.
constexpr int kTakenOut = 2 * kDescRing;
template <class P>
struct BrTree {};
template <>
struct BrTree<TreeParams> {
  int taken_out[kTakenOut];
  int before[kMaxStack];  // see live_row_at
};

__device__ __forceinline__ void mark_taken_out(BrTree<TreeParams>& tree, int number) {
  *static_cast<volatile int*>(tree.taken_out + number % kTakenOut) = number;
}

template <bool kFp8, class P>
struct alignas(1024) BrSmem {
  using Cfg = BrCfg<kFp8>;
  uint8_t q[2][kQBytes];  // also the epilogue's staging
  uint8_t kv[Cfg::kStages][Cfg::kTile];
  BrWide<kFp8> wide;
  Segment desc[kDescRing];
  uint64_t full[2][Cfg::kStages], empty[2][Cfg::kStages];  // [tile]; see the MMA warps
  uint64_t d_full[kDescRing], d_empty[kDescRing];
  uint64_t q_full[2], o_full[2], pv_done[2], wg[2];
  uint64_t s_full[2][2], p_full[2][2];  // [tile][half of a block]; whole blocks use the first
  uint64_t m_sync, drain;
  uint32_t tmem_base;
  int abort_flag;
  BrTree<P> tree;
};
template <bool kFp8, class P>
constexpr size_t br_smem_bytes() {
  return sizeof(BrSmem<kFp8, P>) + 1024;
}
using BrSmemTreeF8 = BrSmem<true, TreeParams>;
static_assert(offsetof(BrSmemTreeF8, wide) % 1024 == 0, "widened V must be aligned to its swizzle");
static_assert(br_smem_bytes<false, TreeParams>() <= 232448 && br_smem_bytes<true, TreeParams>() <= 232448,
              "branch attention needs more than 227 KB");

__device__ __forceinline__ uint32_t e4m3x2_of(uint32_t h2) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(h2));
  return r;
}
// Two values below 448 as the sum of two e4m3 terms each, through f16 (11 bits, so nothing that
// the two 4-bit terms could hold is lost).
__device__ __forceinline__ void split_e4m3x2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const uint32_t h = f16x2_of(a, b);
  hi = e4m3x2_of(h);
  const uint32_t back = f16x2_of_e4m3x2(hi);
  uint32_t rest;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(rest) : "r"(h), "r"(back));
  lo = e4m3x2_of(rest);
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// 2^x of a pair, x below 128, on the multiply-add pipe, which takes over a quarter of full tiles' (joint
// chunks 684 -> 640 us; an eighth 660, three eighths 670, half 716): x = i + f with |f| <= 1/2, 2^f as a polynomial
// (least maximum relative error of its degree with 2^0 = 1 exactly: 2^-18.4), i added to the exponent.
// From x = -127 down the result is 0; NaN stays NaN.
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x2) {
  float x0, x1, r0, r1, t0, t1;
  f2_unpack(x2, x0, x1);
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x0) : "f"(x0), "f"(-127.0f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x1) : "f"(x1), "f"(-127.0f));
  x2 = f2_pack(x0, x1);
  const auto both = [](float c) { return f2_pack(c, c); };
  const uint64_t t2 = f2_add(x2, both(12582912.0f));  // 1.5 * 2^23: i in the last bits
  const uint64_t f2 = f2_fma(f2_add(t2, both(-12582912.0f)), both(-1.0f), x2);
  uint64_t r2 = f2_fma(both(0.009585382416844368f), f2, both(0.05590662732720375f));
  r2 = f2_fma(r2, f2, both(0.24024038016796112f));
  r2 = f2_fma(r2, f2, both(0.6931241750717163f));
  r2 = f2_fma(r2, f2, both(1.0f));
  f2_unpack(t2, t0, t1);
  f2_unpack(r2, r0, r1);
  r0 = __int_as_float(__float_as_int(r0) + (__float_as_int(t0) << 23));
  r1 = __int_as_float(__float_as_int(r1) + (__float_as_int(t1) << 23));
  return f2_fma(x2, both(0.0f), f2_pack(r0, r1));
}

// Softmax of kCols score columns of this thread's row, its copy's share of one half of a block:
// columns [col0, col0 + kCols) of the block, col0 = 64 half + copy * kCols, in TMEM at tS + col0.
// P goes over the half's scores, zeros in the other copies' shares. key0: the block's first key, sight: of
// this row. m / l: running maximum (log2 units) and sum; `pv_done` waits until O holds all earlier halves, before O is rescaled because
// the maximum grew (lazily: only past the threshold).
template <bool kFp8, int kCols, class P, class S, typename Wait>
__device__ __forceinline__ void softmax_half(const P& p, uint32_t tS, uint32_t tO, int half, int copy, int key0, const S& sight,
                                             float sl2, bool first, float& m, float& l, Wait&& pv_done) {
  constexpr float kBoost = kFp8 ? kBoostF8 : 0.0f;
  const int col0 = 64 * half + copy * kCols;
  // Columns at or past `limit` (relative to the block) are hidden from this row, but for nodes that it sees: -inf, of
  // trees in TMEM before the scores are read, which keeps the tests out of the code of whole blocks.
  const int limit = sight.base - key0;
  int hide = __any_sync(0xffffffffu, limit < col0 + kCols) ? 1 : 0;
  asm volatile("" : "+r"(hide));
  if constexpr (std::is_same_v<S, Sight>) {
    static_assert(kCols == 64, "rows of trees are held once");
    if (hide) {
#pragma unroll 1
      for (int c = 0; c < 64; c += 32) {
        uint32_t r[32];
        tmem_ld32(tS + col0 + c, r);
        const uint32_t seen = sight.seen32(p, key0 + col0 + c);
        tmem_wait_ld();
        reg_fence32(r);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (!(seen >> j & 1u)) r[j] = 0xff800000u;
        tmem_st32(tS + col0 + c, r);
      }
      tmem_wait_st();
    }
  }
  float s[kCols];
  if constexpr (kCols >= 32) {
    uint32_t r[kCols / 32][32];
#pragma unroll
    for (int c = 0; c < kCols / 32; ++c) tmem_ld32(tS + col0 + c * 32, r[c]);
    tmem_wait_ld();
#pragma unroll
    for (int c = 0; c < kCols / 32; ++c) {
      reg_fence32(r[c]);
#pragma unroll
      for (int j = 0; j < 32; ++j) s[c * 32 + j] = __uint_as_float(r[c][j]);
    }
  } else {
    uint32_t r[16];
    tmem_ld16(tS + col0, r);
    tmem_wait_ld();
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j] = __uint_as_float(r[j]);
  }
  if (!std::is_same_v<S, Sight> && hide) {
#pragma unroll
    for (int j = 0; j < kCols; ++j)
      if (col0 + j >= limit) s[j] = -INFINITY;
  }
  float mx0 = s[0], mx1 = s[1], mx2 = s[2], mx3 = s[3];
#pragma unroll
  for (int j = 4; j + 4 < kCols; j += 8) {
    mx0 = fmax3(mx0, s[j], s[j + 4]);
    mx1 = fmax3(mx1, s[j + 1], s[j + 5]);
    mx2 = fmax3(mx2, s[j + 2], s[j + 6]);
    mx3 = fmax3(mx3, s[j + 3], s[j + 7]);
  }
  // kCols is a multiple of 8, so four columns are left
  const float mb = fmax3(fmax3(mx0, mx1, mx2), fmax3(mx3, s[kCols - 4], s[kCols - 3]),
                         fmaxf(s[kCols - 2], s[kCols - 1])) * sl2;
  const bool need = mb > m + kGrowth;
  const float m_new = need ? mb : m;
  const float alpha = need ? fast_exp2(m - m_new) : 1.0f;
  const bool any_need = !first && __any_sync(0xffffffffu, need);
  l *= alpha;
  m = m_new;
  // a row that has seen nothing yet keeps m = -inf: x - m would be NaN
  const float bias = kBoost - (m == -INFINITY ? 0.0f : m);
  const uint64_t bias2 = f2_pack(bias, bias), scale2 = f2_pack(sl2, sl2);
  uint64_t sum2 = f2_pack(0.f, 0.f);
  uint32_t pk[kCols / 2];
#pragma unroll
  for (int j = 0; j < kCols; j += 2) {
    const uint64_t x2 = f2_fma(f2_pack(s[j], s[j + 1]), scale2, bias2);
    if (kCols == 64 && (j & 7) == 6) {
      f2_unpack(exp2_pair(x2), s[j], s[j + 1]);
    } else {
      float x0, x1;
      f2_unpack(x2, x0, x1);
      s[j] = fast_exp2(x0);
      s[j + 1] = fast_exp2(x1);
    }
    sum2 = f2_add(sum2, f2_pack(s[j], s[j + 1]));
    pk[j / 2] = kFp8 ? f16x2_of(s[j], s[j + 1]) : pack_bf16x2(s[j], s[j + 1]);
  }
  float sa, sb;
  f2_unpack(sum2, sa, sb);
  l += sa + sb;
  uint32_t w[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) w[j] = kCols == 64 || j / (kCols / 2) == copy ? pk[j % (kCols / 2)] : 0u;
  pv_done();
  if (any_need) {
    tc_fence_after();
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      uint32_t o[32];
      tmem_ld32(tO + c * 32, o);
      tmem_wait_ld();
      reg_fence32(o);
#pragma unroll
      for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
      tmem_st32(tO + c * 32, o);
    }
  }
  tmem_st32(tS + 64 * half, w);
  tmem_wait_st();
}

// Writes query row `my` of a tile that holds `copies` of each row, span rows apart (K-major, 128-byte
// swizzle); `copy` says which of them this thread stands for. bf16: its own copy, as it is; returns
// 1. e4m3: as two terms after scaling by a power of two; returns that power's inverse. The splits
// are some ten instructions an element, so the threads of a row's copies share them out and each
// writes its columns to all copies.
template <bool kFp8>
__device__ __forceinline__ float store_query_row(uint8_t* tile, int my, int copy, int copies, int span,
                                                 const uint4 (&v)[16]) {
  const int sw = my & 7;  // the same for all copies: span is a multiple of 8
  if constexpr (!kFp8) {
    uint8_t* row = tile + (copy * span + my) * 128;
#pragma unroll
    for (int c = 0; c < 16; ++c)
      *reinterpret_cast<uint4*>(row + (c >> 3) * kAtom + (((c & 7) ^ sw) << 4)) = v[c];
    return 1.0f;
  } else {
    // the largest magnitude as bits: those of an infinity or NaN are larger than any number's
    const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < 64; ++i) top = __vmaxu2(top, w[i] & 0x7fff7fffu);
    top = max(top >> 16, top & 0xffffu);
    const int k = row_exponent(top);
    // a row with an infinity or NaN becomes NaN, as its products are; its factor stays finite, so that
    // keys hidden from it stay hidden
    const float up = top >= 0x7f80u ? __int_as_float(0x7fffffff) : exp2_int(k);
#pragma unroll
    for (int c = 0; c < 8; ++c) {  // 16 columns a chunk
      if ((c & (copies - 1)) != copy) continue;
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t h[2], g[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t x = w[c * 8 + j * 2 + t];
          split_e4m3x2(__uint_as_float(x << 16) * up, __uint_as_float(x & 0xffff0000u) * up, h[t], g[t]);
        }
        hi[j] = h[0] | (h[1] << 16);
        lo[j] = g[0] | (g[1] << 16);
      }
      for (int r = my; r < kBlk; r += span) {
        uint8_t* at = tile + r * 128 + ((c ^ sw) << 4);
        *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(at + kAtom) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    return exp2_int(-k);
  }
}

// A V block (128 rows of 128 bytes, 128-byte swizzle) from e4m3 to f16 as a bf16 block lies (two atoms of 64
// columns), by a warp; kTail: rows at or past `rows` become zeros. A lane takes a 16-byte chunk of a row at a
// time, eight rows in two steps, and all its offsets but two are constants. Lanes of the second atom take
// the halves of their chunk the other way round: the eight of a phase write eight different chunks.
// kNodes: NaN in rows at or past `clean` become zeros too; returns whether this lane met one.
template <bool kTail, bool kNodes>
__device__ __forceinline__ bool widen_block(uint32_t from, uint32_t to, int rows, int clean, int lane) {
  uint32_t met = 0u;
  const int c = lane & 7, h = c >> 2, at = 2 * (c & 3);
  const int r = (lane >> 4) + ((lane >> 1) & 4);  // rows r and r ^ 2 of eight; those of a half warp differ by 4
  // Not unrolled, for its code. Unrolled / as it is, us: 24 trees of 64 rows over 16000 keys 198 / 159, four of 635 rows over up to
  // 24001 207 / 179; chains: 24 of 96 rows over 9000 keys 118 / 108, 60 stacked rows over 98304 shared keys 97.4 / 90.7.
#pragma unroll 1
  for (int step = 0; step < 2; ++step) {
    const int row = r ^ (2 * step);
    const uint32_t src = from + row * 128 + ((c ^ row) << 4) + 8 * h;
    const uint32_t dst = to + h * kAtom + row * 128 + (((at + h) ^ row) << 4);
#pragma unroll 1
    for (int i0 = 0; i0 < kBlk / 8; i0 += 8) {
      uint2 x[8][2];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                       : "=r"(x[i][k].x), "=r"(x[i][k].y)
                       : "r"((src ^ (8 * k)) + (i0 + i) * 1024));
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (kTail && (i0 + i) * 8 + row >= rows) x[i][k] = make_uint2(0u, 0u);
          uint32_t w[4] = {f16x2_of_e4m3x2(x[i][k].x), f16x2_of_e4m3x2(x[i][k].x >> 16), f16x2_of_e4m3x2(x[i][k].y),
                           f16x2_of_e4m3x2(x[i][k].y >> 16)};
          if constexpr (kNodes) {
            if ((i0 + i) * 8 + row >= clean) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t bad = non_finite<0x7c00u>(w[j]);
                met |= bad;
                w[j] &= ~bad;
              }
            }
          }
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"((dst ^ (16 * k)) + (i0 + i) * 1024),
                       "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                       : "memory");
        }
    }
  }
  return met != 0u;
}

// Clears what must not be multiplied in V's block of a sequence's last rows: rows at or past `rows` of it may
// hold anything, and nodes' infinities and NaN (rows from `clean` on) belong to those that see them. The block's
// load has completed. Both MMA warps clear a block of two tiles, each what the other has left, so the one that comes second
// may find nothing: the segment is marked before the value goes, and whoever finds it gone passes that on by its
// own barriers.
template <bool kTree, typename Mark>
__device__ __forceinline__ void clear_block(uint32_t base, int rows, int clean, int lane, Mark&& mark) {
  const auto store = [](uint32_t at, const uint4& v) {
    asm volatile("st.volatile.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
  };
  if constexpr (kTree) {
    const int from = max(0, clean);
    for (int i = lane; i < (min(rows, kBlk) - from) * 16; i += 32) {
      const uint32_t at = base + (i >> 3 & 1) * kAtom + (from + (i >> 4)) * 128 + (i & 7) * 16;
      uint4 v;
      asm volatile("ld.volatile.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
      const uint4 bad = make_uint4(non_finite<0x7f80u>(v.x), non_finite<0x7f80u>(v.y), non_finite<0x7f80u>(v.z),
                                   non_finite<0x7f80u>(v.w));
      if (bad.x | bad.y | bad.z | bad.w) {
        mark();
        __threadfence_block();
        store(at, make_uint4(v.x & ~bad.x, v.y & ~bad.y, v.z & ~bad.z, v.w & ~bad.w));
      }
    }
    __threadfence_block();
  }
  for (int i = lane; i < (kBlk - rows) * 16; i += 32)
    store(base + (i >> 3 & 1) * kAtom + (rows + (i >> 4)) * 128 + (i & 7) * 16, make_uint4(0u, 0u, 0u, 0u));
}

template <bool kFp8, class P>
__global__ void __launch_bounds__(kBrThreads, 1)
    branch_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const P p) {
  using Cfg = BrCfg<kFp8>;
  constexpr bool kTree = is_tree<P>;
  constexpr int kS = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  using Smem = BrSmem<kFp8, P>;
  Smem& sm = *reinterpret_cast<Smem*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  volatile int* abort_flag = &sm.abort_flag;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Plan pl;
  const Line& ln = p.tensor;
  if (warp == 0) {  // under way while the others set up
    pl = make_plan(p, ln, lane);
    if constexpr (kTree) {
      if (p.compact && ln.shared_tiles > 0) stack_rows(p, sm.tree.before, lane);
    }
  }
  if (threadIdx.x == 64) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    for (int s = 0; s < kS; ++s) {
      mbar_init(smem_u32(&sm.full[0][s]), 1);
      mbar_init(smem_u32(&sm.full[1][s]), 1);
      mbar_init(smem_u32(&sm.empty[0][s]), 1);
      mbar_init(smem_u32(&sm.empty[1][s]), 1);
    }
    for (int s = 0; s < kDescRing; ++s) {
      mbar_init(smem_u32(&sm.d_full[s]), 1);
      mbar_init(smem_u32(&sm.d_empty[s]), kFp8 ? 11 : 10);  // MMA, softmax and (e4m3) widening warps
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(smem_u32(&sm.q_full[t]), 128);
      for (int h = 0; h < 2; ++h) {
        mbar_init(smem_u32(&sm.s_full[t][h]), 1);
        mbar_init(smem_u32(&sm.p_full[t][h]), 128);
      }
      mbar_init(smem_u32(&sm.pv_done[t]), 1);
      mbar_init(smem_u32(&sm.o_full[t]), kTree ? 2 : 1);
      mbar_init(smem_u32(&sm.wg[t]), 128);
    }
    if constexpr (kFp8) {
      for (int t = 0; t < 2; ++t)
        for (int k = 0; k < kWide; ++k) {
          mbar_init(smem_u32(&sm.wide.full[t][k]), 1);
          mbar_init(smem_u32(&sm.wide.empty[t][k]), 1);
        }
    }
    mbar_init(smem_u32(&sm.m_sync), 2);
    mbar_init(smem_u32(&sm.drain), 2);
    sm.abort_flag = 0;
    if constexpr (kTree) {
      for (int n = 0; n < kTakenOut; ++n) sm.tree.taken_out[n] = 0;
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&sm.tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = sm.tmem_base;

  // Cursor of a consumer in the descriptor ring: waits for the next segment, copies it, releases.
  int d_slot = 0, d_phase = 0;
  auto next_segment = [&](Segment& g) -> bool {
    const bool ok = mbar_wait(smem_u32(&sm.d_full[d_slot]), d_phase, abort_flag, p.err);
    if (!__all_sync(0xffffffffu, ok)) return false;
    g = sm.desc[d_slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sm.d_empty[d_slot]));
    if (++d_slot == kDescRing) {
      d_slot = 0;
      d_phase ^= 1;
    }
    return g.live != 0;
  };

  // every warp of a warpgroup executes the same setmaxnreg at the top of its role
  if (warp == 0) {
    // ================================================================ schedule and TMA
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kBrRegsControl));
    flag_lengths(p, lane);
    const int all = pl.head_weight * p.kv_heads;
    int u = min(all, static_cast<int>(blockIdx.x) * pl.cut);
    int u_end = min(all, u + pl.cut);
    Place at = {0, -1, 0, 0};
    if (u < u_end) at = locate(p, ln, pl, u, lane);
    // A range that starts inside an item and goes on past it takes that rest last. All CTAs then
    // walk their items from the first block on, and those that read the same keys read them at
    // about the same time, from L2.
    int later = 0;
    Place later_at = at;
    if (u < u_end && at.off > 0) {
      const PlaceUnits it = place_units(p, ln, pl, at);
      const int rest = weight_of(ln, it.units, it.cost) - at.off;
      if (rest < u_end - u) {
        later = rest;
        u += rest;
        step_item(p, ln, pl, at);
      }
    }
    // Keys that one item alone reads would push everything else out of L2, the kernel's own code
    // and queries among it, whose next reads then queue behind them for memory.
    const bool once = ln.shared_tiles <= 1 && ln.own_tiles <= 1;
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    int ring = 0;  // next tile of the K/V ring
    int issued = 0, last_tile = 1;
    // A bit per slot: which tiles read its latest load (each releases it on a barrier of its own),
    // the parities of those releases, whose full barrier it signals and that one's parity.
    uint32_t used0 = 0u, used1 = 0u, free0 = 0u, free1 = 0u, on_tile1 = 0u, full0 = 0u, full1 = 0u;
    int ds = 0, ds_phase = 0;
    bool ok = true;
    for (int number = 1; ok; ++number) {
      // ---- the next segment: what is left of the current item within the CTA's range
      Segment g;
      memset(&g, 0, sizeof(g));
      g.number = number;
      int seq = 0;
      while (u < u_end && !g.live) {
        const PlaceUnits it = place_units(p, ln, pl, at);
        const UnitRange in = units_in(ln, it, at.off, u_end - u);
        const int blocks = in.count;
        if (blocks > 0) {
          long long item, row0;
          int slot_rows;
          if (at.b < 0) {
            seq = pl.longest;
            g.row0 = at.t * kSpan;
            g.n_rows = min(kSpan, pl.live - g.row0);
            g.block0 = in.first;
            g.kv_end = g.clean = pl.shared_blocks * kBlk;
            item = at.head * ln.shared_tiles + at.t;
            row0 = 0;
            slot_rows = p.shared_slot_rows;
          } else {
            seq = at.b;
            g.row0 = at.b * p.rows * p.group + at.t * kSpan;
            const Extent x = extent_of(p, at.b);
            g.n_rows = min(kSpan, x.rows - at.t * kSpan);
            g.kv_end = x.all;
            g.clean = x.clean;
            g.block0 = own_lo(p, x) / kBlk + in.first;
            item = (static_cast<long long>(at.head) * p.batch + at.b) * ln.own_tiles + at.t;
            row0 = p.own_row0;
            slot_rows = p.own_slot_rows;
          }
          for (int k = 0; k < 2; ++k) g.slot_row[k] = row0 + ((item + blockIdx.x) * 2 + k) * slot_rows;
          g.live = at.b < 0 ? 2 : 1;
          g.head = at.head;
          g.blocks = blocks;
          g.direct = pl.shared_blocks == 0 && blocks == it.units && (g.n_rows > kBlk || blocks == 1);
        }
        u += in.part;
        if (u < u_end) {
          step_item(p, ln, pl, at);
        } else if (later > 0) {
          at = later_at;
          u_end = u + later;
          later = 0;
        }
      }
      ok = mbar_wait(smem_u32(&sm.d_empty[ds]), ds_phase ^ 1, abort_flag, p.err);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      if (lane == 0) {
        sm.desc[ds] = g;
        mbar_arrive(smem_u32(&sm.d_full[ds]));
      }
      if (++ds == kDescRing) {
        ds = 0;
        ds_phase ^= 1;
      }
      if (!g.live) break;
      // ---- its blocks
      const bool pair = g.n_rows > kBlk;
      const int first_tile = last_tile ^ 1;
      int pages = 0, page = 0, page_before = 0;  // 32 blocks', and those of the last two K
      for (int i = 0, k = 0; ok && i < 2 * g.blocks; ++i) {
        const bool is_k = Cfg::kSkew ? i == 0 || ((i & 1) && k < g.blocks) : (i & 1) == 0;
        if (is_k) {
          if ((k & 31) == 0) {
            pages = k + lane < g.blocks ? __ldg(p.table + static_cast<size_t>(seq) * p.width + g.block0 + k + lane) : 0;
            if (__any_sync(0xffffffffu, pages < 0 || pages >= p.pool_pages)) {
              if (lane == 0) {
                if (p.err) atomicOr(p.err, kErrBadPage);
                *abort_flag = 1;
              }
              ok = false;
              break;
            }
          }
          page_before = page;
          page = __shfl_sync(0xffffffffu, pages, k & 31);
          ++k;
        }
        {
          const int j = is_k || !Cfg::kSkew || i == 2 * g.blocks - 1 ? k - 1 : k - 2;  // the block
          const int pg = j == k - 1 ? page : page_before;
          const uint32_t bit = 1u << ring;
          if (used0 & bit) {
            ok = mbar_wait(smem_u32(&sm.empty[0][ring]), (free0 >> ring) & 1u, abort_flag, p.err);
            free0 ^= bit;
          }
          if (ok && (used1 & bit)) {
            ok = mbar_wait(smem_u32(&sm.empty[1][ring]), (free1 >> ring) & 1u, abort_flag, p.err);
            free1 ^= bit;
          }
          if (!(ok = __all_sync(0xffffffffu, ok))) break;
          // a block of one tile signals that tile's barrier, a shared one tile 0's
          const int side = pair ? 0 : first_tile ^ (j & 1);
          const bool widened = kFp8 && !is_k;  // warp 3 alone reads it, and releases it on tile 0's
          used0 = pair || side == 0 || widened ? used0 | bit : used0 & ~bit;
          used1 = (pair || side == 1) && !widened ? used1 | bit : used1 & ~bit;
          on_tile1 = side ? on_tile1 | bit : on_tile1 & ~bit;
          if (side) full1 ^= bit;
          else full0 ^= bit;
          if (lane == 0) {
            const uint32_t bar = smem_u32(&sm.full[side][ring]);
            mbar_expect_tx(bar, Cfg::kTile);
            const CUtensorMap* map = is_k ? &tmK : &tmV;
            for (int a = 0; a < Cfg::kTile / kAtom; ++a) {
              const uint32_t dst = smem_u32(sm.kv[ring]) + a * kAtom;
              if (once) tma_load_3d_once(dst, map, bar, a * (128 / Cfg::kElem), pg * kBlk, g.head, policy);
              else tma_load_3d(dst, map, bar, a * (128 / Cfg::kElem), pg * kBlk, g.head);
            }
          }
          ++issued;
          if (++ring == kS) ring = 0;
        }
      }
      last_tile = pair ? 1 : first_tile ^ ((g.blocks - 1) & 1);
    }
    if (!ok) {
      // leaving early: no copy may still be in flight when the CTA ends
      for (int i = 0; i < min(issued, kS); ++i) {
        if (--ring < 0) ring = kS - 1;
        const int side = (on_tile1 >> ring) & 1u;
        const uint32_t ph = (((side ? full1 : full0) >> ring) & 1u) ^ 1u;
        const unsigned long long t0 = global_ns();
        while (!mbar_try_wait(smem_u32(&sm.full[side][ring]), ph) && global_ns() - t0 < kWaitTimeoutNs) {
        }
      }
    }
  } else if (warp == 1 || warp == 2) {
    // ================================================================ MMA issue
    // Warp 1 serves tile 0 and warp 2 tile 1: a warp stays blocked in tcgen05.mma until the tensor
    // pipe takes the instruction, so one issuer for both tiles left the pipe idle half the time
    // (2000 cycles a block of one tile, of which 1024 are MMAs).
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kBrRegsControl));
    const int mt = warp - 1;
    const uint32_t klo0 = sdesc_lo(smem_u32(sm.kv[0]), 16);
    constexpr uint32_t kTileDesc = Cfg::kTile >> 4;
    uint32_t vlo0;  // V: a slot of the ring, or a widened block
    if constexpr (kFp8) vlo0 = sdesc_lo(smem_u32(sm.wide.v[0]), kAtom);
    else vlo0 = sdesc_lo(smem_u32(sm.kv[0]), kAtom);
    const uint32_t qlo = sdesc_lo(smem_u32(sm.q[mt]), 16);
    const uint32_t tS = tbase + static_cast<uint32_t>(mt) * 128u;
    const uint32_t tO = tbase + 256u + static_cast<uint32_t>(mt) * 128u;
    const uint32_t q_bar = smem_u32(&sm.q_full[mt]), s_bar = smem_u32(&sm.s_full[mt]);
    const uint32_t p_bar = smem_u32(&sm.p_full[mt]), o_bar = smem_u32(&sm.o_full[mt]);
    const uint32_t pv_bar = smem_u32(&sm.pv_done[mt]);
    int ring = 0;  // K tile of the next unit
    int wide = 0;  // e4m3: the next widened block
    // The next phase of each slot's two full barriers, a bit per slot: a tile's own blocks land
    // on its barrier, blocks of both tiles on that of tile 0. So a warp never waits on a phase
    // whose predecessor it skipped.
    uint32_t phase0 = 0u, phase1 = 0u;
    uint32_t wide0 = 0u, wide1 = 0u;  // and those of the widened blocks' barriers
    uint32_t q_ph = 0u, p_ph = 0u, m_ph = 0u;
    int last_tile = 1;
    bool ok = true, was_solo = false;
    // the P V of this tile's last block, still to be issued
    bool pend = false, pend_acc = false;
    int pend_slot = 0, pend_rows = 0, pend_clean = 0;
    uint32_t pend_bar = 0u, pend_ph = 0u;
    Segment g;  // which holds the pending block
    // Waits for P of one half of the pending block and issues its P V.
    auto finish = [&](int half) {
      const bool w = mbar_wait(p_bar + half * 8, p_ph, abort_flag, p.err);
      if (!(ok = __all_sync(0xffffffffu, w))) return;
      tc_fence_after();
      if (!kFp8 && min(pend_rows, kTree ? pend_clean : kBlk) < kBlk && half == 0) {  // e4m3: done when widened
        clear_block<kTree>(smem_u32(sm.kv[pend_slot]), min(pend_rows, kBlk), pend_clean, lane, [&]() {
          if constexpr (kTree) mark_taken_out(sm.tree, g.number);
        });
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      const uint32_t vh = vlo0 + static_cast<uint32_t>(pend_slot) * (2 * kAtom >> 4) + half * ((64 * 128) >> 4);
      const uint32_t acc = pend_acc || half > 0 ? 1u : 0u;
      const uint32_t tP = tS + 64u * half;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        mma_ts(tO, tP + kk * 8, sdesc_join(vh + ((kk * 16 * 128) >> 4)), Cfg::kIdescPV, kk > 0 ? 1u : acc);
      tc_commit(pv_bar);
      if (half == 1) p_ph ^= 1u;
    };
    // Q K^T over 64 rows of a K tile.
    auto scores = [&](uint32_t klo, int half) {
      const uint32_t kh = klo + half * ((64 * 128) >> 4), tD = tS + 64u * half;
#pragma unroll
      for (int kk = 0; kk < Cfg::kSteps; ++kk) {
        const uint32_t step = ((kk * 32 / 128) * kAtom + (kk * 32) % 128) >> 4;
        if constexpr (kFp8) {
          mma_ss_f8(tD, sdesc_join(qlo + step), sdesc_join(kh + step), Cfg::kIdescQK, kk > 0 ? 1u : 0u);
          mma_ss_f8(tD, sdesc_join(qlo + (kAtom >> 4) + step), sdesc_join(kh + step), Cfg::kIdescQK, 1u);
        } else {
          mma_ss(tD, sdesc_join(qlo + step), sdesc_join(kh + step), Cfg::kIdescQK, kk > 0 ? 1u : 0u);
        }
      }
      tc_commit(s_bar + half * 8u);
    };
    const auto free_slot = [&](int slot) { tc_commit(smem_u32(&sm.empty[mt][slot])); };
    const auto free_v = [&]() {
      if constexpr (kFp8) tc_commit(smem_u32(&sm.wide.empty[mt][pend_slot]));
      else free_slot(pend_slot);
    };
    auto wait_v = [&]() { ok = __all_sync(0xffffffffu, mbar_wait(pend_bar, pend_ph, abort_flag, p.err)); };
    auto finish_item = [&]() {  // the last P V of an item
      pend = false;
      wait_v();
      if (ok) finish(0);
      if (ok) finish(1);
      if (!ok) return;
      tc_commit(o_bar);
      if constexpr (kTree) {  // and what this warp knows of taken_out
        __syncwarp();
        if (lane == 0) mbar_arrive(o_bar);
      }
      free_v();
    };
    const auto wrap = [](int slot) { return slot >= kS ? slot - kS : slot; };
    while (ok && next_segment(g)) {
      const bool pair = g.n_rows > kBlk;
      if (pair && was_solo) {
        // From here this warp also waits on tile 0's barriers: both warps first see all blocks
        // they loaded alone.
        if (lane == 0) mbar_arrive(smem_u32(&sm.m_sync));
        bool w = mbar_wait(smem_u32(&sm.m_sync), m_ph, abort_flag, p.err);
        m_ph ^= 1u;
        if (!(ok = __all_sync(0xffffffffu, w))) break;
      }
      was_solo = !pair;
      bool first = true;
      for (int j = 0; ok && j < g.blocks; ++j) {
        const int owner = pair ? mt : last_tile ^ 1;
        const bool last = j == g.blocks - 1;
        const int vs = wrap(ring + (Cfg::kSkew ? (j == 0 ? 2 : 3) - last : 1));  // its V
        const bool second = !pair && owner == 1;
        if (owner == mt) {
          const uint32_t phases = second ? phase1 : phase0;
          if (first) {
            ok = __all_sync(0xffffffffu, mbar_wait(q_bar, q_ph, abort_flag, p.err));
            q_ph ^= 1u;
          } else {
            wait_v();
          }
          if (!ok) break;
          const uint32_t klo = klo0 + static_cast<uint32_t>(ring) * kTileDesc;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (!first) finish(half);
            if (!ok) break;
            if (half == 0) {
              const bool w = mbar_wait(smem_u32(&sm.full[second][ring]), (phases >> ring) & 1u, abort_flag, p.err);
              if (!(ok = __all_sync(0xffffffffu, w))) break;
            }
            tc_fence_after();
            scores(klo, half);
          }
          if (!ok) break;
          if (!first) free_v();
          free_slot(ring);
          pend = true;
          pend_acc = !first;
          if constexpr (kFp8) {
            pend_slot = wide;
            pend_bar = smem_u32(&sm.wide.full[second][wide]);
            pend_ph = ((second ? wide1 : wide0) >> wide) & 1u;
          } else {
            pend_slot = vs;
            pend_bar = smem_u32(&sm.full[second][vs]);
            pend_ph = (phases >> vs) & 1u;
          }
          pend_rows = g.kv_end - (g.block0 + j) * kBlk;
          pend_clean = g.clean - (g.block0 + j) * kBlk;
          first = false;
        }
        const uint32_t bits = (1u << ring) | (1u << vs);
        if (second) phase1 ^= bits;
        else phase0 ^= bits;
        if constexpr (kFp8) {
          if (second) wide1 ^= 1u << wide;
          else wide0 ^= 1u << wide;
          if (++wide == kWide) wide = 0;
        }
        last_tile = pair ? 1 : owner;
        ring = wrap(last ? vs + 1 : ring + (Cfg::kSkew && j == 0 ? 1 : 2));
      }
      if (ok && pend) finish_item();
    }
    // leave no tensor-core work in flight past the teardown
    tc_commit(smem_u32(&sm.drain));
    const unsigned long long t0 = global_ns();
    while (!mbar_try_wait(smem_u32(&sm.drain), 0)) {
      if (global_ns() - t0 > kWaitTimeoutNs) {
        if (p.err && lane == 0) atomicOr(p.err, kErrWaitTimeout);
        break;
      }
    }
  } else if (warp >= 4) {
    // ================================================================ softmax and epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kBrRegsSoftmax));
    const int t = (warp - 4) >> 2;
    const int quad = warp & 3;
    const int lr = quad * 32 + lane;  // TMEM lane
    const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t tS = tbase + static_cast<uint32_t>(t) * 128u + lane_off;
    const uint32_t tO = tbase + 256u + static_cast<uint32_t>(t) * 128u + lane_off;
    uint32_t s_ph = 0u, o_ph = 0u, wg_ph = 0u;
    int last_tile = 1;
    bool ok = true;
    // all 128 threads of the tile meet (bounded, so a broken pipeline cannot hang it)
    auto meet = [&]() {
      mbar_arrive(smem_u32(&sm.wg[t]));
      ok = mbar_wait(smem_u32(&sm.wg[t]), wg_ph, abort_flag, p.err);
      wg_ph ^= 1u;
      ok = __all_sync(0xffffffffu, ok);
      return ok;
    };
    struct Item {
      int mine, begin, step;  // blocks of this tile: how many, the first, every step-th
      int block0, head, row0, n_rows, span;  // of this tile; span: rows a copy has room for
      int marks;  // four times the segment's number, 2 if against the shared blocks, 1 if direct (in one register)
      long long ws_row;
      RowAt at;  // this thread's row
    };
    uint4 qv[16];  // and its query
    // The next segment that this tile has blocks of; starts loading its query rows.
    auto take = [&](Item& it) -> bool {
      Segment g;
      while (next_segment(g)) {
        const bool pair = g.n_rows > kBlk;
        it.begin = pair ? 0 : ((last_tile ^ 1) == t ? 0 : 1);
        it.step = pair ? 1 : 2;
        it.mine = g.blocks > it.begin ? (g.blocks - it.begin + it.step - 1) / it.step : 0;
        last_tile = pair ? 1 : (last_tile ^ (g.blocks & 1));
        const int r0 = pair ? t * kBlk : 0;
        it.n_rows = min(kBlk, g.n_rows - r0);
        it.ws_row = g.slot_row[t];
        if (it.mine == 0) {
          if (!g.direct && lr < it.n_rows) p.part_ml[it.ws_row + lr] = make_float2(-INFINITY, 0.f);
          continue;
        }
        it.span = kTree || g.n_rows > 64 ? 128 : it.n_rows <= 32 ? 32 : 64;
        it.block0 = g.block0 + it.begin;
        it.head = g.head;
        it.row0 = g.row0 + r0;
        it.marks = 4 * g.number + (g.live == 2 ? 2 : 0) + g.direct;
        const int my = lr & (it.span - 1);
        const int row = it.row0 + min(my, it.n_rows - 1);
        if constexpr (kTree) it.at = (it.marks & 2) && p.compact ? live_row_at(p, sm.tree.before, g.head, row) : row_at(p, g.head, row);
        else it.at = row_at(p, g.head, row);
        const uint4* src = reinterpret_cast<const uint4*>(p.q + it.at.b * p.q_sb + it.at.i * p.q_sn + it.at.h * p.q_sh);
#pragma unroll
        for (int c = 0; c < 16; ++c) qv[c] = my < it.n_rows ? __ldg(src + c) : make_uint4(0u, 0u, 0u, 0u);
        return true;
      }
      return false;
    };
    Item next;
    bool more = take(next);
    while (more) {
      const Item it = next;
      const bool direct = it.marks & 1;
      const int span = kTree ? kBlk : it.span, n_rows = it.n_rows, copies = kBlk / span;
      const int my = lr & (span - 1);  // this thread's row of the tile
      const int copy = lr / span;      // and which copy of it
      float sl2 = p.scale_log2 * store_query_row<kFp8>(sm.q[t], my, copy, copies, span, qv);
      if constexpr (kFp8) sl2 = score_factor(sl2 * __ldg(p.k_scale + it.head));
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(smem_u32(&sm.q_full[t]));
      const auto sight = sight_of(p, it.at, (it.marks & 2) != 0);
      const bool warp_live = quad * 32 % span < n_rows;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; ok && j < it.mine; ++j) {
        const int key0 = (it.block0 + j * it.step) * kBlk;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          ok = mbar_wait(smem_u32(&sm.s_full[t][h]), s_ph, abort_flag, p.err);
          if (!(ok = __all_sync(0xffffffffu, ok))) break;
          tc_fence_after();
          const bool first = j == 0 && h == 0;
          const auto pv_done = [&]() {
            if (!first) ok = mbar_wait(smem_u32(&sm.pv_done[t]), h ^ 1, abort_flag, p.err);
          };
          if (!warp_live) {
            pv_done();
          } else if (span == 128) {
            softmax_half<kFp8, 64>(p, tS, tO, h, 0, key0, sight, sl2, first, m, l, pv_done);
          } else if constexpr (!kTree) {
            if (span == 64) softmax_half<kFp8, 32>(p, tS, tO, h, copy, key0, sight, sl2, first, m, l, pv_done);
            else softmax_half<kFp8, 16>(p, tS, tO, h, copy, key0, sight, sl2, first, m, l, pv_done);
          }
          tc_fence_before();
          mbar_arrive(smem_u32(&sm.p_full[t][h]));
        }
        s_ph ^= 1u;
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if constexpr (kTree) {
        if (sight.hidden()) {
          m = -INFINITY;
          l = 0.f;
        }
      }
      more = take(next);  // its query rows arrive while this item's O is written
      ok = mbar_wait(smem_u32(&sm.o_full[t]), o_ph, abort_flag, p.err);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      o_ph ^= 1u;
      tc_fence_after();
      if constexpr (kTree) {  // what was taken out of V, to the rows that see it
        const volatile int& taken_out = sm.tree.taken_out[it.marks / 4 % kTakenOut];
        if (__any_sync(0xffffffffu, taken_out == it.marks / 4)) {
          const NodeValues<kFp8> nodes(p, it.at.b, it.head);
          const int key_end = (it.block0 + (it.mine - 1) * it.step + 1) * kBlk;
#pragma unroll 1
          for (int c = 0; c < kD; ++c) {  // column by column, for its code: it is seldom needed
            const float lost = my < n_rows ? nodes.non_finite_sum(p, sight, c, it.block0 * kBlk, key_end, it.step) : 0.f;
            __syncwarp();
            const float o = __uint_as_float(tmem_ld1(tO + c));
            tmem_st1(tO + c, __float_as_uint(lost == 0.f ? o : o + lost));  // none: perhaps the other tile's, which may come late
          }
          tmem_wait_st();
        }
      }
      // ---- epilogue, through the query tile's buffer (every Q K^T of this item is complete)
      float* const stage = reinterpret_cast<float*>(sm.q[t]);
      float top = m, sum = l;
      const int n_lanes = n_rows * copies;  // lanes that hold something
      if (span < 128) {  // the copies' maxima and sums; kept clear of the rows staged first
        float2* const ml = reinterpret_cast<float2*>(sm.q[t] + kQBytes - 1024);
        ml[lr] = make_float2(m, l);
        if (!meet()) break;
        float2 v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = c < copies ? ml[c * span + my] : make_float2(-INFINITY, 0.f);
        top = fmax3(fmaxf(v[0].x, v[1].x), v[2].x, v[3].x);
        sum = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) sum += v[c].y != 0.f ? fast_exp2(v[c].x - top) * v[c].y : 0.f;
        if (n_lanes > 124 && !meet()) break;
      }
      // A copy that saw nothing weighs nothing; sums that are NaN stay so.
      float weight = l == 0.f ? 0.f : fast_exp2(m - top);
      if (direct) {
        weight = sum == 0.f ? 0.f : weight / sum;
        if constexpr (kFp8) weight *= __ldg(p.v_scale + it.head);
      }
      if (my < n_rows && copy == 0) {
        const float base = top - (kFp8 ? kBoostF8 : 0.f);
        if (!direct) p.part_ml[it.ws_row + my] = make_float2(base, sum);
        else if (p.lse)
          p.lse[(static_cast<long long>(it.at.b) * p.rows + it.at.i) * p.heads + it.at.h] =
              sum == 0.f ? -INFINITY : (base + log2f(sum)) * 0.6931471805599453f;
      }
      // Four columns of O times the weight. O of a copy that weighs nothing may hold NaN (a hidden
      // infinity of V times P's zeros): it counts as zero.
      const auto scaled = [&](const uint32_t (&o)[32], int j) {
        float4 a;
        a.x = weight == 0.f ? 0.f : __uint_as_float(o[4 * j]) * weight;
        a.y = weight == 0.f ? 0.f : __uint_as_float(o[4 * j + 1]) * weight;
        a.z = weight == 0.f ? 0.f : __uint_as_float(o[4 * j + 2]) * weight;
        a.w = weight == 0.f ? 0.f : __uint_as_float(o[4 * j + 3]) * weight;
        return a;
      };
      const long long own_dst = ((static_cast<long long>(it.at.b) * p.rows + it.at.i) * p.heads + it.at.h) * kD;
      if (span == 128) {
        // a warp turns its 32 rows around by itself, 64 columns at a time, and writes whole lines
        float* const mine = stage + quad * (32 * 64);
#pragma unroll 1
        for (int half = 0; warp_live && half < 2; ++half) {
          uint32_t o[2][32];
          tmem_ld32(tO + half * 64, o[0]);
          tmem_ld32(tO + half * 64 + 32, o[1]);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            reg_fence32(o[c]);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<float4*>(mine + lane * 64 + (((c * 8 + j) ^ (lane & 7)) << 2)) = scaled(o[c], j);
          }
          __syncwarp();
#pragma unroll 4
          for (int i = 0; i < 16; ++i) {
            const int r = i * 2 + (lane >> 4), c4 = lane & 15;
            const float4 a = *reinterpret_cast<const float4*>(mine + r * 64 + ((c4 ^ (r & 7)) << 2));
            const int lo = __shfl_sync(0xffffffffu, static_cast<int>(own_dst), r);
            const int hi = __shfl_sync(0xffffffffu, static_cast<int>(own_dst >> 32), r);
            if (quad * 32 + r >= n_rows) continue;
            if (direct) {
              const long long dst = static_cast<long long>(static_cast<uint32_t>(lo)) | (static_cast<long long>(hi) << 32);
              *reinterpret_cast<uint2*>(p.out + dst + half * 64 + c4 * 4) =
                  make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
            } else {
              *reinterpret_cast<float4*>(p.part_o + (it.ws_row + quad * 32 + r) * kD + half * 64 + c4 * 4) = a;
            }
          }
          __syncwarp();
        }
        ok = meet();
      } else {
        // the copies' rows side by side, all columns at once where they fit, then their sums
        const int shift = n_lanes <= 60 ? 5 : 4;  // float4s of a staged row
        const int slot = copy * n_rows + my;
#pragma unroll 1
        for (int c0 = 0; ok && c0 < 32; c0 += 1 << shift) {
          if (warp_live) {
#pragma unroll 1
            for (int c = 0; c < 1 << shift; c += 16) {
              uint32_t o[2][32];
              tmem_ld32(tO + (c0 + c) * 4, o[0]);
              tmem_ld32(tO + (c0 + c) * 4 + 32, o[1]);
              tmem_wait_ld();
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                reg_fence32(o[half]);
                if (my >= n_rows) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  *reinterpret_cast<float4*>(stage + (((slot << shift) + ((c + half * 8 + j) ^ (slot & 7))) << 2)) =
                      scaled(o[half], j);
              }
            }
          }
          if (!meet()) break;
          for (int i = lr; i < n_rows << shift; i += 128) {
            const int r = i >> shift, c4 = i & ((1 << shift) - 1);
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int c = 0; c < copies; ++c) {
              const int from = c * n_rows + r;
              const float4 v = *reinterpret_cast<const float4*>(stage + (((from << shift) + (c4 ^ (from & 7))) << 2));
              a.x += v.x;
              a.y += v.y;
              a.z += v.z;
              a.w += v.w;
            }
            if (direct) {
              const RowAt ra = row_at(p, it.head, it.row0 + r);
              __nv_bfloat16* dst =
                p.out + ((static_cast<long long>(ra.b) * p.rows + ra.i) * p.heads + ra.h) * kD;
              *reinterpret_cast<uint2*>(dst + (c0 + c4) * 4) = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
            } else {
              *reinterpret_cast<float4*>(p.part_o + (it.ws_row + r) * kD + (c0 + c4) * 4) = a;
            }
          }
          if (!meet()) break;
        }
      }
      tc_fence_before();
      if (!ok) break;
    }
  } else {
    // ================================================================ warp 3
    // of the first CTA writes the schedule down for the merge
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kBrRegsControl));
    if (blockIdx.x == 0) {
      pl = make_plan(p, ln, lane);
      write_plan(p, ln, pl, p.plan, lane);
    }
    if constexpr (kFp8) {
      // Widens V, rows past the sequence's end as zeros.
      int ring = 1, wide = 0, last_tile = 1;
      // a bit per slot of the ring: parities of the two full barriers; a bit per widened block: which
      // tiles read its latest content, and the parities of their releases
      uint32_t phase0 = 0u, phase1 = 0u, used0 = 0u, used1 = 0u, free0 = 0u, free1 = 0u;
      bool ok = true;
      Segment g;
      while (ok && next_segment(g)) {
        const bool pair = g.n_rows > kBlk;
        for (int j = 0; j < g.blocks; ++j) {
          const int side = pair ? 0 : last_tile ^ 1;
          const uint32_t bit = 1u << wide, slot_bit = 1u << ring;
          if (used0 & bit) {
            ok = mbar_wait(smem_u32(&sm.wide.empty[0][wide]), (free0 >> wide) & 1u, abort_flag, p.err);
            free0 ^= bit;
          }
          if (ok && (used1 & bit)) {
            ok = mbar_wait(smem_u32(&sm.wide.empty[1][wide]), (free1 >> wide) & 1u, abort_flag, p.err);
            free1 ^= bit;
          }
          if (ok) ok = mbar_wait(smem_u32(&sm.full[side][ring]), ((side ? phase1 : phase0) >> ring) & 1u, abort_flag, p.err);
          if (!(ok = __all_sync(0xffffffffu, ok))) break;
          if (side) phase1 ^= slot_bit;
          else phase0 ^= slot_bit;
          const int rows = g.kv_end - (g.block0 + j) * kBlk;  // that hold anything
          const int clean = g.clean - (g.block0 + j) * kBlk;
          const uint32_t from = smem_u32(sm.kv[ring]), to = smem_u32(sm.wide.v[wide]);
          if (kTree && clean < kBlk) {
            if constexpr (kTree) {
              if (widen_block<true, true>(from, to, rows, clean, lane)) mark_taken_out(sm.tree, g.number);
            }
          } else if (kTree || rows >= kBlk) {  // a tree's last rows are nodes
            widen_block<false, false>(from, to, kBlk, 0, lane);
          } else {
            widen_block<true, false>(from, to, rows, 0, lane);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(smem_u32(&sm.empty[0][ring]));
            mbar_arrive(smem_u32(&sm.wide.full[side][wide]));
          }
          used0 = pair || side == 0 ? used0 | bit : used0 & ~bit;
          used1 = pair || side == 1 ? used1 | bit : used1 & ~bit;
          last_tile = pair ? 1 : side;
          ring = ring + 2 > kS ? 1 : ring + 2;
          if (++wide == kWide) wide = 0;
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

// Joins the pieces of every row that more than one segment (or tile) contributed to, in the order
// of the units, and writes rows that see nothing. A warp takes a row (kTeam warps share one in long
// shared items) and reads several pieces at a time, maximum, sum and O alike before it needs any of
// them: what bounds this kernel is the latency of reads from L2, and reading O only after the
// weights had been found took 18 us instead of 8.5 for 480 rows of 38 pieces. In the joint form few
// pieces make a row and a warp takes kRows rows at once instead.
constexpr int kMergeWarps = 4;
constexpr int kJointWarpRows = 4;  // joint form: rows of a warp

struct Pieces {  // of one row in one item: workspace rows first + j * stride, j < n
  int n, stride;
  long long first;
};
__device__ __forceinline__ Pieces pieces_of(int cut, int u0, int units, int cost, int n_rows, int r, long long item,
                                            long long row0, int slot_rows, bool warps) {
  if (units == 0) return Pieces{0, 0, 0};
  const int c_lo = u0 / cut, n_cta = (u0 + (units - 1) * cost) / cut - c_lo + 1;
  if (warps) return Pieces{n_cta, slot_rows, row0 + (item + c_lo) * slot_rows + r};
  const long long first = row0 + (item + c_lo) * 2 * slot_rows;
  // items of both tiles: the slot of the row's tile in each CTA; else the slots of both
  if (n_rows > kBlk) return Pieces{n_cta, 2 * slot_rows, first + (r / kBlk) * slot_rows + r % kBlk};
  return Pieces{2 * n_cta, slot_rows, first + r};
}

// Adds the pieces of kRows rows, kB at a time and every kTeam-th batch from the part-th on, to their
// running maxima, sums and O.
template <int kRows, int kB, int kTeam>
__device__ __forceinline__ void add_pieces(const BranchParams& p, const Pieces (&q)[kRows], int part, int lane,
                                         float (&m)[kRows], float (&sum)[kRows], float4 (&acc)[kRows]) {
  const int n = q[0].n;  // the rows of a warp are rows of one item
  const float2* ml_at[kRows];
  const float4* o_at[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    ml_at[k] = p.part_ml + q[k].first;
    o_at[k] = reinterpret_cast<const float4*>(p.part_o) + q[k].first * (kD / 4) + lane;
  }
  for (int i0 = part * kB; i0 < n; i0 += kTeam * kB) {
    float2 ml[kRows][kB];
    float4 v[kRows][kB];
#pragma unroll
    for (int k = 0; k < kRows; ++k)
#pragma unroll
      for (int j = 0; j < kB; ++j) {
        ml[k][j] = make_float2(-INFINITY, 0.f);
        if (i0 + j < n) {
          const long long at = static_cast<long long>(i0 + j) * q[k].stride;
          ml[k][j] = __ldcg(ml_at[k] + at);
          v[k][j] = __ldcg(o_at[k] + at * (kD / 4));
        }
      }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      float top = m[k];
#pragma unroll
      for (int j = 0; j < kB; ++j) top = fmaxf(top, ml[k][j].x);
      // a sum of 0: the piece saw nothing and its O was not written. Sums that are NaN stay so.
      const float keep = sum[k] != 0.f ? fast_exp2(m[k] - top) : 0.f;
      sum[k] = sum[k] != 0.f ? sum[k] * keep : 0.f;
      acc[k] = make_float4(acc[k].x * keep, acc[k].y * keep, acc[k].z * keep, acc[k].w * keep);
#pragma unroll
      for (int j = 0; j < kB; ++j) {
        if (ml[k][j].y != 0.f) {
          const float w = fast_exp2(ml[k][j].x - top);
          sum[k] += w * ml[k][j].y;
          acc[k].x += v[k][j].x * w;
          acc[k].y += v[k][j].y * w;
          acc[k].z += v[k][j].z * w;
          acc[k].w += v[k][j].w * w;
        }
      }
      m[k] = top;
    }
  }
}

template <bool kFp8, bool kJoint, int kTeam, class P>
__global__ void __launch_bounds__(32 * kMergeWarps) branch_merge_kernel(const P p) {
  constexpr int kTeams = kMergeWarps / kTeam;
  constexpr int kRows = kJoint ? kJointWarpRows : 1;
  __shared__ float4 sums[kTeam > 1 ? kMergeWarps : 1][32];
  __shared__ float2 tops[kTeam > 1 ? kMergeWarps : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int team = warp / kTeam, part = warp % kTeam;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // what each line wrote down; own items and shared items each belong to one of them
  const bool shared_by_warps = p.warp.shared_tiles > 0, own_by_warps = !kJoint && p.warp.own_tiles > 0;
  const Line& ls = shared_by_warps ? p.warp : p.tensor;
  const Line& lo = own_by_warps ? p.warp : p.tensor;
  const int line = kPlanHead + 2 * p.batch;
  const int* const ps = p.plan + (shared_by_warps ? line : 0);
  const int* const po = p.plan + (own_by_warps ? line : 0);
  const int shared_blocks = kJoint ? 0 : __ldcg(po);
  const int cut_s = __ldcg(ps + 2), cut_o = __ldcg(po + 2), live = __ldcg(ps + 3);
  const int shared_units = shared_blocks * over_pow2(kBlk, ls.unit);
  const int shared_weight = weight_of(ls, shared_units, shared_cost(p, ls, live, 0));
  bool compact = false;
  if constexpr (is_tree<P>) compact = p.compact != 0;
  const int own_all = p.rows * p.group;
  // split form: stacked rows of all branches, one a team, head by head; joint form: kRows rows of
  // an item a warp
  int head, b, t, r;
  if (!kJoint) {
    const int stacked = p.batch * own_all;
    const uint32_t id = blockIdx.x * kTeams + team;  // rows of all heads are below 2^31
    if (id >= static_cast<uint32_t>(stacked) * p.kv_heads) return;  // a whole block if kTeam > 1
    head = quotient(id, p.stacked_div);
    const int row = id - head * stacked;
    b = quotient(row, p.own_div);
    r = row - b * own_all;
    t = over_pow2(r, lo.span);
  } else {
    constexpr int kGroups = kSpan / (kRows * kMergeWarps);
    const int item = blockIdx.x / kGroups;
    t = item % lo.own_tiles;
    b = item / lo.own_tiles % p.batch;
    head = item / lo.own_tiles / p.batch;
    r = t * kSpan + (static_cast<int>(blockIdx.x % kGroups) * kMergeWarps + warp) * kRows;
    if (r >= min(own_all, (t + 1) * kSpan)) return;
  }
  const Extent ext = extent_of(p, b);
  const auto write_row = [&](int row, const float4& acc, float m, float sum) {
    float scale = sum == 0.f ? 0.f : 1.0f / sum;
    if constexpr (kFp8) scale *= __ldg(p.v_scale + head);
    const int i = quotient(row, p.group_div);
    const long long id = (static_cast<long long>(b) * p.rows + i) * p.heads + head * p.group + row - i * p.group;
    reinterpret_cast<uint2*>(p.out + id * kD)[lane] =
        make_uint2(pack_bf16x2(acc.x * scale, acc.y * scale), pack_bf16x2(acc.z * scale, acc.w * scale));
    if (p.lse && lane == 0) p.lse[id] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
  };
  if constexpr (is_tree<P>) {
    if (r >= ext.rows) {  // rows behind the nodes
      for (int k = part; k < kRows && r + k < min(own_all, (t + 1) * lo.span); k += kTeam)
        write_row(r + k, make_float4(0.f, 0.f, 0.f, 0.f), 0.f, 0.f);
      return;
    }
  }
  int u0 = head * __ldcg(po + 1) + (ps == po ? shared_weight_all(p, ls, shared_units, live, live_tiles(p, ls, live)) : 0) + __ldcg(po + kPlanHead + b);
  for (int k = 0; k < t; ++k) u0 += own_weight(p, lo, ext, k);
  const int units = own_units(p, lo, ext, t), cost_o = own_cost(p, lo, ext, t);
  const int n_rows = min(lo.span, ext.rows - t * lo.span), last = min(own_all, (t + 1) * lo.span);
  if (shared_blocks == 0 && units > 0 && u0 / cut_o == (u0 + (units - 1) * cost_o) / cut_o &&
      (own_by_warps || n_rows > kBlk || units == 1)) {  // written by the segment itself
    if constexpr (is_tree<P>) {  // but for rows behind the nodes
      for (int k = max(0, ext.rows - r); k < kRows && r + k < last; ++k) write_row(r + k, make_float4(0.f, 0.f, 0.f, 0.f), 0.f, 0.f);
    }
    return;
  }
  Pieces sh[kRows], own[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    // rows past the item (and behind the nodes) read its last row again, and what they read is not written
    const int rk = min(r + k, t * lo.span + max(n_rows, 1) - 1);
    const int row = (compact ? __ldcg(ps + kPlanHead + p.batch + b) : b * own_all) + rk, t_sh = over_pow2(row, ls.span);
    sh[k] = pieces_of(cut_s, head * __ldcg(ps + 1) + t_sh * shared_weight, compact && (rk >= ext.rows || !takes_shared(p, ext)) ? 0 : shared_units,
                      shared_cost(p, ls, live, t_sh),
                      min(ls.span, live - t_sh * ls.span), row & (ls.span - 1),
                      head * ls.shared_tiles + t_sh, 0, p.shared_slot_rows, shared_by_warps);
    own[k] = pieces_of(cut_o, u0, units, cost_o, n_rows, rk - t * lo.span,
                       (static_cast<long long>(head) * p.batch + b) * lo.own_tiles + t, p.own_row0,
                       p.own_slot_rows, own_by_warps);
  }
  float m[kRows], sum[kRows];
  float4 acc[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    m[k] = -INFINITY;
    sum[k] = 0.f;
    acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if constexpr (!kJoint) add_pieces<kRows, kTeam == 1 ? 8 : 4, kTeam>(p, sh, part, lane, m, sum, acc);
  add_pieces<kRows, kJoint ? 2 : kTeam == 1 ? 4 : 1, kTeam>(p, own, part, lane, m, sum, acc);
  if constexpr (kTeam > 1) {  // one row a team, and the teams of a block all get here
    sums[warp][lane] = acc[0];
    if (lane == 0) tops[warp] = make_float2(m[0], sum[0]);
    __syncthreads();
    if (part != 0) return;
    float top = m[0];
#pragma unroll
    for (int k = 1; k < kTeam; ++k) top = fmaxf(top, tops[warp + k].x);
    float total = 0.f;
    float4 all = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < kTeam; ++k) {
      const float2 q = tops[warp + k];
      if (q.y != 0.f) {
        const float4 x = sums[warp + k][lane];
        const float w = fast_exp2(q.x - top);
        total += q.y * w;
        all.x += x.x * w;
        all.y += x.y * w;
        all.z += x.z * w;
        all.w += x.w * w;
      }
    }
    m[0] = top;
    sum[0] = total;
    acc[0] = all;
  }
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    if (r + k >= last) break;
    if (is_tree<P> && r + k >= ext.rows) write_row(r + k, make_float4(0.f, 0.f, 0.f, 0.f), 0.f, 0.f);
    else write_row(r + k, acc[k], m[k], sum[k]);
  }
}

struct Shape {
  Line tensor, warp;
  int shared_slot_rows, own_slot_rows, joint;
  long long own_row0, rows;  // workspace rows
  long long bytes;
};

int sm_count() {
  static int counts[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (counts[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    counts[dev] = n;
  }
  return counts[dev];
}

// Branches of up to this many rows have them on the warp line. 2 KV heads over 1024 shared keys, warp /
// tensor (us): 8 branches, own lengths to 2000: 32 rows 16 / 24, 64 rows 19 / 25; 40 branches, to 1000: 25 /
// 34, 39 / 40; over 8192 shared keys and up to 300 59 / 60, e4m3 65 / 66.
constexpr int kWarpOwnRows = 64;

// The split form reads the shared blocks once for all branches and packs their rows into full tiles, but
// every row has partial results to merge; in the joint form an item that no CTA shares is written out
// as it is. So the joint form is taken where items are enough, and where the rows that its last tiles
// lack, times the shared blocks, stay below some blocks a row. 8 KV heads, own lengths to 700, bf16, joint /
// split (us) by branches x rows: 24 x 200, 2048 shared keys 86 / 135, 8192 keys 203 / 267; 8 x 180, 42 / 57
// and 82 / 95; 40 x 130, 112 / 154 and 287 / 290; 3 x 200, 33 / 38 and (13312 keys) 68 / 75; 3 x 300, 46 / 46
// and (13312) 109 / 96; 24 x 128, 1024 keys 58 / 85, 8192 keys 161 / 169; 24 x 100, 55 / 75 and 156 / 143; 40 x
// 70, 77 / 94 and 228 / 177. Few items: 2 x 200, 2048 keys 31 / 30; 1 x 300, 36 / 30; 1 x 100, 35 / 25.
bool joint_form(long long own, int batch, int kv_heads, int shared) {
  const long long workers = sm_count(), items = static_cast<long long>(kv_heads) * batch * ((own + kSpan - 1) / kSpan);
  const long long lack = (kBlk - own % kBlk) % kBlk;
  if (own <= kWarpOwnRows) return false;
  return own > kBlk ? 8 * items >= workers && lack * shared <= 28 * own : 5 * items >= 2 * workers && lack * shared <= 12 * own;
}

// Short tables on the warp line: a warp takes a branch's rows against all its keys, shared ones too, and
// there is nothing to merge. 0.8 us a 32-key unit and warp (P in two terms) then stand against the merge,
// its launch and the better spread. The limits count the launch, some 5 us of a call's host time; on the device alone, as
// in a graph, the forms meet a block or two earlier. Whole / split (us on the device), 1, 3 and 5 blocks a branch: 6 items 6.2 / 9.9, 12.5 / 10.5
// (the call 27.8 / 33, for its launch), 19 / 10.1; 96 items 6.3 / 10.7, 12.8 / 11.8, 19 / 12.2; 128 items 6.4 /
// 14.0, 12.8 / 16.4, 19.2 / 17.3; 512 items 6.9 / 15.2, 13.5 / 21.3, 20.1 / 23.5; 1600 items 14 / 25, 34 / 36,
// 54 / 39; e4m3 512 items 6.6 / 16.6, 12.4 / 23.7, 18.2 / 26.4.
bool whole_form(int width, int kv_heads, int batch, const Line& warp) {
  const long long items = static_cast<long long>(kv_heads) * batch * warp.own_tiles;
  return items > 0 && width <= (5 * items < warp.workers ? 3 : items <= warp.workers ? 6 : 4);
}

// Few rows go to the warp line: a warp takes 16 rows and needs none but itself, where an item of the
// tensor line passes a dozen barriers; what it costs is that every 16 rows read K and V again.
// Shared blocks under 8 KV heads, with merge and own parts (us, warp / tensor): bf16, 60 rows, 1024
// keys 13 / 25, 4096 keys 20 / 27, 16384 keys 42 / 45, 65536 keys 153 / 83; 240 rows, 4096 keys 35 / 40, 16384
// keys 100 / 50; 32 rows, 16384 keys 27 / 39, 65536 keys 94 / 78; 16 rows, 65536 keys 55 / 75. e4m3, 60 rows,
// 16384 keys 39 / 50, 65536 keys 111 / 79; 32 rows, 65536 keys 66 / 71; 16 rows 42 / 66.
// So: always up to one tile of rows, else up to the product where the two meet.
constexpr long long kWarpSharedWork = 600000;  // KV heads x keys x 16-row tiles
// The least part of a worker, in units: a piece costs the merge as much as some more keys cost the
// warp, and more so beside the tensor line, whose time hides the warps'. 24 branches of 4 x 32 rows,
// 8192 shared keys, own lengths to 700 (us): 8 units 50.4, 4 units 53.0, 12 units 52.8; alone, 24 KV
// heads over 1024 keys: 2 units 11.3, 4 units 12.2, 6 units 13.2.
constexpr int kWarpLeast = 2, kWarpLeastBeside = 8;

// Trees of 17 to 64 stacked rows. The warp line reads a tree's keys once for every 16 rows, the tensor line once, but starts
// some 6 us later (e4m3 10), so what decides is the keys, of which the host knows the tables' width. 8 KV heads, bf16, tensor / warp
// (us): 64 rows, 24 trees of up to 1000 keys 48.5 / 46.4, 4000 72 / 112, 16000 164 / 413; 48 rows, 1000 44 / 37, 4000 64 / 77; 32 rows,
// 2000 48 / 42, 4000 59 / 62, 16000 153 / 228; 24 rows, 2000 46 / 36, 8000 91 / 111; one tree of 64 rows over up to 8000 29 / 27, 16000
// 35 / 39, 40000 49 / 82; e4m3: 64 rows, 24 trees of 2000 73 / 64, 4000 90 / 96, 16000 157 / 281; 48 rows, 4000 84 / 74, 8000 114 / 136; 32
// rows, 16000 148 / 153. Shared keys (20 trees of 48 rows over 4096 and up to 700 of their own: 55 / 63, e4m3 64 / 62) count by
// the tiles of all trees' rows. A table wider than its longest sequence stands for keys that are not there. Tables of 8 / 256
// pages, up to 1000 keys (us): 24 trees of 24 rows 23.5 / 34.4 (e4m3 24.6 / 24.6), of 64 rows 45.7 / 46.1 (44.4 / 57.0), 4 trees of 64
// rows 18.3 / 22.9 (19.0 / 25.9); two of 9 rows and 311 keys, 3 / 256 pages, 13.6 / 12.6, but a launch more a call.
bool tree_on_tensor(int batch, int own, int kv_heads, int shared, int width, bool e4m3) {
  if (own <= kRowSpan) return false;
  const auto tiles = [](long long n, int span) { return (n + span - 1) / span; };
  const long long keys = static_cast<long long>(batch) * (width - shared) * kBlk, all = static_cast<long long>(batch) * own;
  const double warps = static_cast<double>(kv_heads) * (keys * tiles(own, kRowSpan) + 1.0 * shared * kBlk * tiles(all, kRowSpan));
  const double tensor = static_cast<double>(kv_heads) * (keys + 1.4 * shared * kBlk * tiles(all, kSpan));
  return e4m3 ? warps - 2.0 * tensor > 420000.0 : warps - 1.3 * tensor > 340000.0;
}

// The shape of a tree's call has the tables' width, a chain's 0.
Shape shape_of(int batch, int rows, int kv_heads, int group, int shared, int width = 0, bool e4m3 = false) {
  Shape s;
  memset(&s, 0, sizeof(s));
  const long long own = static_cast<long long>(rows) * group;
  const long long all = own * batch;
  const auto tiles = [](long long n, int span) { return static_cast<int>((n + span - 1) / span); };
  s.joint = joint_form(own, batch, kv_heads, shared) ? 1 : 0;
  s.tensor = Line{kSpan, kBlk, 2, 1, 1, 0, 0, sm_count(), 1};
  s.warp = Line{kRowSpan, kRowUnit, 2, 1, 1, 0, 0, sm_count() * kRowWarpsPerBlock, kWarpLeast};
  if (width > 0) {
    s.tensor.few = kFewCost;
    s.tensor.many = s.tensor.least = kManyCost;
    s.tensor.pad = e4m3 ? kTreePadF8 : kTreePad;
  }
  bool on_tensor = own > kWarpOwnRows;
  if (width > 0 && !on_tensor) {
    Line whole = s.warp;
    whole.own_tiles = tiles(own, kRowSpan);
    on_tensor = !whole_form(width, kv_heads, batch, whole) &&
                tree_on_tensor(batch, static_cast<int>(own), kv_heads, shared, width, e4m3);
  }
  Line& lo = on_tensor ? s.tensor : s.warp;
  lo.own_tiles = tiles(own, lo.span);
  s.own_slot_rows = static_cast<int>(own < lo.span ? own : lo.span);
  if (&lo == &s.tensor && own > kBlk) s.own_slot_rows = kBlk;
  const int own_slots = &lo == &s.warp ? 1 : 2;
  if (!s.joint && shared > 0) {
    const long long work = static_cast<long long>(kv_heads) * shared * kBlk * tiles(all, kRowSpan);
    const bool few = &lo == &s.warp && (all <= kRowSpan || work <= kWarpSharedWork);
    Line& ls = few ? s.warp : s.tensor;
    if (!few) s.warp.least = kWarpLeastBeside;
    ls.shared_tiles = tiles(all, ls.span);
    s.shared_slot_rows = static_cast<int>(all < ls.span ? all : ls.span);
    if (&ls == &s.tensor && all > kBlk) s.shared_slot_rows = kBlk;
    s.own_row0 = (static_cast<long long>(kv_heads) * ls.shared_tiles + ls.workers) * (&ls == &s.warp ? 1 : 2) *
                 s.shared_slot_rows;
  }
  s.rows = s.own_row0 +
           (static_cast<long long>(kv_heads) * batch * lo.own_tiles + lo.workers) * own_slots * s.own_slot_rows;
  s.bytes = s.rows * (kD * 4 + 8) + 2 * (kPlanHead + 2ll * batch) * 4;
  if (width > 0 && whole_form(width, kv_heads, batch, s.warp)) s.bytes = 0;  // nothing to merge
  return s;
}

template <bool kFp8, class P>
int configure() {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lk(mu);
  if (dev < 64 && done[dev]) return H3SA_OK;
  const auto kernel = branch_attn_kernel<kFp8, P>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(br_smem_bytes<kFp8, P>()));
  if (e != cudaSuccess) return set_cuda_error("cudaFuncSetAttribute(branch attention)", e);
  cudaFuncAttributes attr;
  e = cudaFuncGetAttributes(&attr, kernel);
  if (e != cudaSuccess) return set_cuda_error("cudaFuncGetAttributes(branch attention)", e);
  // setmaxnreg.inc waits for registers of the block's launch allocation: refuse a build that
  // cannot fund the split
  if (attr.numRegs * kBrThreads < kBrRegSplit)
    return set_error(H3SA_ERR_UNSUPPORTED, "branch attention build has %d registers per thread; the "
                     "warp-role register split needs %d", attr.numRegs,
                     (kBrRegSplit + kBrThreads - 1) / kBrThreads);
  if (dev < 64) done[dev] = true;
  return H3SA_OK;
}

template <bool kFp8, class P>
int launch_tensor(const P& p, cudaLaunchConfig_t cfg) {
  int rc = configure<kFp8, P>();
  if (rc) return rc;
  CUtensorMap tmK, tmV;
  if ((rc = encode_pool(&tmK, p, p.key_pool, kFp8, kBlk))) return rc;
  if ((rc = encode_pool(&tmV, p, p.value_pool, kFp8, kBlk))) return rc;
  cfg.gridDim = dim3(p.tensor.workers);
  cfg.blockDim = dim3(kBrThreads);
  cfg.dynamicSmemBytes = br_smem_bytes<kFp8, P>();
  cfg.numAttrs = 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, branch_attn_kernel<kFp8, P>, tmK, tmV, p);
  return e == cudaSuccess ? H3SA_OK : set_cuda_error("branch_attn_kernel launch", e);
}

template <bool kFp8, class P>
int launch(const P& p, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.stream = stream;
  // Each kernel is launched along with the one before it and waits for it on the device.
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  const bool tensor = p.tensor.own_tiles > 0 || p.tensor.shared_tiles > 0;
  if (tensor) {
    const int rc = launch_tensor<kFp8, P>(p, cfg);
    if (rc) return rc;
  }
  if (p.warp.own_tiles > 0) {  // takes the SMs that the other line is done with
    cfg.numAttrs = tensor ? 1 : 0;
    const int rc = launch_branch_rows(p, kFp8, tensor, cfg);
    if (rc || p.whole) return rc;
  }
  // Four warps share a row where rows are few, or not too many and in as many pieces as the tensor line
  // cuts a shared item into: its pieces are read one latency after another. One warp / four (us of the
  // whole call): 126 rows 13.8 / 12.8; 256 rows of 4096 shared keys (warp line) 19.8 / 17.1; 480 rows of
  // 1024 (warp line) 14.6 / 18.0, of 98304 (tensor line, e4m3) 99.2 / 98.9; 2400 rows 57.4 / 58.5.
  const long long stacked = static_cast<long long>(p.batch) * p.rows * p.heads;
  const bool team = !p.joint && stacked <= (p.tensor.shared_tiles > 0 ? 4ll : 2ll) * p.tensor.workers;
  const long long blocks =
      p.joint ? static_cast<long long>(p.kv_heads) * p.batch * p.tensor.own_tiles * (kSpan / (kJointWarpRows * kMergeWarps))
      : team  ? stacked
              : (stacked + kMergeWarps - 1) / kMergeWarps;
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(32 * kMergeWarps);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  e = p.joint ? cudaLaunchKernelEx(&cfg, branch_merge_kernel<kFp8, true, 1, P>, p)
      : team  ? cudaLaunchKernelEx(&cfg, branch_merge_kernel<kFp8, false, kMergeWarps, P>, p)
              : cudaLaunchKernelEx(&cfg, branch_merge_kernel<kFp8, false, 1, P>, p);
  if (e != cudaSuccess) return set_cuda_error("branch_merge_kernel launch", e);
  return H3SA_OK;
}

bool aligned(const void* q, size_t n) { return (reinterpret_cast<uintptr_t>(q) & (n - 1)) == 0; }

// Both attentions; `nodes`: the new rows are nodes of drafted trees, else they are a sequence's last rows.
int attend(const char* what, const TreeParams* nodes, const void* query, int64_t stride_sequence, int64_t stride_row,
           int64_t stride_head, void* out, float* lse, int32_t batch, int32_t rows, int32_t heads, int32_t kv_heads,
           const void* key_pool, const void* value_pool, int32_t pool_pages, int32_t e4m3, const float* k_scale,
           const float* v_scale, const int32_t* table, int32_t width, const int32_t* lengths, int32_t shared_rows,
           int32_t causal, float softmax_scale, void* workspace, int64_t workspace_bytes, int32_t* device_error,
           void* stream) {
  if (batch < 0 || rows < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads)
    return set_error(H3SA_ERR_INVALID, "%s: invalid sizes batch=%d rows=%d heads=%d "
                     "kv_heads=%d (heads must be a multiple of kv_heads)", what, batch, rows, heads, kv_heads);
  if (batch == 0 || rows == 0) return H3SA_OK;
  if (pool_pages <= 0 || width <= 0 || static_cast<int64_t>(pool_pages) * kBlk > INT32_MAX ||
      static_cast<int64_t>(width) * kBlk > INT32_MAX)
    return set_error(H3SA_ERR_INVALID, "%s: invalid pool of %d pages or table of %d "
                     "entries a sequence", what, pool_pages, width);
  if (shared_rows < 0 || shared_rows % kBlk || shared_rows / kBlk > width)
    return set_error(H3SA_ERR_INVALID, "%s: %d shared rows are not whole pages of a "
                     "table of %d entries", what, shared_rows, width);
  if (!query || !out || !key_pool || !value_pool || !table || !lengths ||
      (e4m3 && (!k_scale || !v_scale)))
    return set_error(H3SA_ERR_INVALID, "%s: null pointer argument", what);
  if (!(softmax_scale > 0.f) || softmax_scale > 2.0e38f)
    return set_error(H3SA_ERR_INVALID, "%s: the scale must be positive and finite", what);
  if (!aligned(query, 16) || !aligned(out, 16) || !aligned(key_pool, 16) || !aligned(value_pool, 16) ||
      !aligned(workspace, 16) || stride_sequence % 8 || stride_row % 8 || stride_head % 8)
    return set_error(H3SA_ERR_INVALID, "%s: tensors and query rows must be 16-byte aligned", what);
  if (nodes && (!nodes->masks || static_cast<int64_t>(width) * kBlk + rows > INT32_MAX))
    return set_error(H3SA_ERR_INVALID, "%s: masks are missing, or table of %d entries and %d rows too large", what, width,
                     rows);
  const int group = heads / kv_heads;
  const int64_t stacked = static_cast<int64_t>(batch) * rows * group;
  if (stacked > INT32_MAX / 2 || static_cast<int64_t>(batch) * rows * heads > INT32_MAX)
    return set_error(H3SA_ERR_UNSUPPORTED, "%s: batch %d x rows %d x heads %d is too large", what,
                     batch, rows, heads);
  Shape s = nodes ? shape_of(batch, rows, kv_heads, group, shared_rows / kBlk, width, e4m3 != 0)
                  : shape_of(batch, rows, kv_heads, group, shared_rows / kBlk);
  const auto line_units = [&](const Line& ln) {
    const int64_t blocks = kBlk / ln.unit;
    return kv_heads * (ln.shared_tiles * (shared_rows / kBlk * blocks * ln.many + ln.pad) +
                       static_cast<int64_t>(batch) * ln.own_tiles * (width * blocks * ln.many + ln.pad));
  };
  if (line_units(s.tensor) > INT32_MAX / 2 || line_units(s.warp) > INT32_MAX / 2)
    return set_error(H3SA_ERR_UNSUPPORTED, "%s: batch %d x rows %d x heads %d over %d "
                     "pages exceeds the work index", what, batch, rows, heads, width);
  if (s.bytes > 0 && !workspace) return set_error(H3SA_ERR_INVALID, "%s: null pointer argument", what);
  if (workspace_bytes < s.bytes)
    return set_error(H3SA_ERR_INVALID, "%s: workspace of %lld bytes, %lld needed", what,
                     static_cast<long long>(workspace_bytes), s.bytes);
  TreeParams p;
  memset(&p, 0, sizeof(p));
  p.q = static_cast<const __nv_bfloat16*>(query);
  p.q_sb = stride_sequence;
  p.q_sn = stride_row;
  p.q_sh = stride_head;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.table = table;
  p.lengths = lengths;
  p.width = width;
  p.batch = batch;
  p.rows = rows;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = group;
  p.rows_div = divisor(static_cast<uint32_t>(rows));
  p.group_div = divisor(static_cast<uint32_t>(group));
  p.own_div = divisor(static_cast<uint32_t>(rows) * group);
  p.stacked_div = divisor(static_cast<uint32_t>(stacked));
  p.causal = causal ? 1 : 0;
  p.joint = s.joint;
  if (whole_form(width, kv_heads, batch, s.warp)) {
    p.whole = p.joint = 1;
    s.tensor.shared_tiles = s.warp.shared_tiles = 0;
  }
  p.shared_keys = p.joint ? 0 : shared_rows;
  p.pool_pages = pool_pages;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.key_pool = key_pool;
  p.value_pool = value_pool;
  p.tensor = s.tensor;
  p.warp = s.warp;
  p.shared_slot_rows = s.shared_slot_rows;
  p.own_slot_rows = s.own_slot_rows;
  p.own_row0 = s.own_row0;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(static_cast<float*>(workspace) + s.rows * kD);
  p.plan = reinterpret_cast<int*>(p.part_ml + s.rows);
  p.err = device_error;
  const cudaStream_t s0 = static_cast<cudaStream_t>(stream);
  if (nodes) {
    p.masks = nodes->masks;
    p.counts = nodes->counts;
    p.words = (rows + 31) / 32;
    p.compact = p.shared_keys > 0 && batch <= kMaxStack ? 1 : 0;
    return e4m3 ? launch<true, TreeParams>(p, s0) : launch<false, TreeParams>(p, s0);
  }
  return e4m3 ? launch<true, BranchParams>(p, s0) : launch<false, BranchParams>(p, s0);
}

}  // namespace
}  // namespace h3sa

using namespace h3sa;

extern "C" {

int64_t h3sa_shared_prefix_workspace(int32_t batch, int32_t rows, int32_t heads, int32_t kv_heads,
                                     int32_t shared_rows) {
  if (batch <= 0 || rows <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || shared_rows < 0)
    return 0;
  const Shape s = shape_of(batch, rows, kv_heads, heads / kv_heads, shared_rows / kBlk);
  return s.bytes;
}

int64_t h3sa_tree_workspace(int32_t batch, int32_t rows, int32_t heads, int32_t kv_heads, int32_t shared_rows,
                            int32_t width, int32_t e4m3) {
  if (batch <= 0 || rows <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || shared_rows < 0 || width <= 0 ||
      shared_rows / kBlk > width || static_cast<int64_t>(rows) * (heads / kv_heads) > INT32_MAX / 2)
    return 0;
  const Shape s = shape_of(batch, rows, kv_heads, heads / kv_heads, shared_rows / kBlk, width, e4m3 != 0);
  return s.bytes;
}

int h3sa_shared_prefix_attention(const void* query, int64_t stride_sequence, int64_t stride_row,
                                 int64_t stride_head, void* out, float* lse, int32_t batch,
                                 int32_t rows, int32_t heads, int32_t kv_heads,
                                 const void* key_pool, const void* value_pool, int32_t pool_pages,
                                 int32_t e4m3, const float* k_scale, const float* v_scale,
                                 const int32_t* table, int32_t width, const int32_t* lengths,
                                 int32_t shared_rows, int32_t causal, float softmax_scale,
                                 void* workspace, int64_t workspace_bytes, int32_t* device_error,
                                 void* stream) {
  return attend("shared prefix attention", nullptr, query, stride_sequence, stride_row, stride_head, out, lse, batch, rows,
                heads, kv_heads, key_pool, value_pool, pool_pages, e4m3, k_scale, v_scale, table, width, lengths,
                shared_rows, causal, softmax_scale, workspace, workspace_bytes, device_error, stream);
}

int h3sa_tree_attention(const void* query, int64_t stride_sequence, int64_t stride_row, int64_t stride_head, void* out,
                        float* lse, int32_t batch, int32_t rows, int32_t heads, int32_t kv_heads, const void* key_pool,
                        const void* value_pool, int32_t pool_pages, int32_t e4m3, const float* k_scale,
                        const float* v_scale, const int32_t* table, int32_t width, const int32_t* lengths,
                        const int32_t* masks, const int32_t* counts, int32_t shared_rows, float softmax_scale,
                        void* workspace, int64_t workspace_bytes, int32_t* device_error, void* stream) {
  TreeParams nodes;
  memset(&nodes, 0, sizeof(nodes));
  nodes.masks = reinterpret_cast<const uint32_t*>(masks);
  nodes.counts = counts;
  return attend("tree attention", &nodes, query, stride_sequence, stride_row, stride_head, out, lse, batch, rows, heads,
                kv_heads, key_pool, value_pool, pool_pages, e4m3, k_scale, v_scale, table, width, lengths, shared_rows, 0,
                softmax_scale, workspace, workspace_bytes, device_error, stream);
}

}  // extern "C"
