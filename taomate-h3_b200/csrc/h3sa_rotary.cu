// Rotary positions: rows of heads rotated by themselves, or on their way into a paged cache.
//
// Pair k of a head at position p turns by the angle a = p * f_k:
//
//   (x, y) -> (x cos a - y sin a, x sin a + y cos a) * factor
//
// Pairs are (k, k + pairs) in the half layout and (2k, 2k + 1) interleaved; dimensions behind the last
// pair stay as they are. Positions may have several axes (time, height, width); pair k then belongs to
// axis k / per_axis. Angles are taken in whole turns: of f_k / 2 pi only the fraction of a turn matters, as an integer in
// units of 2^-64 off by half of one, and p times that, cut to 64 bits, is the angle: positions of 32 bits leave it
// exact to 2^-33 of a turn, of which the upper 32 bits are used. Positions between whole numbers take a product of
// doubles instead, off by 2^-52 of itself. Cosine and sine of it are in 32 bits, as are the products, and each result is
// rounded once.
//
// Bound by memory: a value is read and written once. What has to be kept small is the instructions in
// between, for which an SM has some 350 a warp and 2 KB: a thread keeps to one unit of a head row, 8 pairs in two
// vectors of 16 bytes, with their frequencies in registers, works out its 8 angles once a task and turns up to six heads by
// them (appends four, tensors of up to two heads two), all of which are on their way by then. There is nothing to share and
// nothing to wait for in a block.
// Measured: 24605 tokens of 24 heads, bf16, three axes: 48 to 50 us, 6.05 TB/s and more of the 302 MB read and written; 7 prompts of up
// to 3001 rows, 32 / 8 heads, into bf16 pools 66 us of 61 to 63 at the copy rate, into e4m3 pools 69 to 75 us of 57, 5.0 TB/s,
// the divisions and conversions beside the loads; a few rows 2.7 us in a row of launches, 4.2 with the start of a graph.
// 300001 tokens of one head take 42.5 us of 23.6: 8 angles are worked out for 16 values, and the 64 registers of eight blocks an
// SM, which keep enough rows on their way, spill 84 to 120 bytes. (A table of the block's cosines and sines in shared memory took
// 57 and 110.) Appends keep 96 registers and spill up to 80 bytes, most in the half layout into e4m3 pools.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>
#include <type_traits>

#include "h3sa_div.cuh"
#include "h3sa_fp8.cuh"
#include "h3sa_host.h"
#include "h3sa_ptx.cuh"

namespace h3sa {
namespace {

constexpr int kPage = 128;
constexpr int kDim = 128;  // head dimension of a cache
constexpr int kThreads = 128;
constexpr int kMaxDim = 1024;
constexpr int kSms = 148;

enum PositionKind : int { kPosNone = 0, kPosI32 = 1, kPosI64 = 2, kPosF64 = 3 };

struct Angles {
  const void* positions;  // [tokens, axes], or null: row of the sequence
  const double* frequencies;
  int kind, axes, per_axis, pairs;
  float factor;
};

struct Heads {  // [batch, rows, heads, dim] by element strides; the last one is 1
  const void* src;
  void* dst;
  long long sb, sn, db, dn;
  int sh, dh;
  int heads;
};

// Rows of one tensor that go to one place: rotated to a tensor (the rows of h3sa_rotate, the queries of
// h3sa_append_rows), or to a pool, keys rotated and values as they are.
struct Part {
  Heads h;
  void* pool;          // [heads, pool_pages * 128, 128], or null
  const float* scale;  // of e4m3 pools
  // a head row's units: its pairs', then its other dimensions'
  int pair_units, units;
  int tasks, slots;    // tasks of a token: up to kBatch head rows each; slots: tasks that a block's threads cover
  Divisor task_div;
  long long all;       // tasks
  int blocks;
};

struct RowsParams {
  Angles at;
  long long tokens;  // batch * rows, below 2^31
  int rows, dim;
  Divisor row_div;
  Part part[3];  // x, keys, values
  int pool_pages, width;
  const int* table;
  const int* lengths;
  const int* counts;  // or null: all rows
  int* err;
};

// f / 2 pi as a fraction of a turn in units of 2^-64. Whole turns a position do not matter, and p times this, cut to
// 64 bits, is the fraction of p f / 2 pi, off by p 2^-65 (the quotient is taken in two terms). Numbers are brought
// into an integer by adding 1.5 * 2^k, which leaves them in the sum's last bits: conversions of 64 bits are slow.
__device__ __forceinline__ uint64_t turn_of(double f) {
  const double hi = f * 0.15915494309189535;  // 1 / (2 pi), less 9.8e-18
  const double lo = fma(f, 0.15915494309189535, -hi) + f * -9.839338337591243e-18;
  const double r = hi - ((hi + 6755399441055744.0) - 6755399441055744.0);  // 1.5 * 2^52
  const double t = r + lo, off = (r - t) + lo;  // of a large f, lo too has bits in front of 2^-32
  const double top = t + 1572864.0;             // 1.5 * 2^20: last bit 2^-32
  const double rest = t - (top - 1572864.0) + off;
  // 1.5 * 2^-12: last bit 2^-64. As a difference of all 64 bits: where top was a tie, rest may be 2^-33 and have 33 bits.
  const long long low = __double_as_longlong(rest + 0.0003662109375) - __double_as_longlong(0.0003662109375);
  return (static_cast<uint64_t>(static_cast<uint32_t>(__double2loint(top))) << 32) + static_cast<uint64_t>(low);
}
// What a pair needs of its frequency: turn_of it, or for positions between whole numbers the bits of f / 2 pi.
__device__ __forceinline__ uint64_t frequency_word(const Angles& a, int pair) {
  const double f = __ldg(a.frequencies + pair);
  return a.kind == kPosF64 ? static_cast<uint64_t>(__double_as_longlong(f * 0.15915494309189535)) : turn_of(f);
}
// A token's position on one axis, as 64 bits.
__device__ __forceinline__ uint64_t position_word(const Angles& a, long long token, int axis) {
  const long long at = token * a.axes + axis;
  if (a.kind == kPosI32) return static_cast<uint64_t>(static_cast<long long>(__ldg(static_cast<const int*>(a.positions) + at)));
  return __ldg(static_cast<const unsigned long long*>(a.positions) + at);
}
// The fraction of a turn, in [-1/2, 1/2), in units of 2^-32.
__device__ __forceinline__ int fraction(bool between, uint64_t position, uint64_t frequency) {
  if (!between) return static_cast<int>(static_cast<uint32_t>((position * frequency) >> 32));
  // in 64-bit arithmetic, whole turns taken off by one rounding
  const double p = __longlong_as_double(static_cast<long long>(position));
  const double unit = __longlong_as_double(static_cast<long long>(frequency)), t = p * unit;
  const double whole = (t + 6755399441055744.0) - 6755399441055744.0;
  return __double2loint(fma(p, unit, -whole) + 1572864.0);
}
// Cosine and sine of a fraction of a turn. For 16-bit values the approximate functions, which with the roundings of the angle
// are off by under 2^-20: 2^-9 of what rounding a value of 1 to fp16 leaves. For 32 bits the fraction's first 24 bits, which
// a float holds, by the function, and the other 8, an angle below 2^-21, by the first term of the sums' formulas: all 32 in
// one float are off by up to 2^-26 of a turn, more than the results' own rounding (rotations at positions to 2^31 off by
// 4.5e-8 of their length, with one float 5.7e-8; with cosines and sines taken in 64 bits 4.2e-8. 300001 tokens of one head
// 64.6 us, with one float 62.6, others the same).
template <typename T>
__device__ __forceinline__ void cos_sin(int fraction, float factor, float& c, float& s) {
  if constexpr (sizeof(T) == 2) {
    const float a = static_cast<float>(fraction) * 2.3283064365386963e-10f * 6.2831853071795865f;  // 2^-32
    s = __sinf(a);
    c = __cosf(a);
  } else {
    const float rest = static_cast<float>(fraction & 0xff) * 1.4629180792671596e-9f;  // 2 pi 2^-32
    float c0, s0;
    sincospif(static_cast<float>(fraction & ~0xff) * 4.6566128730773926e-10f, &s0, &c0);  // 2^-31
    c = fmaf(-s0, rest, c0);
    s = fmaf(c0, rest, s0);
  }
  c *= factor;
  s *= factor;
}

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float(float x) { return x; }
template <> __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float(float x) { return x; }
template <> __device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }

template <typename T, int kN>
struct alignas(sizeof(T) * kN) Vec {
  T v[kN];
};
template <typename T, int kN>
__device__ __forceinline__ Vec<T, kN> load(const T* p) {
  return *reinterpret_cast<const Vec<T, kN>*>(p);
}
// A vector of kN values in 32 bits, two a register pair (a single one in the first half).
template <typename T, int kN>
struct Values {
  uint64_t v[(kN + 1) / 2];
};
template <typename T, int kN>
__device__ __forceinline__ Values<T, kN> widen(const Vec<T, kN>& x) {
  Values<T, kN> r;
  if constexpr (std::is_same_v<T, __nv_bfloat16> && kN >= 2) {
    const uint32_t* const w = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
    for (int j = 0; j < kN / 2; ++j)
      r.v[j] = f2_pack(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
  } else {
#pragma unroll
    for (int j = 0; j < kN; j += 2) r.v[j / 2] = f2_pack(to_float(x.v[j]), kN > 1 ? to_float(x.v[j + 1]) : 0.f);
  }
  return r;
}
template <typename T, int kN>
__device__ __forceinline__ void store_values(T* p, const Values<T, kN>& x) {
  Vec<T, kN> v;
  if constexpr (std::is_same_v<T, __nv_bfloat16> && kN >= 2) {
    uint32_t* const w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int j = 0; j < kN / 2; ++j) {
      float lo, hi;
      f2_unpack(x.v[j], lo, hi);
      w[j] = pack_bf16x2(lo, hi);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kN; j += 2) {
      float lo, hi;
      f2_unpack(x.v[j / 2], lo, hi);
      v.v[j] = from_float<T>(lo);
      if (kN > 1) v.v[j + 1] = from_float<T>(hi);
    }
  }
  *reinterpret_cast<Vec<T, kN>*>(p) = v;
}

// x / scale, rounded once, from inverse = 1 / scale: two corrections of the quotient (see h3sa_fp8.cuh); one that is
// past the numbers or not a number needs none.
__device__ __forceinline__ float quotient_of(float x, float scale, float inverse) {
  const float q0 = x * inverse;
  return fabsf(q0) < INFINITY ? div_by_scale(x, scale, inverse) : q0;
}
// Two values divided by their head's scale as e4m3: largest numbers for what is past them and for infinities,
// NaN for NaN.
__device__ __forceinline__ uint32_t e4m3_pair(float x, float y) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(y), "f"(x));
  return r;
}
template <typename T, int kN>
__device__ __forceinline__ void store_e4m3(uint8_t* dst, const Values<T, kN>& v, float scale) {
  const float inverse = 1.0f / scale;
  float x[kN + kN % 2];
#pragma unroll
  for (int j = 0; j < kN; j += 2) f2_unpack(v.v[j / 2], x[j], x[j + 1]);
  if (scale > 1e-30f && scale < 1e30f) {
#pragma unroll
    for (int j = 0; j < kN; ++j) x[j] = quotient_of(x[j], scale, inverse);
  } else {  // whose inverse or residues would leave the normal numbers
#pragma unroll
    for (int j = 0; j < kN; ++j) x[j] = __fdiv_rn(x[j], scale);
  }
  if constexpr (kN >= 4) {
    uint32_t w[kN / 4];
#pragma unroll
    for (int j = 0; j < kN; j += 4) w[j / 4] = e4m3_pair(x[j], x[j + 1]) | (e4m3_pair(x[j + 2], x[j + 3]) << 16);
    if constexpr (kN == 4) *reinterpret_cast<uint32_t*>(dst) = w[0];
    else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  } else {
    *dst = static_cast<uint8_t>(e4m3_pair(x[0], 0.f));
  }
}

// Cosines and sines of a unit's kN pairs, in the order of its values: two pairs a register pair, or (interleaved) each
// pair's twice.
template <int kN, bool kInterleaved>
struct Turn {
  static constexpr int kWords = kInterleaved ? kN : (kN + 1) / 2;
  uint64_t c[kWords], s[kWords];
};
template <typename T, int kN, bool kInterleaved>
__device__ __forceinline__ void make_turn(Turn<kN, kInterleaved>& t, bool between, uint64_t position, const uint64_t (&frequency)[kN],
                                          float factor) {
  float c[kN + kN % 2], s[kN + kN % 2];
  c[kN - 1 + kN % 2] = s[kN - 1 + kN % 2] = 0.f;
#pragma unroll
  for (int j = 0; j < kN; ++j) cos_sin<T>(fraction(between, position, frequency[j]), factor, c[j], s[j]);
  if constexpr (kInterleaved && kN > 1) {
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      t.c[j] = f2_pack(c[j], c[j]);
      t.s[j] = f2_pack(-s[j], s[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kN; j += 2) {
      t.c[j / 2] = f2_pack(c[j], c[j + 1]);
      t.s[j / 2] = f2_pack(s[j], s[j + 1]);
    }
  }
}
// (x, y) -> (x c - y s, x s + y c). y0 are the values at the pairs' first columns, y1 at the second ones; interleaved
// the pairs themselves, one after the other.
template <typename T, int kN, bool kInterleaved>
__device__ __forceinline__ void turn(Values<T, kN>& y0, Values<T, kN>& y1, const Turn<kN, kInterleaved>& t) {
  if constexpr (kInterleaved && kN > 1) {
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      uint64_t& y = j < kN / 2 ? y0.v[j] : y1.v[j - kN / 2];
      float a, b;
      f2_unpack(y, a, b);
      y = f2_fma(f2_pack(b, a), t.s[j], f2_mul(y, t.c[j]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < (kN + 1) / 2; ++j) {
      const uint64_t x = y0.v[j], y = y1.v[j], minus = f2_pack(-1.f, -1.f);
      y0.v[j] = f2_fma(f2_mul(y, t.s[j]), minus, f2_mul(x, t.c[j]));
      y1.v[j] = f2_fma(x, t.s[j], f2_mul(y, t.c[j]));
    }
  }
}

// A block's share of one part. A task is up to kBatch head rows of a token, `tasks` apart; a thread has one unit of each,
// kN pairs or 2 kN other dimensions (two vectors, or one at an odd end), and takes every `stride`-th task.
constexpr int kFew = 2, kMany = 6, kAppended = 4;  // kBatch
enum Kind : int { kRotated = 0, kQueries = 1, kKeys = 2, kValues = 3 };
template <typename T, int kN, bool kInterleaved, bool kFp8, int kKind, int kBatch>
__device__ __forceinline__ void rows_block(const RowsParams& p, const Part& q, uint32_t block) {
  constexpr bool kPaged = kKind != kRotated, kPool = kKind >= kKeys, kTurns = kKind != kValues;
  const int pairs = kTurns ? p.at.pairs : 0;
  const int slot = q.units <= kThreads ? static_cast<int>(threadIdx.x) / q.units : 0;
  if (slot >= q.slots) return;
  const bool between = p.at.kind == kPosF64;
  const uint32_t stride = static_cast<uint32_t>(q.blocks) * q.slots;
  for (int unit = static_cast<int>(threadIdx.x) - slot * q.units; unit < q.units; unit += kThreads) {
    const bool turns = kTurns && unit < q.pair_units;
    const int pair = unit * kN;
    const int c0 = turns ? (kInterleaved ? 2 * pair : pair) : 2 * pairs + (unit - q.pair_units) * 2 * kN;
    const int c1 = turns && !kInterleaved ? c0 + pairs : c0 + kN;
    const bool two = kPaged || c1 < p.dim;
    const int axis = turns ? pair / p.at.per_axis : 0;  // of all its pairs
    uint64_t frequency[kN];
    if (turns) {
#pragma unroll
      for (int j = 0; j < kN; ++j) frequency[j] = frequency_word(p.at, pair + j);
    }
    for (uint32_t task = block * q.slots + slot; task < q.all; task += stride) {
      const uint32_t token = quotient(task, q.task_div);
      const int h0 = static_cast<int>(task - token * q.tasks);
      const long long b = quotient(token, p.row_div), i = token - b * p.rows;
      const bool live = !kPaged || !p.counts || i < __ldg(p.counts + b);
      if (kPool && !live) continue;
      Vec<T, kN> va[kBatch], vb[kBatch];
      if (live) {
        const T* const src = static_cast<const T*>(q.h.src) + b * q.h.sb + i * q.h.sn;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int h = h0 + j * q.tasks;
          if (h < q.h.heads) {
            const T* const row = src + static_cast<long long>(h) * q.h.sh;
            va[j] = load<T, kN>(row + c0);
            if (two) vb[j] = load<T, kN>(row + c1);
          }
        }
      }
      long long place = 0;  // the row of the pool
      if constexpr (kPool) {
        const int length = __ldg(p.lengths + b);
        const long long row = length + i;
        const bool inside = length >= 0 && row < static_cast<long long>(p.width) * kPage;
        const int page = inside ? __ldg(p.table + b * p.width + row / kPage) : 0;
        if (!inside || page < 0 || page >= p.pool_pages) {
          if (p.err && unit == 0 && h0 == 0) atomicOr(p.err, inside ? kErrBadPage : kErrBadIndex);
          continue;
        }
        place = (static_cast<long long>(page) * kPage + row % kPage) * kDim;
      }
      T* const out = kPool ? nullptr : static_cast<T*>(q.h.dst) + b * q.h.db + i * q.h.dn;
      if (!live) {  // queries behind a count
        for (int h = h0; h < q.h.heads; h += q.tasks) {
          store_values(out + static_cast<long long>(h) * q.h.dh + c0, Values<T, kN>{});
          store_values(out + static_cast<long long>(h) * q.h.dh + c1, Values<T, kN>{});
        }
        continue;
      }
      Turn<kN, kInterleaved> cs;
      if (turns) {
        const uint64_t where = kPaged && p.at.kind == kPosNone
                                   ? static_cast<uint64_t>(static_cast<long long>(__ldg(p.lengths + b)) + i)
                                   : position_word(p.at, token, axis);
        make_turn<T>(cs, between, where, frequency, p.at.factor);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int h = h0 + j * q.tasks;
        if (h < q.h.heads) {
          Values<T, kN> y0 = widen(va[j]), y1 = widen(vb[j]);
          if (turns) turn(y0, y1, cs);
          if constexpr (!kPool) {
            T* const dst = out + static_cast<long long>(h) * q.h.dh;
            store_values(dst + c0, y0);
            if (two) store_values(dst + c1, y1);
          } else {
            const long long to = static_cast<long long>(h) * p.pool_pages * (kPage * kDim) + place;
            if constexpr (kFp8) {
              const float scale = __ldg(q.scale + h);
              store_e4m3(static_cast<uint8_t*>(q.pool) + to + c0, y0, scale);
              store_e4m3(static_cast<uint8_t*>(q.pool) + to + c1, y1, scale);
            } else {
              store_values(static_cast<T*>(q.pool) + to + c0, y0);
              store_values(static_cast<T*>(q.pool) + to + c1, y1);
            }
          }
        }
      }
    }
  }
}

template <typename T, int kN, bool kInterleaved, int kBatch>
__global__ void __launch_bounds__(kThreads, kBatch == kFew ? 8 : kN == 8 ? 4 : 5) rotate_kernel(const __grid_constant__ RowsParams p) {
  rows_block<T, kN, kInterleaved, false, kRotated, kBatch>(p, p.part[0], blockIdx.x);
}

// Queries, keys and values have blocks of their own, in this order.
template <int kN, bool kInterleaved, bool kFp8>
__global__ void __launch_bounds__(kThreads, 5) append_rows_kernel(const __grid_constant__ RowsParams p) {
  using T = __nv_bfloat16;
  uint32_t block = blockIdx.x;
  if (block < p.part[0].blocks) {
    rows_block<T, kN, kInterleaved, kFp8, kQueries, kAppended>(p, p.part[0], block);
  } else if ((block -= p.part[0].blocks) < p.part[1].blocks) {
    rows_block<T, kN, kInterleaved, kFp8, kKeys, kAppended>(p, p.part[1], block);
  } else {
    rows_block<T, kN, kInterleaved, kFp8, kValues, kAppended>(p, p.part[2], block - p.part[1].blocks);
  }
}

template <typename T, int kN, int kBatch>
int launch_rotate(const RowsParams& p, bool interleaved, cudaStream_t stream) {
  const auto kernel = interleaved ? rotate_kernel<T, kN, true, kBatch> : rotate_kernel<T, kN, false, kBatch>;
  kernel<<<p.part[0].blocks, kThreads, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? H3SA_OK : set_cuda_error("rotate_kernel launch", e);
}
template <typename T>
int launch_rotate(const RowsParams& p, int n, bool few, bool interleaved, cudaStream_t stream) {
  constexpr int kWide = 16 / sizeof(T);
  if (n == kWide)
    return few ? launch_rotate<T, kWide, kFew>(p, interleaved, stream) : launch_rotate<T, kWide, kMany>(p, interleaved, stream);
  if (n == 4) return few ? launch_rotate<T, 4, kFew>(p, interleaved, stream) : launch_rotate<T, 4, kMany>(p, interleaved, stream);
  return few ? launch_rotate<T, 1, kFew>(p, interleaved, stream) : launch_rotate<T, 1, kMany>(p, interleaved, stream);
}
template <bool kFp8>
int launch_append(const RowsParams& p, int n, bool interleaved, cudaStream_t stream) {
  const auto kernel = n == 8   ? (interleaved ? append_rows_kernel<8, true, kFp8> : append_rows_kernel<8, false, kFp8>)
                      : n == 4 ? (interleaved ? append_rows_kernel<4, true, kFp8> : append_rows_kernel<4, false, kFp8>)
                               : (interleaved ? append_rows_kernel<1, true, kFp8> : append_rows_kernel<1, false, kFp8>);
  unsigned blocks = 0;
  for (const Part& q : p.part) blocks += static_cast<unsigned>(q.blocks);
  kernel<<<blocks, kThreads, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? H3SA_OK : set_cuda_error("append_rows_kernel launch", e);
}

// The values of a vector: 16 bytes where columns, strides and addresses allow it, 8, or single values.
bool fits(const Heads& h, int size, int n) {
  const long long bytes = static_cast<long long>(size) * n;
  const auto ok = [&](const void* base, long long sb, long long sn, long long sh) {
    return reinterpret_cast<uintptr_t>(base) % bytes == 0 && sb % n == 0 && sn % n == 0 && sh % n == 0;
  };
  return h.heads == 0 || (ok(h.src, h.sb, h.sn, h.sh) && (!h.dst || ok(h.dst, h.db, h.dn, h.dh)));
}
int vector_of(const RowsParams& p, int size) {
  for (int n = 16 / size; n >= 4; n /= 2)
    if (p.at.per_axis % n == 0 && p.at.pairs % n == 0 && p.dim % n == 0 && fits(p.part[0].h, size, n) &&
        fits(p.part[1].h, size, n) && fits(p.part[2].h, size, n))
      return n;
  return 1;
}

// A task is a head row while threads are few, `most_rows` of them from there on, of which a thread takes up to four, or two
// where most_rows is kMany (whose tasks pay for a thread's frequencies sooner). Two / four, us: 24605 tokens of 24 heads 50.1 /
// 51.3, 30000 of 16 in fp32 78.5 / 83.9, 60000 of 8 heads of 64 26.8 / 26.3; but one head of 300001 49.5 / 44.9, e4m3 prompts
// 74.9 / 74.3.
void lay_out(RowsParams& p, int n, int batch, int most_rows) {
  p.tokens = static_cast<long long>(batch) * p.rows;
  p.row_div = divisor(static_cast<uint32_t>(p.rows));
  long long threads = 0;
  for (Part& q : p.part) {
    const int pairs = &q == p.part + 2 ? 0 : p.at.pairs;
    q.pair_units = pairs / n;
    q.units = q.pair_units + (p.dim - 2 * pairs + 2 * n - 1) / (2 * n);
    threads += p.tokens * q.h.heads * q.units;
  }
  const int rows = threads >= 768ll * kSms * most_rows ? most_rows : 1;
  for (Part& q : p.part) {
    if (q.h.heads == 0) continue;
    q.tasks = (q.h.heads + rows - 1) / rows;
    q.slots = q.units <= kThreads ? kThreads / q.units : 1;
    q.task_div = divisor(static_cast<uint32_t>(q.tasks));
    q.all = p.tokens * q.tasks;
    const long long once = (q.all + q.slots - 1) / q.slots, some = 8 * kSms;
    const int each = most_rows == kMany ? 2 : 4;
    q.blocks = static_cast<int>(once <= some ? once : once <= each * some ? some : (once + each - 1) / each);
  }
}

int check_rotary(const char* what, const h3sa_rotary* r, int dim, bool rows_known, Angles& a) {
  memset(&a, 0, sizeof(a));
  a.axes = 1;
  if (!r || r->pairs == 0) return H3SA_OK;
  if (r->pairs < 0 || r->pairs > dim / 2 || r->axes <= 0 || r->pairs % r->axes)
    return set_error(H3SA_ERR_INVALID, "%s: %d pairs over %d axes do not fit a head of %d", what, r->pairs, r->axes, dim);
  if (r->position_kind < 0 || r->position_kind > kPosF64 || (r->position_kind == kPosNone && (!rows_known || r->axes != 1)))
    return set_error(H3SA_ERR_INVALID, "%s: positions must be int32, int64 or float64", what);
  if (!r->frequencies || (r->position_kind != kPosNone && !r->positions))
    return set_error(H3SA_ERR_INVALID, "%s: null pointer argument", what);
  if (!(r->factor >= -3.0e38f && r->factor <= 3.0e38f))
    return set_error(H3SA_ERR_INVALID, "%s: the factor must be finite", what);
  a.positions = r->positions;
  a.frequencies = r->frequencies;
  a.kind = r->position_kind;
  a.axes = r->axes;
  a.pairs = r->pairs;
  a.per_axis = r->pairs / r->axes;
  a.factor = r->factor;
  return H3SA_OK;
}

// Strides of heads are kept in 32 bits.
bool head_stride_ok(const h3sa_heads* h) { return !h || (h->stride_head >= INT32_MIN && h->stride_head <= INT32_MAX); }

// Rows that are written lie apart: those of a tensor that repeats some by a stride of zero, or by one axis' steps into
// another's, would be written from several places, and read and written at once in place. Every axis steps over all that
// the ones of smaller steps reach, as the axes of any slice or transposed view do.
bool rows_apart(const h3sa_heads* h, int batch, int rows, int dim) {
  struct Axis {
    long long n;
    unsigned long long step;
  };
  const auto axis = [](long long n, int64_t stride) {
    return Axis{n, n < 2 ? 0 : stride < 0 ? 0ull - static_cast<uint64_t>(stride) : static_cast<uint64_t>(stride)};
  };
  Axis axes[3] = {axis(batch, h->stride_sequence), axis(rows, h->stride_row), axis(h->heads, h->stride_head)};
  std::sort(axes, axes + 3, [](const Axis& a, const Axis& b) { return a.step < b.step; });
  unsigned __int128 reach = static_cast<unsigned>(dim);
  for (const Axis& a : axes) {
    if (a.n < 2) continue;
    if (a.step < reach) return false;
    reach += static_cast<unsigned __int128>(a.n - 1) * a.step;
  }
  return true;
}

Heads heads_of(const h3sa_heads* from, const h3sa_heads* to) {
  Heads h;
  memset(&h, 0, sizeof(h));
  if (!from) return h;
  h.src = from->base;
  h.sb = from->stride_sequence;
  h.sn = from->stride_row;
  h.sh = static_cast<int>(from->stride_head);
  h.heads = from->heads;
  if (to) {
    h.dst = to->base;
    h.db = to->stride_sequence;
    h.dn = to->stride_row;
    h.dh = static_cast<int>(to->stride_head);
  }
  return h;
}

}  // namespace
}  // namespace h3sa

using namespace h3sa;

extern "C" {

int h3sa_rotate(const h3sa_heads* x, const h3sa_heads* out, int32_t dtype, int32_t batch, int32_t rows, int32_t dim,
                const h3sa_rotary* rotary, void* stream) {
  if (!x || !out || batch < 0 || rows < 0 || x->heads < 0 || x->heads != out->heads || dim <= 0 || dim > kMaxDim)
    return set_error(H3SA_ERR_INVALID, "rotate: invalid sizes batch=%d rows=%d heads=%d dim=%d (at most %d)", batch, rows,
                     x ? x->heads : 0, dim, kMaxDim);
  if (dtype < H3SA_BF16 || dtype > H3SA_FP32) return set_error(H3SA_ERR_UNSUPPORTED, "rotate: unknown type %d", dtype);
  RowsParams p;
  memset(&p, 0, sizeof(p));
  if (batch == 0 || rows == 0 || x->heads == 0) return H3SA_OK;
  if (const int rc = check_rotary("rotate", rotary, dim, false, p.at)) return rc;
  if (static_cast<int64_t>(batch) * rows > INT32_MAX / 2 || static_cast<int64_t>(batch) * rows * x->heads > INT32_MAX / 2)
    return set_error(H3SA_ERR_UNSUPPORTED, "rotate: batch %d x rows %d x heads %d is too large", batch, rows, x->heads);
  if (!head_stride_ok(x) || !head_stride_ok(out))
    return set_error(H3SA_ERR_UNSUPPORTED, "rotate: strides of heads must fit 32 bits");
  if (!rows_apart(out, batch, rows, dim)) return set_error(H3SA_ERR_INVALID, "rotate: rows of out overlap");
  const int size = dtype == H3SA_FP32 ? 4 : 2;
  if (!x->base || !out->base) return set_error(H3SA_ERR_INVALID, "rotate: null pointer argument");
  if ((reinterpret_cast<uintptr_t>(x->base) | reinterpret_cast<uintptr_t>(out->base)) % size)
    return set_error(H3SA_ERR_INVALID, "rotate: tensors must be aligned to their type");
  p.part[0].h = heads_of(x, out);
  p.rows = rows;
  p.dim = dim;
  const int n = vector_of(p, size);
  const bool few = x->heads <= kFew;
  lay_out(p, n, batch, few ? kFew : kMany);
  const bool inter = rotary && rotary->interleaved;
  const cudaStream_t at = static_cast<cudaStream_t>(stream);
  return dtype == H3SA_FP32   ? launch_rotate<float>(p, n, few, inter, at)
         : dtype == H3SA_FP16 ? launch_rotate<__half>(p, n, few, inter, at)
                              : launch_rotate<__nv_bfloat16>(p, n, few, inter, at);
}

int h3sa_append_rows(const h3sa_heads* key, const h3sa_heads* value, const h3sa_heads* query, const h3sa_heads* query_out,
                     int32_t batch, int32_t rows, void* key_pool, void* value_pool, int32_t pool_pages, int32_t e4m3,
                     const float* k_scale, const float* v_scale, const int32_t* table, int32_t width,
                     const int32_t* lengths, const int32_t* counts, const h3sa_rotary* rotary, int32_t* device_error,
                     void* stream) {
  if (!key || !value || batch < 0 || rows < 0 || key->heads <= 0 || value->heads != key->heads ||
      (query && (query->heads < 0 || !query_out || query_out->heads != query->heads)))
    return set_error(H3SA_ERR_INVALID, "append rows: invalid sizes batch=%d rows=%d kv_heads=%d", batch, rows,
                     key ? key->heads : 0);
  RowsParams p;
  memset(&p, 0, sizeof(p));
  if (batch == 0 || rows == 0) return H3SA_OK;
  if (const int rc = check_rotary("append rows", rotary, kDim, true, p.at)) return rc;
  if (pool_pages <= 0 || width <= 0 || static_cast<int64_t>(pool_pages) * kPage > INT32_MAX ||
      static_cast<int64_t>(width) * kPage > INT32_MAX)
    return set_error(H3SA_ERR_INVALID, "append rows: invalid pool of %d pages or table of %d entries a sequence",
                     pool_pages, width);
  const bool with_query = query && query->heads > 0;
  const int64_t heads = 2ll * key->heads + (with_query ? query->heads : 0);
  if (static_cast<int64_t>(batch) * rows > INT32_MAX / 2 || static_cast<int64_t>(batch) * rows * heads > INT32_MAX / 2)
    return set_error(H3SA_ERR_UNSUPPORTED, "append rows: batch %d x rows %d x heads %lld is too large", batch, rows,
                     static_cast<long long>(heads));
  if (!head_stride_ok(key) || !head_stride_ok(value) || !head_stride_ok(query) || !head_stride_ok(query_out))
    return set_error(H3SA_ERR_UNSUPPORTED, "append rows: strides of heads must fit 32 bits");
  if (with_query && !rows_apart(query_out, batch, rows, kDim))
    return set_error(H3SA_ERR_INVALID, "append rows: rows of query_out overlap");
  if (!key->base || !value->base || !key_pool || !value_pool || !table || !lengths ||
      (with_query && (!query->base || !query_out->base)) || (e4m3 && (!k_scale || !v_scale)))
    return set_error(H3SA_ERR_INVALID, "append rows: null pointer argument");
  if ((reinterpret_cast<uintptr_t>(key_pool) | reinterpret_cast<uintptr_t>(value_pool)) & 15u)
    return set_error(H3SA_ERR_INVALID, "append rows: pools must be 16-byte aligned");
  Part &x = p.part[0], &k = p.part[1], &v = p.part[2];
  x.h = heads_of(with_query ? query : nullptr, query_out);
  k.h = heads_of(key, nullptr);
  v.h = heads_of(value, nullptr);
  const uintptr_t odd = reinterpret_cast<uintptr_t>(x.h.src) | reinterpret_cast<uintptr_t>(x.h.dst) |
                        reinterpret_cast<uintptr_t>(k.h.src) | reinterpret_cast<uintptr_t>(v.h.src);
  if (odd & 1u) return set_error(H3SA_ERR_INVALID, "append rows: tensors must be aligned to their type");
  p.rows = rows;
  p.dim = kDim;
  k.pool = key_pool;
  k.scale = k_scale;
  v.pool = value_pool;
  v.scale = v_scale;
  p.pool_pages = pool_pages;
  p.width = width;
  p.table = table;
  p.lengths = lengths;
  p.counts = counts;
  p.err = device_error;
  const int n = vector_of(p, 2);
  lay_out(p, n, batch, kAppended);
  const bool inter = rotary && rotary->interleaved;
  const cudaStream_t at = static_cast<cudaStream_t>(stream);
  return e4m3 ? launch_append<true>(p, n, inter, at) : launch_append<false>(p, n, inter, at);
}

}  // extern "C"
