// Rotary positions: rows of heads rotated by themselves, or on their way into a paged cache.
//
// Pair k of a head at position p turns by the angle a = p * f_k:
//
//   (x, y) -> (x cos a - y sin a, x sin a + y cos a) * factor
//
// Pairs are (k, k + pairs) in the half layout and (2k, 2k + 1) interleaved; dimensions behind the last
// pair stay as they are. Positions may have several axes (time, height, width); pair k then belongs to
// axis k / per_axis. Angles are taken in whole turns: t = p * (f_k / 2 pi) in 64 bits, whose fraction is
// then exact to 2^-25 of a turn for any position of 32 bits; cosine and sine of it are in 32 bits, as are
// the products, and each result is rounded once.
//
// Both kernels are bound by memory: a value is read and written once, 6 flops stand against 8 bytes. All
// heads of a token share its angles, so a block takes a few tokens, writes their cosines and
// sines to shared memory once (some 60 instructions each) and then streams the heads past them, two
// vectors of 16 bytes a thread and step.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstring>
#include <type_traits>

#include "h3sa_fp8.cuh"
#include "h3sa_host.h"
#include "h3sa_ptx.cuh"

namespace h3sa {
namespace {

constexpr int kPage = 128;
constexpr int kDim = 128;  // head dimension of a cache
constexpr int kThreads = 256;
constexpr int kMaxDim = 1024;

// x / d for x below 2^31 by one multiplication: m = ceil(2^(32 + s) / d) with 2^s >= d (Granlund and
// Montgomery's division by invariant integers; m needs 33 bits, of which the first is a plain add).
struct Divisor {
  uint32_t d, m, s;
};
Divisor divisor(uint32_t d) {
  Divisor v;
  v.d = d;
  v.s = 0;
  while ((1ull << v.s) < d) ++v.s;
  v.m = static_cast<uint32_t>(((((1ull << v.s) - d) << 32) / d) + 1);
  return v;
}
__device__ __forceinline__ uint32_t quotient(uint32_t x, const Divisor& v) {
  const uint32_t hi = __umulhi(x, v.m);
  return (hi + x) >> v.s;  // x below 2^31: the sum stays below 2^32
}

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
  int group;           // tokens of a block
  // a head row's units: its pairs', then its other dimensions'
  int pair_units, units;
  int tasks, slots;    // tasks of a token: up to kBatch head rows each; slots: tasks that a block's threads cover
  Divisor task_div;
  int blocks;
};

struct RowsParams {
  Angles at;
  long long tokens;  // batch * rows, below 2^31
  int rows, dim;
  Divisor row_div, pair_div, axis_div;
  Part part[3];  // x, keys, values
  int pool_pages, width;
  const int* table;
  const int* lengths;
  const int* counts;  // or null: all rows
  int* err;
};

// A token's row of the pool, as an element offset: kNoRow behind a sequence's count, kNoPlace for one that the table
// has no page for.
constexpr long long kNoRow = -1, kNoPlace = -2;

__device__ __forceinline__ double position(const Angles& a, long long token, int axis) {
  const long long i = token * a.axes + axis;
  if (a.kind == kPosI32) return static_cast<double>(__ldg(static_cast<const int*>(a.positions) + i));
  if (a.kind == kPosI64) return static_cast<double>(__ldg(static_cast<const long long*>(a.positions) + i));
  return __ldg(static_cast<const double*>(a.positions) + i);
}

__device__ __forceinline__ float2 cos_sin(double p, double frequency, float factor) {
  const double turn = frequency * 0.15915494309189535;
  const double t = p * turn;
  // the fraction by one rounding: whole turns are exact in 64 bits
  const float f = static_cast<float>(fma(p, turn, -rint(t)));
  float s, c;
  sincospif(2.0f * f, &s, &c);
  return make_float2(c * factor, s * factor);
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
template <int kN, bool kInterleaved>
__device__ __forceinline__ void load_turn(Turn<kN, kInterleaved>& t, const float* cosines, const float* sines) {
  float c[kN], s[kN];
  if constexpr (kN >= 4) {
#pragma unroll
    for (int j = 0; j < kN; j += 4) {
      const float4 x = *reinterpret_cast<const float4*>(cosines + j);
      const float4 y = *reinterpret_cast<const float4*>(sines + j);
      c[j] = x.x, c[j + 1] = x.y, c[j + 2] = x.z, c[j + 3] = x.w;
      s[j] = y.x, s[j + 1] = y.y, s[j + 2] = y.z, s[j + 3] = y.w;
    }
  } else {
    c[0] = cosines[0];
    s[0] = sines[0];
  }
  if constexpr (kInterleaved && kN > 1) {
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      t.c[j] = f2_pack(c[j], c[j]);
      t.s[j] = f2_pack(-s[j], s[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kN; j += 2) {
      t.c[j / 2] = f2_pack(c[j], kN > 1 ? c[j + 1] : 0.f);
      t.s[j / 2] = f2_pack(s[j], kN > 1 ? s[j + 1] : 0.f);
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

// A block's tokens in one part. A task is up to kBatch head rows of a token, `tasks` apart; a thread has one unit of each,
// kN pairs or 2 kN other dimensions (two vectors, or one at an odd end), so it reads its cosines and sines once, and
// has all rows on their way before it needs the first; those of its first task before the block works out its angles
// and places.
constexpr int kBatch = 4;
enum Kind : int { kRotated = 0, kQueries = 1, kKeys = 2, kValues = 3 };
template <typename T, int kN, bool kInterleaved, bool kFp8, int kKind>
__device__ __forceinline__ void rows_block(const RowsParams& p, const Part& q, uint32_t block, float4* smem) {
  constexpr bool kPaged = kKind != kRotated, kPool = kKind >= kKeys, kTurns = kKind != kValues;
  const int pairs = kTurns ? p.at.pairs : 0;
  const uint32_t first = block * static_cast<uint32_t>(q.group);
  const int n_tokens = static_cast<int>(min(static_cast<uint32_t>(q.group), static_cast<uint32_t>(p.tokens) - first));
  float* const cs_all = reinterpret_cast<float*>(smem);                                  // [group][2][pairs]
  long long* const places = reinterpret_cast<long long*>(cs_all + q.group * 2 * pairs);  // [group]
  const int slot = q.units <= kThreads ? static_cast<int>(threadIdx.x) / q.units : 0;
  const int all = slot < q.slots ? n_tokens * q.tasks : 0, unit0 = static_cast<int>(threadIdx.x) - slot * q.units;
  bool turns, two;  // of a unit, and its columns
  int pair, c0, c1;
  const auto take_unit = [&](int unit) {
    turns = kTurns && unit < q.pair_units;
    pair = unit * kN;
    c0 = turns ? (kInterleaved ? 2 * pair : pair) : 2 * pairs + (unit - q.pair_units) * 2 * kN;
    c1 = turns && !kInterleaved ? c0 + pairs : c0 + kN;
    two = kPaged || c1 < p.dim;
  };
  Vec<T, kN> va[kBatch], vb[kBatch];
  // Loads of a task's rows, if they are not behind their sequence's count.
  const auto fetch = [&](int task) {
    const int t = static_cast<int>(quotient(static_cast<uint32_t>(task), q.task_div)), h0 = task - t * q.tasks;
    const long long b = quotient(first + t, p.row_div), i = first + t - b * p.rows;
    if (kPaged && p.counts && i >= __ldg(p.counts + b)) return;
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
  };
  take_unit(unit0);
  if (slot < all) fetch(slot);
  if constexpr (kPaged) {  // by the last warps, the first ones have angles
    for (int t = kThreads - 1 - static_cast<int>(threadIdx.x); t < n_tokens; t += kThreads) {
      const long long b = quotient(first + t, p.row_div), i = first + t - b * p.rows;
      long long place = kNoRow;
      if (!p.counts || i < __ldg(p.counts + b)) {
        place = kNoPlace;
        if constexpr (kPool) {
          const int length = __ldg(p.lengths + b);
          const long long row = length + i;
          if (length < 0 || row >= static_cast<long long>(p.width) * kPage) {
            if (p.err) atomicOr(p.err, kErrBadIndex);
          } else {
            const int page = __ldg(p.table + b * p.width + row / kPage);
            if (page >= 0 && page < p.pool_pages) place = (static_cast<long long>(page) * kPage + row % kPage) * kDim;
            else if (p.err) atomicOr(p.err, kErrBadPage);
          }
        }
      }
      places[t] = place;
    }
  }
  for (int k = threadIdx.x; k < n_tokens * pairs; k += kThreads) {
    const int t = quotient(k, p.pair_div), at = k - t * pairs;
    double where;
    if (kPaged && p.at.kind == kPosNone) {
      const uint32_t b = quotient(first + t, p.row_div);
      where = static_cast<double>(__ldg(p.lengths + b)) + (first + t - b * p.rows);
    } else {
      where = position(p.at, first + t, quotient(at, p.axis_div));
    }
    const float2 v = cos_sin(where, __ldg(p.at.frequencies + at), p.at.factor);
    cs_all[t * 2 * pairs + at] = v.x;
    cs_all[t * 2 * pairs + pairs + at] = v.y;
  }
  __syncthreads();
  const int unit_step = q.units <= kThreads ? q.units : kThreads;
  for (int unit = unit0; unit < q.units; unit += unit_step) {
    for (int task = slot; task < all; task += q.slots) {
      if (unit != unit0 || task != slot) {
        take_unit(unit);
        fetch(task);
      }
      const int t = static_cast<int>(quotient(static_cast<uint32_t>(task), q.task_div)), h0 = task - t * q.tasks;
      const long long place = kPaged ? places[t] : kNoPlace;
      if (kPool && place < 0) continue;
      T* out = nullptr;
      if constexpr (!kPool) {
        const long long b = quotient(first + t, p.row_div), i = first + t - b * p.rows;
        out = static_cast<T*>(q.h.dst) + b * q.h.db + i * q.h.dn;
      }
      if (kPaged && place == kNoRow) {
        for (int h = h0; h < q.h.heads; h += q.tasks) {
          store_values(out + static_cast<long long>(h) * q.h.dh + c0, Values<T, kN>{});
          store_values(out + static_cast<long long>(h) * q.h.dh + c1, Values<T, kN>{});
        }
        continue;
      }
      Turn<kN, kInterleaved> cs;
      if (turns) load_turn(cs, cs_all + t * 2 * pairs + pair, cs_all + t * 2 * pairs + pairs + pair);
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

template <typename T, int kN, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, kN == 8 ? 3 : 4) rotate_kernel(const __grid_constant__ RowsParams p) {
  extern __shared__ float4 smem[];
  rows_block<T, kN, kInterleaved, false, kRotated>(p, p.part[0], blockIdx.x, smem);
}

// Queries, keys and values have blocks of their own, in this order.
template <int kN, bool kInterleaved, bool kFp8>
__global__ void __launch_bounds__(kThreads, 3) append_rows_kernel(const __grid_constant__ RowsParams p) {
  using T = __nv_bfloat16;
  extern __shared__ float4 smem[];
  uint32_t block = blockIdx.x;
  if (block < p.part[0].blocks) {
    rows_block<T, kN, kInterleaved, kFp8, kQueries>(p, p.part[0], block, smem);
  } else if ((block -= p.part[0].blocks) < p.part[1].blocks) {
    rows_block<T, kN, kInterleaved, kFp8, kKeys>(p, p.part[1], block, smem);
  } else {
    rows_block<T, kN, kInterleaved, kFp8, kValues>(p, p.part[2], block - p.part[1].blocks, smem);
  }
}

size_t token_bytes(const Angles& a) { return 8 * static_cast<size_t>(a.pairs) + sizeof(long long); }

template <typename T>
int launch_rotate(const RowsParams& p, int n, bool interleaved, cudaStream_t stream) {
  const auto kernel = n == 8   ? (interleaved ? rotate_kernel<T, sizeof(T) == 2 ? 8 : 4, true> : rotate_kernel<T, sizeof(T) == 2 ? 8 : 4, false>)
                      : n == 4 ? (interleaved ? rotate_kernel<T, 4, true> : rotate_kernel<T, 4, false>)
                               : (interleaved ? rotate_kernel<T, 1, true> : rotate_kernel<T, 1, false>);
  kernel<<<p.part[0].blocks, kThreads, token_bytes(p.at) * p.part[0].group, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? H3SA_OK : set_cuda_error("rotate_kernel launch", e);
}
template <bool kFp8>
int launch_append(const RowsParams& p, int n, bool interleaved, cudaStream_t stream) {
  const auto kernel = n == 8   ? (interleaved ? append_rows_kernel<8, true, kFp8> : append_rows_kernel<8, false, kFp8>)
                      : n == 4 ? (interleaved ? append_rows_kernel<4, true, kFp8> : append_rows_kernel<4, false, kFp8>)
                               : (interleaved ? append_rows_kernel<1, true, kFp8> : append_rows_kernel<1, false, kFp8>);
  size_t group = 0;
  unsigned blocks = 0;
  for (const Part& q : p.part) {
    if (q.blocks > 0 && static_cast<size_t>(q.group) > group) group = q.group;
    blocks += static_cast<unsigned>(q.blocks);
  }
  kernel<<<blocks, kThreads, token_bytes(p.at) * group, stream>>>(p);
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
    if (p.at.pairs % n == 0 && p.dim % n == 0 && fits(p.part[0].h, size, n) && fits(p.part[1].h, size, n) &&
        fits(p.part[2].h, size, n))
      return n;
  return 1;
}

constexpr int kSms = 148;

// A task is a head row while threads are few, kBatch of them from there on; a block has as many tokens as give
// its threads a task each, as far as that leaves every SM some blocks.
void lay_out(RowsParams& p, int n, int batch) {
  p.tokens = static_cast<long long>(batch) * p.rows;
  p.row_div = divisor(static_cast<uint32_t>(p.rows));
  p.pair_div = divisor(static_cast<uint32_t>(p.at.pairs > 0 ? p.at.pairs : 1));
  p.axis_div = divisor(static_cast<uint32_t>(p.at.per_axis > 0 ? p.at.per_axis : 1));
  long long threads = 0;
  for (Part& q : p.part) {
    const int pairs = &q == p.part + 2 ? 0 : p.at.pairs;
    q.pair_units = pairs / n;
    q.units = q.pair_units + (p.dim - 2 * pairs + 2 * n - 1) / (2 * n);
    threads += p.tokens * q.h.heads * q.units;
  }
  const int rows = threads >= static_cast<long long>(kSms) * kThreads * 3 * kBatch ? kBatch : 1;
  for (Part& q : p.part) {
    if (q.h.heads == 0) continue;
    q.tasks = (q.h.heads + rows - 1) / rows;
    q.slots = q.units <= kThreads ? kThreads / q.units : 1;
    q.task_div = divisor(static_cast<uint32_t>(q.tasks));
    long long group = q.slots / q.tasks;
    const long long most = p.tokens / (4 * kSms), room = static_cast<long long>(32768 / token_bytes(p.at));
    if (group > most) group = most;
    if (group > room) group = room;
    q.group = group < 1 ? 1 : static_cast<int>(group);
    q.blocks = static_cast<int>((p.tokens + q.group - 1) / q.group);
  }
}

int check_rotary(const char* what, const h3sa_rotary* r, int dim, bool rows_known, Angles& a) {
  memset(&a, 0, sizeof(a));
  a.axes = a.per_axis = 1;
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
  if (static_cast<int64_t>(batch) * rows > INT32_MAX / 2 || static_cast<int64_t>(x->heads) * dim > INT32_MAX / 4096)
    return set_error(H3SA_ERR_UNSUPPORTED, "rotate: batch %d x rows %d x heads %d is too large", batch, rows, x->heads);
  if (!head_stride_ok(x) || !head_stride_ok(out))
    return set_error(H3SA_ERR_UNSUPPORTED, "rotate: strides of heads must fit 32 bits");
  const int size = dtype == H3SA_FP32 ? 4 : 2;
  if (!x->base || !out->base) return set_error(H3SA_ERR_INVALID, "rotate: null pointer argument");
  if ((reinterpret_cast<uintptr_t>(x->base) | reinterpret_cast<uintptr_t>(out->base)) % size)
    return set_error(H3SA_ERR_INVALID, "rotate: tensors must be aligned to their type");
  p.part[0].h = heads_of(x, out);
  p.rows = rows;
  p.dim = dim;
  const int n = vector_of(p, size);
  lay_out(p, n, batch);
  const bool inter = rotary && rotary->interleaved;
  const cudaStream_t at = static_cast<cudaStream_t>(stream);
  return dtype == H3SA_FP32   ? launch_rotate<float>(p, n, inter, at)
         : dtype == H3SA_FP16 ? launch_rotate<__half>(p, n, inter, at)
                              : launch_rotate<__nv_bfloat16>(p, n, inter, at);
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
  if (static_cast<int64_t>(batch) * rows > INT32_MAX / 2 || heads > INT32_MAX / (4096 * kDim))
    return set_error(H3SA_ERR_UNSUPPORTED, "append rows: batch %d x rows %d x heads %lld is too large", batch, rows,
                     static_cast<long long>(heads));
  if (!head_stride_ok(key) || !head_stride_ok(value) || !head_stride_ok(query) || !head_stride_ok(query_out))
    return set_error(H3SA_ERR_UNSUPPORTED, "append rows: strides of heads must fit 32 bits");
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
  lay_out(p, n, batch);
  const bool inter = rotary && rotary->interleaved;
  const cudaStream_t at = static_cast<cudaStream_t>(stream);
  return e4m3 ? launch_append<true>(p, n, inter, at) : launch_append<false>(p, n, inter, at);
}

}  // extern "C"
