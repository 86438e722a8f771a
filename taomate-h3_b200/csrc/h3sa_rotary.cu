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
  long long sb, sn, sh, db, dn, dh;
  int heads;
};

struct RowsParams {
  Angles at;
  Heads x;             // rotated to a tensor: the rows of h3sa_rotate, the queries of h3sa_append_rows
  long long tokens;    // batch * rows
  int rows, dim, group;  // group: tokens of a block
  Divisor row_div;
  // units of work of a token's x, k and v; a head's units are its pairs' and then its other dimensions'
  int pair_units, head_units, x_units, k_units, units;
  Divisor unit_div, head_div, value_div;
  // ---- the cache
  Heads k, v;
  void* key_pool;
  void* value_pool;
  int pool_pages, width;
  const int* table;
  const int* lengths;
  const int* counts;  // or null: all rows
  const float* k_scale;
  const float* v_scale;
  int* err;
};

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
template <typename T, int kN>
__device__ __forceinline__ void store(T* p, const Vec<T, kN>& v) {
  *reinterpret_cast<Vec<T, kN>*>(p) = v;
}

// Two values divided by their head's scale as e4m3: largest numbers for what is past them and for infinities,
// NaN for NaN.
__device__ __forceinline__ uint32_t e4m3_pair(float x, float y, float scale) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(__fdiv_rn(y, scale)), "f"(__fdiv_rn(x, scale)));
  return r;
}
template <int kN>
__device__ __forceinline__ void store_e4m3(uint8_t* dst, const float (&x)[kN], float scale) {
  if constexpr (kN >= 4) {
    uint32_t w[kN / 4];
#pragma unroll
    for (int j = 0; j < kN; j += 4)
      w[j / 4] = e4m3_pair(x[j], x[j + 1], scale) | (e4m3_pair(x[j + 2], x[j + 3], scale) << 16);
    if constexpr (kN == 4) *reinterpret_cast<uint32_t*>(dst) = w[0];
    else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  } else {
    *dst = static_cast<uint8_t>(e4m3_pair(x[0], 0.f, scale));
  }
}

// A thread's unit of one token: kN pairs (two vectors), or kN other dimensions (one vector); of values,
// 2 kN dimensions (two vectors).
template <typename T, int kN, bool kInterleaved>
struct Unit {
  Vec<T, kN> a, b;
  int c0, c1;  // their columns; c1 < 0: there is no second one
  int pair;    // first pair, or -1
};

template <typename T, int kN, bool kInterleaved>
__device__ __forceinline__ void locate(Unit<T, kN, kInterleaved>& u, int at, int pair_units, int pairs) {
  if (at < pair_units) {
    u.pair = at * kN;
    u.c0 = kInterleaved ? 2 * u.pair : u.pair;
    u.c1 = kInterleaved ? u.c0 + kN : u.c0 + pairs;
  } else {
    u.pair = -1;
    u.c0 = 2 * pairs + (at - pair_units) * kN;
    u.c1 = -1;
  }
}

// The unit's values in 32 bits, turned: y0 at c0, y1 at c1. cs: cosines of the token, then its sines.
template <typename T, int kN, bool kInterleaved>
__device__ __forceinline__ void turn(const Unit<T, kN, kInterleaved>& u, const float* cs, int pairs, float (&y0)[kN],
                                     float (&y1)[kN]) {
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    y0[j] = to_float(u.a.v[j]);
    y1[j] = to_float(u.b.v[j]);
  }
  if (u.pair < 0) return;
  float c[kN], s[kN];
  if constexpr (kN >= 4) {
#pragma unroll
    for (int j = 0; j < kN; j += 4) {
      const float4 x = *reinterpret_cast<const float4*>(cs + u.pair + j);
      const float4 y = *reinterpret_cast<const float4*>(cs + pairs + u.pair + j);
      c[j] = x.x, c[j + 1] = x.y, c[j + 2] = x.z, c[j + 3] = x.w;
      s[j] = y.x, s[j + 1] = y.y, s[j + 2] = y.z, s[j + 3] = y.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      c[j] = cs[u.pair + j];
      s[j] = cs[pairs + u.pair + j];
    }
  }
  if constexpr (kInterleaved && kN > 1) {  // pair j is (2j, 2j + 1) of the two vectors one after the other
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float(&y)[kN] = h ? y1 : y0;
#pragma unroll
      for (int j = 0; j < kN; j += 2) {
        const int k = (h * kN + j) / 2;
        const float p = y[j], q = y[j + 1];
        y[j] = p * c[k] - q * s[k];
        y[j + 1] = p * s[k] + q * c[k];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      const float p = y0[j], q = y1[j];
      y0[j] = p * c[j] - q * s[j];
      y1[j] = p * s[j] + q * c[j];
    }
  }
}

// kPaged: keys and values go to the pools too, keys rotated, as bf16 or (kFp8) divided by their head's
// scale as e4m3. kN: values of a vector.
template <typename T, int kN, bool kInterleaved, bool kPaged, bool kFp8>
__global__ void __launch_bounds__(kThreads) rotate_rows_kernel(const RowsParams p) {
  extern __shared__ float4 smem[];
  float* const cs_all = reinterpret_cast<float*>(smem);  // [group][2][pairs]
  __shared__ long long dst_rows[kPaged ? kThreads : 1];  // of a token: its row of the pool, -1 for none
  const int pairs = p.at.pairs;
  const long long first = static_cast<long long>(blockIdx.x) * p.group;
  const int n_tokens = static_cast<int>(min(static_cast<long long>(p.group), p.tokens - first));
  // a token of a sequence: (b, i); tokens stay below 2^31
  const auto split = [&](long long token, int& b, int& i) {
    b = static_cast<int>(quotient(static_cast<uint32_t>(token), p.row_div));
    i = static_cast<int>(token) - b * p.rows;
  };
  for (int k = threadIdx.x; k < n_tokens * pairs; k += kThreads) {
    const int t = k / pairs, pair = k - t * pairs;
    double where;
    if (kPaged && p.at.kind == kPosNone) {
      int b, i;
      split(first + t, b, i);
      where = static_cast<double>(__ldg(p.lengths + b)) + i;
    } else {
      where = position(p.at, first + t, pair / p.at.per_axis);
    }
    const float2 v = cos_sin(where, __ldg(p.at.frequencies + pair), p.at.factor);
    cs_all[t * 2 * pairs + pair] = v.x;
    cs_all[t * 2 * pairs + pairs + pair] = v.y;
  }
  if constexpr (kPaged) {
    for (int t = threadIdx.x; t < n_tokens; t += kThreads) {
      int b, i;
      split(first + t, b, i);
      long long row = -1;
      if (!p.counts || i < __ldg(p.counts + b)) {
        const int len = __ldg(p.lengths + b);
        const long long at = static_cast<long long>(len) + i;
        if (len < 0 || at >= static_cast<long long>(p.width) * kPage) {
          if (p.err) atomicOr(p.err, kErrBadIndex);
        } else {
          const int page = __ldg(p.table + static_cast<size_t>(b) * p.width + at / kPage);
          if (page >= 0 && page < p.pool_pages) row = static_cast<long long>(page) * kPage + at % kPage;
          else if (p.err) atomicOr(p.err, kErrBadPage);
        }
        if (row < 0) row = -2;  // a row that has no place, but is one
      }
      dst_rows[t] = row;
    }
  }
  __syncthreads();
  const uint32_t all = static_cast<uint32_t>(n_tokens) * static_cast<uint32_t>(p.units);
  for (uint32_t n = threadIdx.x; n < all; n += kThreads) {
    const int t = static_cast<int>(quotient(n, p.unit_div));
    int at = static_cast<int>(n) - t * p.units;
    int b, i;
    split(first + t, b, i);
    const float* const cs = cs_all + t * 2 * pairs;
    Unit<T, kN, kInterleaved> u;
    float y0[kN], y1[kN];
    const bool is_x = !kPaged || at < p.x_units;
    const bool is_k = kPaged && !is_x && at < p.x_units + p.k_units;
    const Heads& h = is_x ? p.x : is_k ? p.k : p.v;
    int head;
    if (!kPaged || is_x || is_k) {
      if (is_k) at -= p.x_units;
      head = static_cast<int>(quotient(at, p.head_div));
      locate(u, at - head * p.head_units, p.pair_units, pairs);
    } else {
      at -= p.x_units + p.k_units;
      head = static_cast<int>(quotient(at, p.value_div));
      u.pair = -1;
      u.c0 = (at - head * static_cast<int>(p.value_div.d)) * 2 * kN;
      u.c1 = u.c0 + kN;
    }
    const long long row = kPaged ? dst_rows[t] : 0;
    const bool live = row != -1;  // rows of x behind a sequence's count come out zero
    if (kPaged && !is_x && row < 0) continue;
    const T* const src = static_cast<const T*>(h.src) + b * h.sb + i * h.sn + head * h.sh;
    if (live) {
      u.a = load<T, kN>(src + u.c0);
      if (u.c1 >= 0) u.b = load<T, kN>(src + u.c1);
    } else {
      memset(&u.a, 0, sizeof(u.a));
    }
    if (u.c1 < 0 || !live) memset(&u.b, 0, sizeof(u.b));
    turn(u, cs, pairs, y0, y1);
    if (!live) {  // whatever the position was
#pragma unroll
      for (int j = 0; j < kN; ++j) y0[j] = y1[j] = 0.f;
    }
    if (kFp8 && !is_x) {
      const float scale = __ldg((is_k ? p.k_scale : p.v_scale) + head);
      uint8_t* const dst = static_cast<uint8_t*>(is_k ? p.key_pool : p.value_pool) +
                           (static_cast<long long>(head) * p.pool_pages * kPage + row) * kDim;
      store_e4m3<kN>(dst + u.c0, y0, scale);
      if (u.c1 >= 0) store_e4m3<kN>(dst + u.c1, y1, scale);
      continue;
    }
    T* const dst = is_x ? static_cast<T*>(h.dst) + b * h.db + i * h.dn + head * h.dh
                        : static_cast<T*>(is_k ? p.key_pool : p.value_pool) +
                              (static_cast<long long>(head) * p.pool_pages * kPage + row) * kDim;
    Vec<T, kN> r;
#pragma unroll
    for (int j = 0; j < kN; ++j) r.v[j] = from_float<T>(y0[j]);
    store(dst + u.c0, r);
    if (u.c1 >= 0) {
#pragma unroll
      for (int j = 0; j < kN; ++j) r.v[j] = from_float<T>(y1[j]);
      store(dst + u.c1, r);
    }
  }
}

template <typename T, int kN, bool kInterleaved, bool kPaged, bool kFp8>
int launch(const RowsParams& p, cudaStream_t stream) {
  const long long blocks = (p.tokens + p.group - 1) / p.group;
  rotate_rows_kernel<T, kN, kInterleaved, kPaged, kFp8>
      <<<static_cast<unsigned>(blocks), kThreads, static_cast<size_t>(p.group) * 8 * p.at.pairs, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? H3SA_OK : set_cuda_error("rotate_rows_kernel launch", e);
}
template <typename T, int kN, bool kPaged, bool kFp8>
int launch(const RowsParams& p, bool interleaved, cudaStream_t stream) {
  return interleaved ? launch<T, kN, true, kPaged, kFp8>(p, stream) : launch<T, kN, false, kPaged, kFp8>(p, stream);
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
    if (p.at.pairs % n == 0 && p.dim % n == 0 && fits(p.x, size, n) && fits(p.k, size, n) && fits(p.v, size, n)) return n;
  return 1;
}

// Blocks of a few tokens: enough units that a thread has four, as far as that leaves every SM some blocks.
void lay_out(RowsParams& p, int n, int batch) {
  p.tokens = static_cast<long long>(batch) * p.rows;
  p.pair_units = p.at.pairs / n;
  p.head_units = p.pair_units + (p.dim - 2 * p.at.pairs) / n;
  p.x_units = p.x.heads * p.head_units;
  p.k_units = p.k.heads * p.head_units;
  const int value_units = kDim / (2 * n);
  p.units = p.x_units + p.k_units + p.v.heads * value_units;
  p.row_div = divisor(static_cast<uint32_t>(p.rows));
  p.unit_div = divisor(static_cast<uint32_t>(p.units));
  p.head_div = divisor(static_cast<uint32_t>(p.head_units));
  p.value_div = divisor(static_cast<uint32_t>(value_units));
  constexpr int kSms = 148;
  int group = 4 * kThreads / p.units;
  if (p.at.pairs > 0 && group > 32768 / (8 * p.at.pairs)) group = 32768 / (8 * p.at.pairs);
  if (group > kThreads) group = kThreads;
  const long long most = p.tokens / (4 * kSms);
  if (group > most) group = static_cast<int>(most);
  p.group = group < 1 ? 1 : group;
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

Heads heads_of(const h3sa_heads* from, const h3sa_heads* to) {
  Heads h;
  memset(&h, 0, sizeof(h));
  if (!from) return h;
  h.src = from->base;
  h.sb = from->stride_sequence;
  h.sn = from->stride_row;
  h.sh = from->stride_head;
  h.heads = from->heads;
  if (to) {
    h.dst = to->base;
    h.db = to->stride_sequence;
    h.dn = to->stride_row;
    h.dh = to->stride_head;
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
  const int size = dtype == H3SA_FP32 ? 4 : 2;
  if (!x->base || !out->base) return set_error(H3SA_ERR_INVALID, "rotate: null pointer argument");
  if ((reinterpret_cast<uintptr_t>(x->base) | reinterpret_cast<uintptr_t>(out->base)) % size)
    return set_error(H3SA_ERR_INVALID, "rotate: tensors must be aligned to their type");
  p.x = heads_of(x, out);
  p.rows = rows;
  p.dim = dim;
  const int n = vector_of(p, size);
  lay_out(p, n, batch);
  const bool inter = rotary && rotary->interleaved;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == H3SA_FP32)
    return n == 4 ? launch<float, 4, false, false>(p, inter, s) : launch<float, 1, false, false>(p, inter, s);
  if (dtype == H3SA_FP16)
    return n == 8   ? launch<__half, 8, false, false>(p, inter, s)
           : n == 4 ? launch<__half, 4, false, false>(p, inter, s)
                    : launch<__half, 1, false, false>(p, inter, s);
  return n == 8   ? launch<__nv_bfloat16, 8, false, false>(p, inter, s)
         : n == 4 ? launch<__nv_bfloat16, 4, false, false>(p, inter, s)
                  : launch<__nv_bfloat16, 1, false, false>(p, inter, s);
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
  if (!key->base || !value->base || !key_pool || !value_pool || !table || !lengths ||
      (with_query && (!query->base || !query_out->base)) || (e4m3 && (!k_scale || !v_scale)))
    return set_error(H3SA_ERR_INVALID, "append rows: null pointer argument");
  if ((reinterpret_cast<uintptr_t>(key_pool) | reinterpret_cast<uintptr_t>(value_pool)) & 15u)
    return set_error(H3SA_ERR_INVALID, "append rows: pools must be 16-byte aligned");
  p.x = heads_of(with_query ? query : nullptr, query_out);
  p.k = heads_of(key, nullptr);
  p.v = heads_of(value, nullptr);
  const uintptr_t odd = reinterpret_cast<uintptr_t>(p.x.src) | reinterpret_cast<uintptr_t>(p.x.dst) |
                        reinterpret_cast<uintptr_t>(p.k.src) | reinterpret_cast<uintptr_t>(p.v.src);
  if (odd & 1u) return set_error(H3SA_ERR_INVALID, "append rows: tensors must be aligned to their type");
  p.rows = rows;
  p.dim = kDim;
  p.key_pool = key_pool;
  p.value_pool = value_pool;
  p.pool_pages = pool_pages;
  p.width = width;
  p.table = table;
  p.lengths = lengths;
  p.counts = counts;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.err = device_error;
  const int n = vector_of(p, 2);
  lay_out(p, n, batch);
  const bool inter = rotary && rotary->interleaved;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (e4m3)
    return n == 8   ? launch<__nv_bfloat16, 8, true, true>(p, inter, s)
           : n == 4 ? launch<__nv_bfloat16, 4, true, true>(p, inter, s)
                    : launch<__nv_bfloat16, 1, true, true>(p, inter, s);
  return n == 8   ? launch<__nv_bfloat16, 8, true, false>(p, inter, s)
         : n == 4 ? launch<__nv_bfloat16, 4, true, false>(p, inter, s)
                  : launch<__nv_bfloat16, 1, true, false>(p, inter, s);
}

}  // extern "C"
