// Branch attention for few query rows: the items of the warp line (h3sa_branch.cuh), up to 16 rows
// each against the shared blocks or a branch's own.
//
//   x_j = scale * q . k_j,   O = sum_j 2^(x_j' - m) v_j,   l = sum_j 2^(x_j' - m),   x' = x log2 e
//
// Sixteen rows use a key 2 * 16 * 2 * 128 flops for its 512 bytes: the kernel is bound by reading K
// and V, and for a branch's own few blocks by latency. So a warp works alone: it takes 32 keys at a
// time straight from global memory into registers in the order the tensor instruction wants them,
// with the next 32 keys of K (then of V) in flight, and passes no barrier and no shared memory
// but its own query's.
//
// mma.m16n8k16 leaves the order of the contracted index open as long as both operands agree, and so
// the column order of the result:
//   S = Q K^T: lane 4r + c holds key r of each group of eight and contracts d = 32c + 4s .. + 3 in step
//      s, a quarter of the key's row that it reads in one piece.
//   O += P V: lane 4r + c holds keys 2c, 2c + 1, 2c + 8, 2c + 9 of sixteen and the columns 16r .. + 15 of
//      each, so a row's 256 (128) bytes are read by eight lanes side by side; two keys' words are
//      woven into the operand's pairs by byte permutes. Lane 4r + c ends up with columns 32c ..
//      32c + 31 of rows r and r + 8.
// e4m3 caches become f16 pairs, exactly, on the way; the query row is scaled by a power of two and
// taken as f16 (11 bits to bf16's 8), and P is f16 too.
#include <cstring>

#include "h3sa_branch.cuh"

namespace h3sa {
namespace {

constexpr int kRowWarps = 8;
// P is at most 2^threshold; f16 and bf16 both hold it, and O is rescaled only past it.
constexpr float kThreshold = 8.0f;

// 32 bytes of read-once data.
__device__ __forceinline__ void load32(const void* at, uint32_t* r) {
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(at));
}
__device__ __forceinline__ void load16(const void* at, uint32_t* r) {
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "l"(at));
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

template <bool kFp8>
__global__ void __launch_bounds__(32 * kRowWarps, 1) branch_rows_kernel(const BranchParams p, const bool after) {
  constexpr int kElem = kFp8 ? 1 : 2;
  constexpr int kRowBytes = kD * kElem;
  constexpr int kKWords = kRowBytes / 16;  // a lane's quarter of a key row
  constexpr int kVWords = kRowBytes / 32;  // a lane's sixteen columns of a value row
  __shared__ uint4 q_frag[kRowWarps][8][32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const Line& ln = p.warp;
  const int worker = blockIdx.x * kRowWarps + warp;
  const Plan pl = make_plan(p, ln, lane);
  const int all = pl.head_weight * p.kv_heads;
  int u = min(all, worker * pl.cut);
  const int u_end = min(all, u + pl.cut);
  Place at = {0, -1, 0, 0};
  if (u < u_end) at = locate(p, ln, pl, u, lane);
  while (u < u_end) {
    const int units = place_units(p, ln, pl, at), part = min(weight_of(ln, units) - at.off, u_end - u);
    const int n_units = min(units, at.off + part) - at.off;
    if (n_units > 0) {
      // ---- a segment: rows row0 .. of KV head `head` against keys [key0, key0 + 32 n_units)
      const int head = at.head, seq = at.b < 0 ? pl.longest : at.b;
      const int own_all = p.rows * p.group;
      const int row0 = (at.b < 0 ? 0 : at.b * own_all) + at.t * kRowSpan;
      const int n_rows = min(kRowSpan, (at.b < 0 ? p.batch * own_all : (at.b + 1) * own_all) - row0);
      const int key0 = (at.b < 0 ? 0 : own_lo(p)) + at.off * kRowUnit;
      const int kv_end = at.b < 0 ? pl.max_len : seq_length(p, at.b);
      const bool direct = pl.shared_blocks == 0 && n_units == units;
      // this lane's rows, r and r + 8 of the item
      const RowAt at0 = row_at(p, head, row0 + min(r, n_rows - 1)), at1 = row_at(p, head, row0 + min(r + 8, n_rows - 1));
      const int hide0 = p.causal ? p.rows - 1 - at0.i : 0, hide1 = p.causal ? p.rows - 1 - at1.i : 0;
      const int lim0 = seq_length(p, at0.b) - hide0, lim1 = seq_length(p, at1.b) - hide1;
      float sl2 = p.scale_log2, sl2b = p.scale_log2;  // of row r and row r + 8
      if constexpr (kFp8) sl2 = sl2b = p.scale_log2 * __ldg(p.k_scale + head);
      {
        uint32_t a[16], b[16];
        const __nv_bfloat16* qa = p.q + at0.b * p.q_sb + at0.i * p.q_sn + at0.h * p.q_sh + 32 * c;
        const __nv_bfloat16* qb = p.q + at1.b * p.q_sb + at1.i * p.q_sn + at1.h * p.q_sh + 32 * c;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          load16(qa + 8 * k, a + 4 * k);
          load16(qb + 8 * k, b + 4 * k);
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          if (r >= n_rows) a[k] = 0u;
          if (r + 8 >= n_rows) b[k] = 0u;
        }
        if constexpr (kFp8) {
          uint32_t ta = 0u, tb = 0u;
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            ta = __vmaxu2(ta, a[k] & 0x7fff7fffu);
            tb = __vmaxu2(tb, b[k] & 0x7fff7fffu);
          }
          ta = max(ta >> 16, ta & 0xffffu);
          tb = max(tb >> 16, tb & 0xffffu);
          for (int d = 1; d < 4; d <<= 1) {
            ta = max(ta, __shfl_xor_sync(0xffffffffu, ta, d));
            tb = max(tb, __shfl_xor_sync(0xffffffffu, tb, d));
          }
          const int ka = row_exponent(ta), kb = row_exponent(tb);
          const float ua = exp2_int(ka), ub = exp2_int(kb);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            a[k] = f16x2_of(__uint_as_float(a[k] << 16) * ua, __uint_as_float(a[k] & 0xffff0000u) * ua);
            b[k] = f16x2_of(__uint_as_float(b[k] << 16) * ub, __uint_as_float(b[k] & 0xffff0000u) * ub);
          }
          // infinities and NaN stay what they are in f16
          sl2 *= exp2_int(-ka);
          sl2b *= exp2_int(-kb);
        }
        __syncwarp();
#pragma unroll
        for (int s = 0; s < 8; ++s) q_frag[warp][s][lane] = make_uint4(a[2 * s], b[2 * s], a[2 * s + 1], b[2 * s + 1]);
        __syncwarp();
      }

      const int* pages = p.table + static_cast<size_t>(seq) * p.width;
      const size_t plane = static_cast<size_t>(head) * p.pool_pages * kBlk;
      // the pool row of key `key`; a page outside the pool is flagged and read as page 0
      const auto row_of = [&](int key) -> size_t {
        int page = __ldg(pages + (key >> 7));
        if (page < 0 || page >= p.pool_pages) {
          if (p.err && lane == 0) atomicOr(p.err, kErrBadPage);
          page = 0;
        }
        return plane + static_cast<size_t>(page) * kBlk + (key & (kBlk - 1));
      };
      uint32_t kr[4][kKWords], vr[2][4][kVWords];
      const auto load_k = [&](size_t row) {
        const char* base = static_cast<const char*>(p.key_pool) + (row + r) * kRowBytes + c * (kKWords * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int k = 0; k < kKWords; k += 8) load32(base + j * 8 * kRowBytes + k * 4, kr[j] + k);
      };
      const auto load_v = [&](size_t row) {
        const char* base = static_cast<const char*>(p.value_pool) + (row + 2 * c) * kRowBytes + r * (kVWords * 4);
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const char* from = base + (g * 16 + (k >> 1) * 8 + (k & 1)) * kRowBytes;
            if constexpr (kFp8) load16(from, vr[g][k]);
            else load32(from, vr[g][k]);
          }
      };
      float o[16][4];
#pragma unroll
      for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
      size_t row = row_of(key0);
      load_k(row);
      load_v(row);
#pragma unroll 1
      for (int i = 0; i < n_units; ++i) {
        const int key = key0 + i * kRowUnit;
        float s[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
        for (int st = 0; st < 8; ++st) {
          const uint4 a = q_frag[warp][st][lane];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (kFp8) mma16<true>(s[j], a, f16x2_of_e4m3x2(kr[j][st]), f16x2_of_e4m3x2(kr[j][st] >> 16));
            else mma16<false>(s[j], a, kr[j][2 * st], kr[j][2 * st + 1]);
          }
        }
        size_t next_row = row;
        if (i + 1 < n_units) {
          next_row = (key + kRowUnit) & (kBlk - 1) ? row + kRowUnit : row_of(key + kRowUnit);
          load_k(next_row);
        }
        // keys at or past a row's limit are hidden from it
        if (__any_sync(0xffffffffu, key + kRowUnit > min(lim0, lim1))) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int at_key = key + 8 * j + 2 * c + k;
              if (at_key >= lim0) s[j][k] = -INFINITY;
              if (at_key >= lim1) s[j][2 + k] = -INFINITY;
            }
        }
        float t0 = fmaxf(fmax3(fmaxf(s[0][0], s[0][1]), s[1][0], s[1][1]), fmax3(fmaxf(s[2][0], s[2][1]), s[3][0], s[3][1]));
        float t1 = fmaxf(fmax3(fmaxf(s[0][2], s[0][3]), s[1][2], s[1][3]), fmax3(fmaxf(s[2][2], s[2][3]), s[3][2], s[3][3]));
        t0 = quad_max(t0) * sl2;
        t1 = quad_max(t1) * sl2b;
        const bool need0 = t0 > m0 + kThreshold, need1 = t1 > m1 + kThreshold;
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
        const float b0 = m0 == -INFINITY ? 0.f : -m0, b1 = m1 == -INFINITY ? 0.f : -m1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[j][0] = fast_exp2(fmaf(s[j][0], sl2, b0));
          s[j][1] = fast_exp2(fmaf(s[j][1], sl2, b0));
          s[j][2] = fast_exp2(fmaf(s[j][2], sl2b, b1));
          s[j][3] = fast_exp2(fmaf(s[j][3], sl2b, b1));
          l0 += s[j][0] + s[j][1];
          l1 += s[j][2] + s[j][3];
        }
        // values past the sequence's end may be anything, NaN too, and P's zeros do not undo that
        if (key + kRowUnit > kv_end) {
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (key + g * 16 + 2 * c + (k >> 1) * 8 + (k & 1) >= kv_end)
#pragma unroll
                for (int w = 0; w < kVWords; ++w) vr[g][k][w] = 0u;
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          uint4 a;
          if constexpr (kFp8)
            a = make_uint4(f16x2_of(s[2 * g][0], s[2 * g][1]), f16x2_of(s[2 * g][2], s[2 * g][3]),
                           f16x2_of(s[2 * g + 1][0], s[2 * g + 1][1]), f16x2_of(s[2 * g + 1][2], s[2 * g + 1][3]));
          else
            a = make_uint4(pack_bf16x2(s[2 * g][0], s[2 * g][1]), pack_bf16x2(s[2 * g][2], s[2 * g][3]),
                           pack_bf16x2(s[2 * g + 1][0], s[2 * g + 1][1]), pack_bf16x2(s[2 * g + 1][2], s[2 * g + 1][3]));
#pragma unroll
          for (int w = 0; w < kVWords; ++w) {
            const uint32_t x = vr[g][0][w], y = vr[g][1][w], z = vr[g][2][w], v = vr[g][3][w];
            if constexpr (kFp8) {  // four columns a word
              const uint32_t xy = __byte_perm(x, y, 0x5140), zv = __byte_perm(z, v, 0x5140);
              const uint32_t xy2 = __byte_perm(x, y, 0x7362), zv2 = __byte_perm(z, v, 0x7362);
              mma16<true>(o[4 * w], a, f16x2_of_e4m3x2(xy), f16x2_of_e4m3x2(zv));
              mma16<true>(o[4 * w + 1], a, f16x2_of_e4m3x2(xy >> 16), f16x2_of_e4m3x2(zv >> 16));
              mma16<true>(o[4 * w + 2], a, f16x2_of_e4m3x2(xy2), f16x2_of_e4m3x2(zv2));
              mma16<true>(o[4 * w + 3], a, f16x2_of_e4m3x2(xy2 >> 16), f16x2_of_e4m3x2(zv2 >> 16));
            } else {  // two
              mma16<false>(o[2 * w], a, __byte_perm(x, y, 0x5410), __byte_perm(z, v, 0x5410));
              mma16<false>(o[2 * w + 1], a, __byte_perm(x, y, 0x7632), __byte_perm(z, v, 0x7632));
            }
          }
        }
        if (i + 1 < n_units) load_v(next_row);
        row = next_row;
      }
      l0 = quad_sum(l0);
      l1 = quad_sum(l1);
      // ---- columns 32c .. + 31 of rows r and r + 8: o[j][0 / 2] is column j, o[j][1 / 3] column 16 + j
      const long long item = at.b < 0 ? static_cast<long long>(head) * ln.shared_tiles + at.t
                                      : (static_cast<long long>(head) * p.batch + at.b) * ln.own_tiles + at.t;
      const long long slot = (at.b < 0 ? 0 : p.own_row0) + (item + worker) * (at.b < 0 ? p.shared_slot_rows : p.own_slot_rows);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row_in = r + 8 * half;
        if (row_in >= n_rows) continue;
        const float l = half ? l1 : l0, m = half ? m1 : m0;
        if (direct) {
          float w = l == 0.f ? 0.f : 1.0f / l;
          if constexpr (kFp8) w *= __ldg(p.v_scale + head);
          const RowAt& ra = half ? at1 : at0;
          const long long id = (static_cast<long long>(ra.b) * p.rows + ra.i) * p.heads + ra.h;
          uint4* dst = reinterpret_cast<uint4*>(p.out + id * kD + 32 * c);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int j = (k & 1) * 8, e = 2 * half + (k >> 1);
            dst[k] = make_uint4(pack_bf16x2(o[j][e] * w, o[j + 1][e] * w), pack_bf16x2(o[j + 2][e] * w, o[j + 3][e] * w),
                                pack_bf16x2(o[j + 4][e] * w, o[j + 5][e] * w), pack_bf16x2(o[j + 6][e] * w, o[j + 7][e] * w));
          }
          if (p.lse && c == 0) p.lse[id] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        } else {
          if (c == 0) p.part_ml[slot + row_in] = make_float2(m, l);
          float4* dst = reinterpret_cast<float4*>(p.part_o + (slot + row_in) * kD + 32 * c);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int j = (k & 3) * 4, e = 2 * half + (k >> 2);
            dst[k] = make_float4(o[j][e], o[j + 1][e], o[j + 2][e], o[j + 3][e]);
          }
        }
      }
    }
    u += part;
    if (u < u_end) step_item(p, ln, pl, at);
  }
  if (worker == 0) {
    flag_lengths(p, lane);
    write_plan(p, ln, pl, p.plan + 3 + p.batch, lane);
  }
  // what follows this kernel needs the other line's too
  if (after) asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace

cudaError_t launch_branch_rows(const BranchParams& p, bool e4m3, bool after, cudaLaunchConfig_t cfg) {
  cfg.gridDim = dim3(p.warp.workers / kRowWarps);
  cfg.blockDim = dim3(32 * kRowWarps);
  cfg.dynamicSmemBytes = 0;
  return e4m3 ? cudaLaunchKernelEx(&cfg, branch_rows_kernel<true>, p, after)
              : cudaLaunchKernelEx(&cfg, branch_rows_kernel<false>, p, after);
}

}  // namespace h3sa
