// Drafted trees: ancestor bits and positions of a tree's rows, and the move of an accepted path's rows
// behind the history in every pool tensor.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>
#include <functional>
#include <memory>
#include <new>

#include "h3sa_host.h"
#include "h3sa_ptx.cuh"

namespace h3sa {
namespace {

constexpr int kPage = 128;
constexpr int kTreeThreads = 128;  // nodes of a block
constexpr int kMaxNodes = 1024;

struct TreeArgs {
  const int* parents;  // [batch, nodes]
  const int* lengths;
  const int* counts;  // or null
  int batch, nodes, words;
  uint32_t* masks;  // [batch, nodes, words]
  int* positions;   // [batch, nodes]
  int* err;
};

// A thread walks from its node to the root through parents in shared memory, and as they only get
// smaller it meets the words of its mask once each, the last one first. Bound by latency: the loads of the
// parents, some 30 cycles a step of the deepest chain, and the way out. Masks go out through shared memory in whole lines.
// Measured: a few nodes of two sequences 4.2 us, an empty kernel's 2 and three dependent loads; 64 trees of up to 500 nodes 8.3.
__global__ void __launch_bounds__(kTreeThreads) draft_tree_kernel(const TreeArgs a) {
  extern __shared__ int tree_smem[];
  const int b = blockIdx.y, n0 = blockIdx.x * kTreeThreads;
  const int n_end = min(a.nodes, n0 + kTreeThreads), stride = a.words | 1;  // an odd stride: no bank conflicts
  int* const parent = tree_smem;  // [n_end]
  uint32_t* const rows = reinterpret_cast<uint32_t*>(tree_smem + a.nodes);  // [kTreeThreads][stride]
  const int length = __ldg(a.lengths + b);
  const int count = a.counts ? min(a.nodes, __ldg(a.counts + b)) : a.nodes;
  bool bad = a.counts && threadIdx.x == 0 && (__ldg(a.counts + b) < 0 || __ldg(a.counts + b) > a.nodes);
  for (int i = threadIdx.x; i < n_end; i += kTreeThreads) {
    const int q = __ldg(a.parents + static_cast<size_t>(b) * a.nodes + i);
    const bool ok = q >= -1 && q < i;
    bad |= !ok && i < count;
    parent[i] = ok ? q : -1;  // so that every walk ends
  }
  if (bad && a.err && blockIdx.x == gridDim.x - 1) atomicOr(a.err, kErrBadIndex);
  __syncthreads();
  const int node = n0 + threadIdx.x;
  if (node < n_end) {
    uint32_t* const row = rows + threadIdx.x * stride;
    int depth = -1, w = a.words;
    if (node < count) {
      uint32_t bits = 0u;
      w = node >> 5;
      for (int k = a.words - 1; k > w; --k) row[k] = 0u;
      for (int at = node; at >= 0; at = parent[at], ++depth) {
        for (; w > at >> 5; --w) {
          row[w] = bits;
          bits = 0u;
        }
        bits |= 1u << (at & 31);
      }
      row[w--] = bits;
      for (; w >= 0; --w) row[w] = 0u;
    } else {
      for (int k = 0; k < a.words; ++k) row[k] = 0u;
    }
    a.positions[static_cast<size_t>(b) * a.nodes + node] = depth < 0 ? 0 : length + depth;
  }
  __syncthreads();
  uint32_t* const out = a.masks + (static_cast<size_t>(b) * a.nodes + n0) * a.words;
  for (int i = threadIdx.x; i < (n_end - n0) * a.words; i += kTreeThreads) {
    const int r = i / a.words;
    out[i] = rows[r * stride + i - r * a.words];
  }
}

constexpr int kMaxPools = 128;  // tensors a launch
struct KeepArgs {
  char* base[kMaxPools];
  int count, heads, pages, row_vecs;  // a row: 16-byte vectors
  const int* table;
  const int* lengths;
  const int* path;  // [batch, steps]
  int batch, width, steps;
  int* lengths_out;  // null in launches after the first
  int* err;
};

// Row lengths + path[k] of a sequence goes to lengths + k. The path ascends, so path[k] >= k and no row is
// written before the ones in front of it have been read: a warp that takes a sequence's rows of one
// plane in order, all of a batch read before any is written, moves them in place. Bound by latency: path and
// length, then the table, then the rows, eight loads a lane on their way. Measured: one layer's two tensors 4.2 us, 100 tensors of 50 layers 8.3 (0.8 TB/s of the rows moved).
constexpr int kKeepWarps = 4;
constexpr int kKeepLoads = 8;
__global__ void __launch_bounds__(32 * kKeepWarps) keep_rows_kernel(const KeepArgs a) {
  const int lane = threadIdx.x & 31, half = lane >> 4, col = lane & 15;
  const long long item = static_cast<long long>(blockIdx.x) * kKeepWarps + (threadIdx.x >> 5);
  const int planes = a.count * a.heads;
  if (item >= static_cast<long long>(planes) * a.batch) return;
  const int b = static_cast<int>(item / planes), plane = static_cast<int>(item - static_cast<long long>(b) * planes);
  const int length = __ldg(a.lengths + b);
  const int* const path = a.path + static_cast<size_t>(b) * a.steps;
  const int* const table = a.table + static_cast<size_t>(b) * a.width;
  const long long room = static_cast<long long>(a.width) * kPage - length;  // rows that the table has places for
  const auto page_of = [&](int row) { return __ldg(table + ((length + row) >> 7)); };
  // the path's end, and whether all of it can be moved
  int kept = a.steps, last = -1;
  bool order = length >= 0, pages_ok = true;
  for (int k0 = 0; k0 < kept; k0 += 32) {
    const int k = k0 + lane, at = k < a.steps ? __ldg(path + k) : -1;
    const uint32_t ends = __ballot_sync(0xffffffffu, at < 0);
    const int n = ends ? __ffs(ends) - 1 : 32;
    const int before = __shfl_up_sync(0xffffffffu, at, 1);
    if (lane < n) {
      order = order && at > (lane > 0 ? before : last) && at < room;
      if (order) {
        const int from = page_of(at), to = page_of(k);
        pages_ok = pages_ok && from >= 0 && from < a.pages && to >= 0 && to < a.pages;
      }
    }
    last = __shfl_sync(0xffffffffu, at, 31);
    if (ends) kept = k0 + n;
  }
  order = __all_sync(0xffffffffu, order);
  pages_ok = __all_sync(0xffffffffu, pages_ok);
  const bool ok = order && pages_ok;
  if (plane == 0 && lane == 0 && a.lengths_out) {
    a.lengths_out[b] = ok ? length + kept : length;
    if (!ok && a.err) atomicOr(a.err, order ? kErrBadPage : kErrBadIndex);
  }
  if (!ok) return;
  uint4* const rows = reinterpret_cast<uint4*>(a.base[plane / a.heads]) +
                      static_cast<size_t>(plane % a.heads) * a.pages * kPage * a.row_vecs;
  const auto place = [&](int row) {
    return (static_cast<size_t>(page_of(row)) * kPage + ((length + row) & (kPage - 1))) * a.row_vecs;
  };
  for (int c = col; c - col < a.row_vecs; c += 16) {
    for (int k0 = 0; k0 < kept; k0 += 2 * kKeepLoads) {
      uint4 v[kKeepLoads];
      size_t to[kKeepLoads];
      bool moves[kKeepLoads];
#pragma unroll
      for (int j = 0; j < kKeepLoads; ++j) {
        const int k = k0 + 2 * j + half;
        const int at = k < kept ? __ldg(path + k) : k;
        moves[j] = at != k && c < a.row_vecs;
        if (moves[j]) {
          to[j] = place(k) + c;
          v[j] = rows[place(at) + c];
        }
      }
      __syncwarp();
#pragma unroll
      for (int j = 0; j < kKeepLoads; ++j)
        if (moves[j]) rows[to[j]] = v[j];
      __syncwarp();
    }
  }
}

// Whether pool tensors are apart: rows move in place, and a tensor given twice would see them move twice.
int check_apart(const h3sa_pools* p) {
  const int64_t bytes = static_cast<int64_t>(p->heads) * p->pages * kPage * p->row_bytes;
  bool apart = true;
  if (!p->list) {
    apart = p->count < 2 || p->stride >= bytes || p->stride <= -bytes;
  } else if (p->count > 1) {
    const std::unique_ptr<const char*[]> at(new (std::nothrow) const char*[p->count]);
    if (!at) return set_error(H3SA_ERR_INVALID, "keep_rows: no host memory for %d addresses", p->count);
    for (int i = 0; i < p->count; ++i) at[i] = static_cast<const char*>(p->list[i]);
    std::sort(at.get(), at.get() + p->count, std::less<const char*>());
    for (int i = 1; i < p->count; ++i) apart = apart && at[i] - at[i - 1] >= bytes;
  }
  return apart ? H3SA_OK : set_error(H3SA_ERR_INVALID, "keep_rows: pool tensors overlap");
}

}  // namespace
}  // namespace h3sa

using namespace h3sa;

extern "C" {

int h3sa_draft_tree(const int32_t* parents, int32_t batch, int32_t nodes, const int32_t* lengths, const int32_t* counts,
                    int32_t* masks, int32_t* positions, int32_t* device_error, void* stream) {
  if (batch < 0 || nodes < 0 || batch > 65535 || nodes > kMaxNodes)
    return set_error(H3SA_ERR_INVALID, "draft tree: invalid sizes batch=%d (at most 65535) nodes=%d (at most %d)", batch,
                     nodes, kMaxNodes);
  if (batch == 0 || nodes == 0) return H3SA_OK;
  if (!parents || !lengths || !masks || !positions)
    return set_error(H3SA_ERR_INVALID, "draft tree: null pointer argument");
  TreeArgs a{parents, lengths, counts, batch, nodes, (nodes + 31) / 32, reinterpret_cast<uint32_t*>(masks), positions,
             device_error};
  const size_t smem = 4 * (static_cast<size_t>(nodes) + kTreeThreads * (a.words | 1));
  static_assert(4 * (kMaxNodes + kTreeThreads * (kMaxNodes / 32 + 1)) <= 48 * 1024, "a tree needs more than 48 KB");
  draft_tree_kernel<<<dim3((nodes + kTreeThreads - 1) / kTreeThreads, batch), kTreeThreads, smem,
                      static_cast<cudaStream_t>(stream)>>>(a);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? H3SA_OK : set_cuda_error("draft_tree_kernel launch", e);
}

int h3sa_keep_rows(const h3sa_pools* pools, const int32_t* table, int32_t sequences, int32_t width,
                   const int32_t* lengths, const int32_t* path, int32_t steps, int32_t* lengths_out,
                   int32_t* device_error, void* stream) {
  if (const int rc = check_pools("keep_rows", pools)) return rc;
  if (!ledger_sizes_ok(sequences, width) || steps < 0 || static_cast<int64_t>(sequences) * steps > INT32_MAX)
    return set_error(H3SA_ERR_INVALID, "keep_rows: invalid sizes sequences=%d width=%d steps=%d", sequences, width, steps);
  if (sequences == 0) return H3SA_OK;
  if (!table || !lengths || !lengths_out || (steps > 0 && !path))
    return set_error(H3SA_ERR_INVALID, "keep_rows: null pointer argument");
  const long long items = static_cast<long long>(pools->count < kMaxPools ? pools->count : kMaxPools) * pools->heads * sequences;
  if (pools->count == 0 || items > static_cast<long long>(INT32_MAX))
    return set_error(H3SA_ERR_INVALID, "keep_rows: %d pool tensors of %d heads and %d sequences are none or too many",
                     pools->count, pools->heads, sequences);
  if (const int rc = check_apart(pools)) return rc;
  for (int first = 0; first < pools->count; first += kMaxPools) {
    KeepArgs a;
    memset(&a, 0, sizeof(a));
    a.count = pools->count - first < kMaxPools ? pools->count - first : kMaxPools;
    for (int i = 0; i < a.count; ++i)
      a.base[i] = pools->list ? static_cast<char*>(pools->list[first + i])
                              : static_cast<char*>(pools->base) + (first + i) * pools->stride;
    a.heads = pools->heads;
    a.pages = pools->pages;
    a.row_vecs = pools->row_bytes / 16;
    a.table = table;
    a.lengths = lengths;
    a.path = path;
    a.batch = sequences;
    a.width = width;
    a.steps = steps;
    a.lengths_out = first == 0 ? lengths_out : nullptr;
    a.err = device_error;
    const long long warps = static_cast<long long>(a.count) * a.heads * sequences;
    keep_rows_kernel<<<static_cast<unsigned>((warps + kKeepWarps - 1) / kKeepWarps), 32 * kKeepWarps, 0,
                       static_cast<cudaStream_t>(stream)>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error("keep_rows_kernel launch", e);
  }
  return H3SA_OK;
}

}  // extern "C"
