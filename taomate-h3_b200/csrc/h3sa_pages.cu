// Page bookkeeping of a pool that several branches share: fork, free and compact.
//
// A pool's ledger is a table [sequences, width] of page indices (-1: none), a length per sequence
// and a reference count per page (the number of table entries that hold it; 0: free). The tensors
// that hold rows (K and V of every layer) are planes of the same pages, so one ledger serves them
// all and one launch copies rows in all of them. Everything is decided on the device from the
// ledger; fresh pages are the lowest free ones, taken in branch order, so results do not depend on
// timing.
#include <cuda_runtime.h>

#include <climits>
#include <cstring>

#include "h3sa_host.h"
#include "h3sa_ptx.cuh"

namespace h3sa {
namespace {

constexpr int kPage = 128;
constexpr int kMetaThreads = 1024;
constexpr int kMaxPools = 128;  // tensors per copy launch
struct Pools {
  char* base[kMaxPools];
  int count, heads, pages, row_bytes;
};

// Exclusive prefix sum of one value per thread over the block; `total` gets the sum.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int mine = 0, all = 0;
  for (int w = 0; w < kMetaThreads / 32; ++w) {
    if (w == warp) mine = all;
    all += warp_sums[w];
  }
  total = all;
  return mine + x - v;
}

struct ForkArgs {
  const int* table;
  const int* lengths;
  const int* refs;
  const int* parents;
  int sequences, width, pages, children, reserve, deep;
  int* child_table;
  int* child_lengths;
  int* refs_out;
  int* fresh;   // [pages] free pages in order
  int* start;   // [children] first fresh page of each child, then first move
  int4* moves;  // (source page, destination page, rows, 0)
  int* n_moves;
  int* err;
};

__global__ void __launch_bounds__(kMetaThreads) fork_kernel(const ForkArgs a) {
  __shared__ int sums[kMetaThreads / 32];
  __shared__ int bad;
  const int tid = threadIdx.x;
  if (tid == 0) bad = 0;
  __syncthreads();
  // fresh pages of each child
  int need_all = 0;
  for (int c0 = 0; c0 < a.children; c0 += kMetaThreads) {
    const int c = c0 + tid;
    int n = 0;
    if (c < a.children) {
      const int parent = a.parents[c];
      int len = 0;
      if (parent >= a.sequences) atomicOr(&bad, kErrBadIndex);
      else if (parent >= 0) len = a.lengths[parent];
      const long long end = static_cast<long long>(len) + a.reserve;
      if (len < 0 || (end + kPage - 1) / kPage > a.width) atomicOr(&bad, kErrBadIndex);
      else n = static_cast<int>((end + kPage - 1) / kPage) - (a.deep ? 0 : len / kPage);
    }
    int total;
    const int before = block_scan(n, sums, total);
    if (c < a.children) a.start[c] = need_all + before;
    need_all += total;
  }
  // the free pages in order
  int n_free = 0;
  for (int p0 = 0; p0 < a.pages; p0 += kMetaThreads) {
    const int p = p0 + tid;
    const int r = p < a.pages ? a.refs[p] : 1;
    if (p < a.pages) a.refs_out[p] = r;
    int total;
    const int before = block_scan(r == 0 ? 1 : 0, sums, total);
    if (r == 0) a.fresh[n_free + before] = p;
    n_free += total;
  }
  __syncthreads();
  if (need_all > n_free && tid == 0) bad |= kErrNoPages;
  // pages that parents hold must be pages of the pool
  for (int c = tid >> 5; c < a.children; c += kMetaThreads / 32) {
    const int parent = a.parents[c];
    if (parent < 0 || parent >= a.sequences) continue;
    const int len = a.lengths[parent];
    if (len < 0 || len > a.width * static_cast<long long>(kPage)) continue;
    for (int j = tid & 31; j < (len + kPage - 1) / kPage; j += 32) {
      const int page = a.table[static_cast<size_t>(parent) * a.width + j];
      if (page < 0 || page >= a.pages || a.refs[page] <= 0) atomicOr(&bad, kErrBadPage);
    }
  }
  __syncthreads();
  const bool ok = bad == 0;
  if (!ok && tid == 0 && a.err) atomicOr(a.err, bad);
  if (tid == 0) *a.n_moves = 0;
  __syncthreads();
  for (int c = tid >> 5; c < a.children; c += kMetaThreads / 32) {
    const int parent = a.parents[c];
    const int len = ok && parent >= 0 ? a.lengths[parent] : 0;
    const int held = (len + kPage - 1) / kPage;
    const int kept = a.deep ? 0 : len / kPage;
    const int need = ok ? static_cast<int>((static_cast<long long>(len) + a.reserve + kPage - 1) / kPage) : 0;
    const int start = a.start[c];
    const int* mine = a.table + static_cast<size_t>(parent < 0 ? 0 : parent) * a.width;
    for (int j = tid & 31; j < a.width; j += 32) {
      int page = -1;
      if (j < kept) {
        page = mine[j];
        atomicAdd(a.refs_out + page, 1);
      } else if (j < need) {
        page = a.fresh[start + j - kept];
        a.refs_out[page] = 1;
        if (j < held)
          a.moves[atomicAdd(a.n_moves, 1)] = make_int4(mine[j], page, min(kPage, len - j * kPage), 0);
      }
      a.child_table[static_cast<size_t>(c) * a.width + j] = page;
    }
    if ((tid & 31) == 0) a.child_lengths[c] = len;
  }
}

struct CompactArgs {
  const int* table;
  const int* refs;
  int entries, pages;
  int* table_out;
  int* refs_out;
  int* live;
  int* to;      // [pages]
  int4* moves;
  int* n_moves;
  int* err;
};

__global__ void __launch_bounds__(kMetaThreads) compact_kernel(const CompactArgs a) {
  __shared__ int sums[kMetaThreads / 32];
  const int tid = threadIdx.x;
  int live = 0;
  for (int p0 = 0; p0 < a.pages; p0 += kMetaThreads) {
    int total;
    const int p = p0 + tid;
    block_scan(p < a.pages && a.refs[p] > 0 ? 1 : 0, sums, total);
    live += total;
  }
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < a.pages; p0 += kMetaThreads) {
    const int p = p0 + tid;
    const bool used = p < a.pages && a.refs[p] > 0;
    const bool hole = p < live && !used, mover = p >= live && used;
    int n_hole, n_mover;
    const int h = holes + block_scan(hole ? 1 : 0, sums, n_hole);
    const int m = movers + block_scan(mover ? 1 : 0, sums, n_mover);
    if (hole) a.moves[h].y = p;
    if (mover) {
      a.moves[m].x = p;
      a.moves[m].z = kPage;
    }
    if (p < a.pages) {
      a.to[p] = used && p < live ? p : -1;
      a.refs_out[p] = used && p < live ? a.refs[p] : 0;
    }
    holes += n_hole;
    movers += n_mover;
  }
  __syncthreads();
  for (int i = tid; i < movers; i += kMetaThreads) {
    const int4 mv = a.moves[i];
    a.to[mv.x] = mv.y;
    a.refs_out[mv.y] = a.refs[mv.x];
  }
  if (tid == 0) {
    *a.n_moves = movers;
    *a.live = live;
  }
  __syncthreads();
  for (int i = tid; i < a.entries; i += kMetaThreads) {
    const int page = a.table[i];
    int now = -1;
    if (page >= 0) {
      if (page < a.pages) now = a.to[page];
      if (now < 0 && a.err) atomicOr(a.err, kErrBadPage);  // no such page, or a free one
    }
    a.table_out[i] = now;
  }
}

struct FreeArgs {
  const int* table;
  const int* lengths;
  const int* refs;
  const uint8_t* release;
  int sequences, width, pages;
  int* table_out;
  int* lengths_out;
  int* refs_out;
  int* err;
};

__global__ void __launch_bounds__(kMetaThreads) free_kernel(const FreeArgs a) {
  const int tid = threadIdx.x;
  for (int p = tid; p < a.pages; p += kMetaThreads) a.refs_out[p] = a.refs[p];
  __syncthreads();
  for (int i = tid; i < a.sequences * a.width; i += kMetaThreads) {
    const int page = a.table[i];
    const bool gone = a.release[i / a.width] != 0;
    if (gone && page >= 0) {
      if (page >= a.pages || atomicSub(a.refs_out + page, 1) <= 0) {
        if (page < a.pages) atomicAdd(a.refs_out + page, 1);
        if (a.err) atomicOr(a.err, kErrBadPage);
      }
    }
    a.table_out[i] = gone ? -1 : page;
  }
  for (int s = tid; s < a.sequences; s += kMetaThreads) a.lengths_out[s] = a.release[s] ? 0 : a.lengths[s];
}

// Rows [0, rows) of each move's source page to its destination page, in every plane.
__global__ void __launch_bounds__(256) copy_pages_kernel(const Pools pools, const int4* moves,
                                                         const int* n_moves) {
  const int planes = pools.count * pools.heads;
  const long long items = static_cast<long long>(*n_moves) * planes;
  for (long long i = blockIdx.x; i < items; i += gridDim.x) {
    const int plane = static_cast<int>(i % planes);
    const int4 mv = moves[i / planes];
    const size_t plane_rows = static_cast<size_t>(plane % pools.heads) * pools.pages * kPage;
    char* base = pools.base[plane / pools.heads];
    const uint4* src = reinterpret_cast<const uint4*>(base + (plane_rows + static_cast<size_t>(mv.x) * kPage) * pools.row_bytes);
    uint4* dst = reinterpret_cast<uint4*>(base + (plane_rows + static_cast<size_t>(mv.y) * kPage) * pools.row_bytes);
    const int n = mv.z * (pools.row_bytes >> 4);
    for (int j = threadIdx.x; j < n; j += 256) dst[j] = src[j];
  }
}

int copy_launch(const h3sa_pools* pools, const int4* moves, const int* n_moves, cudaStream_t stream) {
  for (int first = 0; first < pools->count; first += kMaxPools) {
    Pools p;
    memset(&p, 0, sizeof(p));
    p.count = pools->count - first < kMaxPools ? pools->count - first : kMaxPools;
    p.heads = pools->heads;
    p.pages = pools->pages;
    p.row_bytes = pools->row_bytes;
    for (int i = 0; i < p.count; ++i)
      p.base[i] = pools->list ? static_cast<char*>(pools->list[first + i])
                              : static_cast<char*>(pools->base) + (first + i) * pools->stride;
    copy_pages_kernel<<<148 * 8, 256, 0, stream>>>(p, moves, n_moves);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error("copy_pages_kernel launch", e);
  }
  return H3SA_OK;
}

int check_pools(const char* what, const h3sa_pools* p) {
  if (!p || p->count < 0 || p->heads <= 0 || p->pages <= 0 || p->row_bytes <= 0 || p->row_bytes % 16)
    return set_error(H3SA_ERR_INVALID, "%s: invalid pools (row bytes must be a positive multiple of 16)", what);
  if (static_cast<int64_t>(p->pages) * kPage > INT32_MAX)
    return set_error(H3SA_ERR_INVALID, "%s: pool of %d pages too large", what, p->pages);
  for (int i = 0; i < p->count; ++i) {
    const char* base = p->list ? static_cast<const char*>(p->list[i])
                               : (p->base ? static_cast<const char*>(p->base) + i * p->stride : nullptr);
    if (!base || (reinterpret_cast<uintptr_t>(base) & 15u))
      return set_error(H3SA_ERR_INVALID, "%s: pool tensors must be non-null and 16-byte aligned", what);
  }
  return H3SA_OK;
}

}  // namespace
}  // namespace h3sa

using namespace h3sa;

extern "C" {

int64_t h3sa_pages_workspace(int32_t pages, int32_t children) {
  if (pages <= 0 || children < 0) return 0;
  // the moves come first (16 bytes each), then free pages / the page map, starts and the count
  return 16ll * pages + 4ll * pages + 4ll * children + 16;
}

int h3sa_fork_pages(const h3sa_pools* pools, const int32_t* table, int32_t sequences, int32_t width,
                    const int32_t* lengths, const int32_t* refs, const int32_t* parents,
                    int32_t children, int32_t reserve_rows, int32_t private_copy,
                    int32_t* child_table, int32_t* child_lengths, int32_t* refs_out, void* workspace,
                    int32_t* device_error, void* stream) {
  int rc = check_pools("fork_pages", pools);
  if (rc) return rc;
  if (sequences < 0 || width <= 0 || children < 0 || reserve_rows < 0 ||
      static_cast<int64_t>(width) * kPage > INT32_MAX ||
      static_cast<int64_t>(sequences) * width > INT32_MAX || static_cast<int64_t>(children) * width > INT32_MAX)
    return set_error(H3SA_ERR_INVALID, "fork_pages: invalid sizes sequences=%d width=%d children=%d reserve=%d",
                     sequences, width, children, reserve_rows);
  if ((sequences > 0 && (!table || !lengths)) || !refs || !refs_out || !workspace ||
      (children > 0 && (!parents || !child_table || !child_lengths)))
    return set_error(H3SA_ERR_INVALID, "fork_pages: null pointer argument");
  if (reinterpret_cast<uintptr_t>(workspace) & 15u)
    return set_error(H3SA_ERR_INVALID, "fork_pages: workspace must be 16-byte aligned");
  ForkArgs a;
  a.table = table;
  a.lengths = lengths;
  a.refs = refs;
  a.parents = parents;
  a.sequences = sequences;
  a.width = width;
  a.pages = pools->pages;
  a.children = children;
  a.reserve = reserve_rows;
  a.deep = private_copy ? 1 : 0;
  a.child_table = child_table;
  a.child_lengths = child_lengths;
  a.refs_out = refs_out;
  a.moves = static_cast<int4*>(workspace);
  a.fresh = reinterpret_cast<int*>(a.moves + pools->pages);
  a.start = a.fresh + pools->pages;
  a.n_moves = a.start + children;
  a.err = device_error;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  fork_kernel<<<1, kMetaThreads, 0, s>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error("fork_kernel launch", e);
  return copy_launch(pools, a.moves, a.n_moves, s);
}

int h3sa_compact_pages(const h3sa_pools* pools, const int32_t* table, int32_t sequences, int32_t width,
                       const int32_t* refs, int32_t* table_out, int32_t* refs_out, int32_t* live,
                       void* workspace, int32_t* device_error, void* stream) {
  int rc = check_pools("compact_pages", pools);
  if (rc) return rc;
  if (sequences < 0 || width <= 0 || static_cast<int64_t>(sequences) * width > INT32_MAX)
    return set_error(H3SA_ERR_INVALID, "compact_pages: invalid sizes sequences=%d width=%d", sequences, width);
  if ((sequences > 0 && (!table || !table_out)) || !refs || !refs_out || !live || !workspace)
    return set_error(H3SA_ERR_INVALID, "compact_pages: null pointer argument");
  if (reinterpret_cast<uintptr_t>(workspace) & 15u)
    return set_error(H3SA_ERR_INVALID, "compact_pages: workspace must be 16-byte aligned");
  CompactArgs a;
  a.table = table;
  a.refs = refs;
  a.entries = sequences * width;
  a.pages = pools->pages;
  a.table_out = table_out;
  a.refs_out = refs_out;
  a.live = live;
  a.moves = static_cast<int4*>(workspace);
  a.to = reinterpret_cast<int*>(a.moves + pools->pages);
  a.n_moves = a.to + pools->pages;
  a.err = device_error;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  compact_kernel<<<1, kMetaThreads, 0, s>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error("compact_kernel launch", e);
  return copy_launch(pools, a.moves, a.n_moves, s);
}

int h3sa_free_pages(const int32_t* table, int32_t sequences, int32_t width, const int32_t* lengths,
                    const int32_t* refs, int32_t pages, const uint8_t* release, int32_t* table_out,
                    int32_t* lengths_out, int32_t* refs_out, int32_t* device_error, void* stream) {
  if (sequences < 0 || width <= 0 || pages <= 0 || static_cast<int64_t>(sequences) * width > INT32_MAX)
    return set_error(H3SA_ERR_INVALID, "free_pages: invalid sizes sequences=%d width=%d pages=%d", sequences,
                     width, pages);
  if ((sequences > 0 && (!table || !lengths || !release || !table_out || !lengths_out)) || !refs || !refs_out)
    return set_error(H3SA_ERR_INVALID, "free_pages: null pointer argument");
  FreeArgs a{table, lengths, refs, release, sequences, width, pages, table_out, lengths_out, refs_out, device_error};
  free_kernel<<<1, kMetaThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error("free_kernel launch", e);
  return H3SA_OK;
}

}  // extern "C"
