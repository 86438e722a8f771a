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

// The ledger kernels are one thread block, or for large ledgers one cluster of eight: every phase
// needs the one before it whole, and a cluster's barrier is far cheaper than another launch.
template <int kCtas>
__device__ __forceinline__ int cluster_rank() {
  if constexpr (kCtas == 1) return 0;
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return static_cast<int>(r);
}
// All threads of the kernel meet; what they wrote to global memory before is visible after.
template <int kCtas>
__device__ __forceinline__ void meet() {
  if constexpr (kCtas == 1) {
    __syncthreads();
  } else {
    __threadfence();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

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
  int sum = warp_sums[lane];  // 32 warps
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += y;
  }
  total = __shfl_sync(0xffffffffu, sum, 31);
  const int before = __shfl_sync(0xffffffffu, sum, (warp + 31) & 31);
  return (warp > 0 ? before : 0) + x - v;
}

// The same over all threads of the kernel; `slots` are kCtas words of global memory of this call.
template <int kCtas>
__device__ __forceinline__ int kernel_scan(int v, int* warp_sums, int* slots, int& total) {
  int here;
  int before = block_scan(v, warp_sums, here);
  if constexpr (kCtas == 1) {
    total = here;
  } else {
    const int rank = cluster_rank<kCtas>();
    if (threadIdx.x == 0) slots[rank] = here;
    meet<kCtas>();
    total = 0;
    for (int k = 0; k < kCtas; ++k) {
      const int n = __ldcg(slots + k);
      if (k < rank) before += n;
      total += n;
    }
  }
  return before;
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
  int* start;   // [children] first fresh page of each child
  int4* moves;  // (source page, destination page, rows, 0)
  int* n_moves;
  int* bad;     // device error bits of this call
  int* slots;   // [kCtas]
  int* err;
};

// Two passes over a contiguous range of pages per thread, one to count and one to write, with one
// scan between them. Bound by latency: some six dependent reads and barriers.
template <int kCtas>
__global__ void __launch_bounds__(kMetaThreads) fork_kernel(const ForkArgs a) {
  __shared__ int sums[kMetaThreads / 32];
  const int tid = threadIdx.x, rank = cluster_rank<kCtas>();
  const int all_tid = rank * kMetaThreads + tid;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (all_tid == 0) {
    *a.n_moves = 0;
    *a.bad = 0;
  }
  meet<kCtas>();
  // fresh pages of each child (every block counts them all)
  int need_all = 0;
  for (int c0 = 0; c0 < a.children; c0 += kMetaThreads) {
    const int c = c0 + tid;
    int n = 0;
    if (c < a.children) {
      const int parent = a.parents[c];
      int len = 0;
      bool ok = parent < a.sequences;
      if (ok && parent >= 0) len = a.lengths[parent];
      const long long end = static_cast<long long>(len) + a.reserve;
      ok = ok && len >= 0 && (end + kPage - 1) / kPage <= a.width;
      if (ok) n = static_cast<int>((end + kPage - 1) / kPage) - (a.deep ? 0 : len / kPage);
      else if (rank == 0) atomicOr(a.bad, kErrBadIndex);
    }
    int total;
    const int before = block_scan(n, sums, total);
    if (rank == 0 && c < a.children) a.start[c] = need_all + before;
    need_all += total;
  }
  // the free pages in order
  const int per = (a.pages + kCtas * kMetaThreads - 1) / (kCtas * kMetaThreads);
  const int p_lo = min(a.pages, all_tid * per), p_hi = min(a.pages, p_lo + per);
  int mine = 0, n_free;
  for (int p = p_lo; p < p_hi; ++p) {
    const int r = a.refs[p];
    a.refs_out[p] = r;
    mine += r == 0 ? 1 : 0;
  }
  int at = kernel_scan<kCtas>(mine, sums, a.slots, n_free);
  for (int p = p_lo; mine > 0 && p < p_hi; ++p)
    if (a.refs[p] == 0) a.fresh[at++] = p;
  if (need_all > n_free && all_tid == 0) atomicOr(a.bad, kErrNoPages);
  // pages that parents hold must be pages of the pool that are in use
  constexpr int kWarps = kCtas * kMetaThreads / 32;
  for (int c = all_tid >> 5; c < a.children; c += kWarps) {
    const int parent = a.parents[c];
    if (parent < 0 || parent >= a.sequences) continue;
    const int len = a.lengths[parent];
    if (len < 0 || len > a.width * static_cast<long long>(kPage)) continue;
    for (int j = tid & 31; j < (len + kPage - 1) / kPage; j += 32) {
      const int page = a.table[static_cast<size_t>(parent) * a.width + j];
      if (page < 0 || page >= a.pages || a.refs[page] <= 0) atomicOr(a.bad, kErrBadPage);
    }
  }
  meet<kCtas>();
  const int bad = __ldcg(a.bad);
  const bool ok = bad == 0;
  if (!ok && all_tid == 0 && a.err) atomicOr(a.err, bad);
  for (int c = all_tid >> 5; c < a.children; c += kWarps) {
    const int parent = a.parents[c];
    const int len = ok && parent >= 0 ? a.lengths[parent] : 0;
    const int held = (len + kPage - 1) / kPage;
    const int kept = a.deep ? 0 : len / kPage;
    const int need = ok ? static_cast<int>((static_cast<long long>(len) + a.reserve + kPage - 1) / kPage) : 0;
    const int start = __ldcg(a.start + c);
    const int* from = a.table + static_cast<size_t>(parent < 0 ? 0 : parent) * a.width;
    for (int j = tid & 31; j < a.width; j += 32) {
      int page = -1;
      if (j < kept) {
        page = from[j];
        atomicAdd(a.refs_out + page, 1);
      } else if (j < need) {
        page = __ldcg(a.fresh + start + j - kept);
        a.refs_out[page] = 1;
        if (j < held)  // the order of the moves does not matter: they touch different pages
          a.moves[atomicAdd(a.n_moves, 1)] = make_int4(from[j], page, min(kPage, len - j * kPage), 0);
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
  int* slots;   // [2 * kCtas]
  int* err;
};

template <int kCtas>
__global__ void __launch_bounds__(kMetaThreads) compact_kernel(const CompactArgs a) {
  __shared__ int sums[kMetaThreads / 32];
  const int all_tid = cluster_rank<kCtas>() * kMetaThreads + threadIdx.x;
  constexpr int kThreads = kCtas * kMetaThreads;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int per = (a.pages + kThreads - 1) / kThreads;
  const int p_lo = min(a.pages, all_tid * per), p_hi = min(a.pages, p_lo + per);
  int used = 0, live;
  for (int p = p_lo; p < p_hi; ++p) used += a.refs[p] > 0 ? 1 : 0;
  const int before = kernel_scan<kCtas>(used, sums, a.slots, live);
  int movers = 0;
  for (int p = max(p_lo, live); p < p_hi; ++p) movers += a.refs[p] > 0 ? 1 : 0;
  int n_movers;
  // free pages in front of p_lo are p_lo less the used ones; only those below `live` are holes
  int h = p_lo <= live ? p_lo - before : 0;
  int m = kernel_scan<kCtas>(movers, sums, a.slots + kCtas, n_movers);
  for (int p = p_lo; p < p_hi; ++p) {
    const int r = a.refs[p];
    if (p < live && r <= 0) a.moves[h++].y = p;
    if (p >= live && r > 0) {
      a.moves[m].x = p;
      a.moves[m++].z = kPage;
    }
    a.to[p] = r > 0 && p < live ? p : -1;
    a.refs_out[p] = r > 0 && p < live ? r : 0;
  }
  meet<kCtas>();
  for (int i = all_tid; i < n_movers; i += kThreads) {
    const int4 mv = __ldcg(a.moves + i);
    a.to[mv.x] = mv.y;
    a.refs_out[mv.y] = a.refs[mv.x];
  }
  if (all_tid == 0) {
    *a.n_moves = n_movers;
    *a.live = live;
  }
  meet<kCtas>();
  for (int i = all_tid; i < a.entries; i += kThreads) {
    const int page = a.table[i];
    int now = -1;
    if (page >= 0) {
      if (page < a.pages) now = __ldcg(a.to + page);
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

// A warp takes 256 entries of a row at a time, loading all of them before it uses any. What is left
// is the atomics on the counts and one barrier; a single block with a division per entry took 68 us
// for 256 rows of 1000.
template <int kCtas>
__global__ void __launch_bounds__(kMetaThreads) free_kernel(const FreeArgs a) {
  constexpr int kThreads = kCtas * kMetaThreads, kRun = 8;
  const int all_tid = cluster_rank<kCtas>() * kMetaThreads + threadIdx.x, lane = threadIdx.x & 31;
  for (int p = all_tid; p < a.pages; p += kThreads) a.refs_out[p] = a.refs[p];
  for (int s = all_tid; s < a.sequences; s += kThreads) a.lengths_out[s] = a.release[s] ? 0 : a.lengths[s];
  meet<kCtas>();
  const int parts = (a.width + 32 * kRun - 1) / (32 * kRun);
  for (int i = all_tid >> 5; i < a.sequences * parts; i += kThreads / 32) {
    const int s = i / parts, j0 = (i - s * parts) * 32 * kRun + lane;
    const bool gone = a.release[s] != 0;
    const int* row = a.table + static_cast<size_t>(s) * a.width;
    int* out = a.table_out + static_cast<size_t>(s) * a.width;
    int page[kRun];
#pragma unroll
    for (int k = 0; k < kRun; ++k) page[k] = j0 + 32 * k < a.width ? row[j0 + 32 * k] : -1;
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      if (j0 + 32 * k < a.width) out[j0 + 32 * k] = gone ? -1 : page[k];
      if (gone && page[k] >= 0) {
        if (page[k] >= a.pages || atomicSub(a.refs_out + page[k], 1) <= 0) {
          if (page[k] < a.pages) atomicAdd(a.refs_out + page[k], 1);
          if (a.err) atomicOr(a.err, kErrBadPage);
        }
      }
    }
  }
}

// Ledgers of more than this many words take the cluster, whose barriers cost more than they bring
// on smaller ones. Measured, one block and eight: free of 4048 words 4.2 / 4.3 us, 12192 words
// 7.2 / 5.1, 296000 words 54 / 12.9; compact 5600 words 7.6 / 10.1, 11200 words 17.5 / 10.1; fork
// 5280 words 7.0 / 9.1, 9280 words 13.4 / 9.6.
constexpr int kClusterWords = 7168;
constexpr int kCluster = 8;

template <typename Args>
int launch_meta(const char* what, void (*one)(Args), void (*many)(Args), long long words, const Args& a,
                cudaStream_t stream) {
  const bool cluster = words > kClusterWords;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(cluster ? kCluster : 1);
  cfg.blockDim = dim3(kMetaThreads);
  cfg.stream = stream;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = kCluster;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = cluster ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, cluster ? many : one, a);
  return e == cudaSuccess ? H3SA_OK : set_cuda_error(what, e);
}

// Rows [0, rows) of each move's source page to its destination page, in every plane. Bound by
// memory: a warp takes 4 KB (16 rows of 256 bytes) at a time and has all of it in flight before
// it writes, eight warps a page side by side.
constexpr int kCopyBytes = 4096;
constexpr int kCopyThreads = 256;
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const Pools pools, const int4* moves,
                                                                  const int* n_moves) {
  // launched along with the ledger kernel, whose end it waits for here
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int planes = pools.count * pools.heads, lane = threadIdx.x & 31;
  const int parts = (kPage * pools.row_bytes + kCopyBytes - 1) / kCopyBytes;
  const long long items = static_cast<long long>(*n_moves) * planes * parts;
  const long long step = static_cast<long long>(gridDim.x) * (kCopyThreads / 32);
  for (long long i = static_cast<long long>(blockIdx.x) * (kCopyThreads / 32) + (threadIdx.x >> 5); i < items;
       i += step) {
    const long long page = i / parts;
    const int part = static_cast<int>(i - page * parts);
    const int plane = static_cast<int>(page % planes);
    const int4 mv = moves[page / planes];
    const int from = part * (kCopyBytes / 16) + lane, end = mv.z * (pools.row_bytes >> 4);
    if (part * (kCopyBytes / 16) >= end) continue;
    const size_t plane_rows = static_cast<size_t>(plane % pools.heads) * pools.pages * kPage;
    char* base = pools.base[plane / pools.heads];
    const uint4* src = reinterpret_cast<const uint4*>(base + (plane_rows + static_cast<size_t>(mv.x) * kPage) * pools.row_bytes);
    uint4* dst = reinterpret_cast<uint4*>(base + (plane_rows + static_cast<size_t>(mv.y) * kPage) * pools.row_bytes);
    uint4 v[kCopyBytes / 512];
#pragma unroll
    for (int k = 0; k < kCopyBytes / 512; ++k)
      if (from + 32 * k < end) v[k] = src[from + 32 * k];
#pragma unroll
    for (int k = 0; k < kCopyBytes / 512; ++k)
      if (from + 32 * k < end) dst[from + 32 * k] = v[k];
  }
}

constexpr int kCopyBlocks = 148 * 8;  // a full GPU at 256 threads a block

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
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(kCopyBlocks);
    cfg.blockDim = dim3(kCopyThreads);
    cfg.stream = stream;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = first == 0 ? 1 : 0;  // a second launch waits for the first one whole
    const cudaError_t e = cudaLaunchKernelEx(&cfg, copy_pages_kernel, p, moves, n_moves);
    if (e != cudaSuccess) return set_cuda_error("copy_pages_kernel launch", e);
  }
  return H3SA_OK;
}

// Loops run past the end of a table or a list by up to the threads of a cluster: what they count stays as
// much below 2^31.
constexpr int64_t kMaxEntries = INT32_MAX - 65536;
bool sizes_ok(int32_t sequences, int32_t width) {
  return sequences >= 0 && width > 0 && static_cast<int64_t>(width) * kPage <= INT32_MAX &&
         static_cast<int64_t>(sequences) * width <= kMaxEntries;
}

int check_pools(const char* what, const h3sa_pools* p) {
  if (!p || p->count < 0 || p->heads <= 0 || p->pages <= 0 || p->row_bytes <= 0 || p->row_bytes % 16 ||
      static_cast<int64_t>(p->row_bytes) * kPage > INT32_MAX)
    return set_error(H3SA_ERR_INVALID, "%s: invalid pools (row bytes must be a positive multiple of 16, below 2^24)",
                     what);
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
  // the moves come first (16 bytes each), then free pages or the page map, starts, the count of
  // moves, error bits and the blocks' slots
  return 16ll * pages + 4ll * pages + 4ll * children + 4ll * (2 + 2 * kCluster);
}

int h3sa_fork_pages(const h3sa_pools* pools, const int32_t* table, int32_t sequences, int32_t width,
                    const int32_t* lengths, const int32_t* refs, const int32_t* parents,
                    int32_t children, int32_t reserve_rows, int32_t private_copy,
                    int32_t* child_table, int32_t* child_lengths, int32_t* refs_out, void* workspace,
                    int32_t* device_error, void* stream) {
  int rc = check_pools("fork_pages", pools);
  if (rc) return rc;
  if (!sizes_ok(sequences, width) || !sizes_ok(children, width) || reserve_rows < 0)
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
  a.bad = a.n_moves + 1;
  a.slots = a.bad + 1;
  a.err = device_error;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = launch_meta("fork_kernel launch", fork_kernel<1>, fork_kernel<kCluster>,
                   static_cast<long long>(pools->pages) + 2ll * children * width, a, s);
  if (rc) return rc;
  return copy_launch(pools, a.moves, a.n_moves, s);
}

int h3sa_compact_pages(const h3sa_pools* pools, const int32_t* table, int32_t sequences, int32_t width,
                       const int32_t* refs, int32_t* table_out, int32_t* refs_out, int32_t* live,
                       void* workspace, int32_t* device_error, void* stream) {
  int rc = check_pools("compact_pages", pools);
  if (rc) return rc;
  if (!sizes_ok(sequences, width))
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
  a.slots = a.n_moves + 1;
  a.err = device_error;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = launch_meta("compact_kernel launch", compact_kernel<1>, compact_kernel<kCluster>,
                   static_cast<long long>(pools->pages) + a.entries, a, s);
  if (rc) return rc;
  return copy_launch(pools, a.moves, a.n_moves, s);
}

int h3sa_free_pages(const int32_t* table, int32_t sequences, int32_t width, const int32_t* lengths,
                    const int32_t* refs, int32_t pages, const uint8_t* release, int32_t* table_out,
                    int32_t* lengths_out, int32_t* refs_out, int32_t* device_error, void* stream) {
  if (!sizes_ok(sequences, width) || pages <= 0 || static_cast<int64_t>(pages) * kPage > INT32_MAX)
    return set_error(H3SA_ERR_INVALID, "free_pages: invalid sizes sequences=%d width=%d pages=%d", sequences,
                     width, pages);
  if ((sequences > 0 && (!table || !lengths || !release || !table_out || !lengths_out)) || !refs || !refs_out)
    return set_error(H3SA_ERR_INVALID, "free_pages: null pointer argument");
  FreeArgs a{table, lengths, refs, release, sequences, width, pages, table_out, lengths_out, refs_out, device_error};
  return launch_meta("free_kernel launch", free_kernel<1>, free_kernel<kCluster>,
                     static_cast<long long>(pages) + static_cast<long long>(sequences) * width, a,
                     static_cast<cudaStream_t>(stream));
}

}  // extern "C"
