// li4_fork.cu -- requests of a paged KV cache that go on from others, or end: tables, free pages, page copies, sm_100a.
//
// Which pages come back is a question about all tables at once: a page that a request lets go may be held by another, before
// the call and after it.  One cluster answers it in passes over the lines of held pages (a line: the pages of all requests,
// request after request, as prefix sums of their counts number them; a warp takes a run of a line):
//   1  owner[page] = none, everywhere, while the requests are read and their needs summed
//   2  owner[page] = 0 for every page that some request holds after the call, the least 1 + place on the line among
//      the requests that let it go otherwise (a minimum, so the order of threads does not matter); the entries that
//      requests take over are set aside, since the rows they come from may be written
//   3  a let-go entry whose place stands in owner is where a page comes back: counted, and by the warps' counts
//      before it numbered
//   4  those pages go on the stack, and the rows are written
// Bound by latency: trips to L2 one after another and cluster barriers between them.  A warp keeps its entries from pass 2 on
// where its run is short (kForkKept); otherwise it reads them again.
// A second launch copies the pages that are not full, bound by their bytes.
#include <cooperative_groups.h>

#include <algorithm>
#include <vector>

#include "li4_common.cuh"
#include "li4_internal.h"

namespace li4 {

namespace cg = cooperative_groups;

constexpr int kForkMaxRequests = 8192;
constexpr int kForkThreads = 512;
constexpr int kForkWarps = kForkThreads / 32;
constexpr int kForkCtas = 8;
constexpr int kForkKept = 4;  // groups of 32 entries of the line that a warp keeps
constexpr int kCopyThreads = 256;
constexpr int kCopyBytes = 8192;  // of a page that a CTA copies at a time

struct ForkArgs {
  const int* kv_lens;
  const int* parents;
  int* tables;
  int* free_pages;
  const int* n_free;
  long long table_stride;
  int B, width, log_page, capacity;
  int* kv_out;
  int* n_free_out;
  unsigned char* granted;
  unsigned* owner;   // [capacity]
  int* aside;        // [B * width] entries that requests take over, by place on the line of taken pages
  int* counts;       // [warps of the cluster]
  int2* copies;      // [B] (page, its copy)
  int* n_copies;
};

// Shared memory: by request, what happens to it.
struct ForkShared {
  int* source;  // [B] whose tokens it holds after the call (-1: none)
  int* old_at;  // [B + 1] first place on the line of pages held before
  int* take_at; // [B + 1] and on that of pages taken over
  int* fresh;   // [B] number of its page for the part of a page; -1: none
  int* len;     // [B] tokens it holds after the call
};

// Exclusive sums of three counts over the CTA's threads.
struct Counts3 {
  int a, b, c;
};
__device__ __forceinline__ Counts3 block_scan3(Counts3 v, Counts3* warp_sums, Counts3* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Counts3 s = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int x = __shfl_up_sync(0xffffffffu, s.a, d), y = __shfl_up_sync(0xffffffffu, s.b, d),
              z = __shfl_up_sync(0xffffffffu, s.c, d);
    if (lane >= d) s.a += x, s.b += y, s.c += z;
  }
  __syncthreads();  // (the sums of an earlier call have been read)
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  Counts3 base = {0, 0, 0}, all = {0, 0, 0};
  for (int w = 0; w < kForkWarps; ++w) {
    const Counts3 p = warp_sums[w];
    if (w < warp) base.a += p.a, base.b += p.b, base.c += p.c;
    all.a += p.a, all.b += p.b, all.c += p.c;
  }
  *total = all;
  return {base.a + s.a - v.a, base.b + s.b - v.b, base.c + s.c - v.c};
}

// Pages that a request holds; a length that does not fit its table holds what the table has.
__device__ __forceinline__ int held_pages(const ForkArgs& a, int len) {
  const int page = 1 << a.log_page;
  return len <= 0 ? 0 : (int)min((long long)a.width, ((long long)len + page - 1) >> a.log_page);
}
__device__ __forceinline__ bool fits(const ForkArgs& a, int len) {
  return len >= 0 && (long long)len <= ((long long)a.width << a.log_page);
}

// Calls f(request, block, place) for every entry of the warp's run of a line.  All lanes of a warp stay together: f is called
// with request -1 past the run's end.
template <typename F>
__device__ __forceinline__ void for_line(const int* at, int B, int warp, int warps, F&& f) {
  const int lane = threadIdx.x & 31;
  const long long total = at[B];
  const int from = (int)(total * warp / warps), to = (int)(total * (warp + 1) / warps);
  int r = 0;
  if (from < to) {  // the last request with at <= from
    int lo = 0, hi = B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (at[mid] <= from) lo = mid;
      else hi = mid;
    }
    r = lo;
  }
  for (int p0 = from; p0 < to; p0 += 32) {
    const int p = p0 + lane;
    if (p < to)
      while (at[r + 1] <= p) ++r;
    f(p < to ? r : -1, p < to ? p - at[r] : 0, p);
  }
}

__global__ void __launch_bounds__(kForkThreads) paged_fork_kernel(const __grid_constant__ ForkArgs a) {
  extern __shared__ int sm[];
  __shared__ Counts3 warp_sums[kForkWarps];
  ForkShared s;
  s.source = sm;
  s.old_at = s.source + a.B;
  s.take_at = s.old_at + a.B + 1;
  s.fresh = s.take_at + a.B + 1;
  s.len = s.fresh + a.B;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, rank = (int)cluster.block_rank(), C = (int)cluster.num_blocks();
  const int warp = rank * kForkWarps + (tid >> 5), warps = C * kForkWarps;
  const int page = 1 << a.log_page;
  pdl_launch_dependents();
  pdl_wait_primary();

  // ---- 1: no owner yet
  for (int p = rank * kForkThreads + tid; p < a.capacity; p += C * kForkThreads) a.owner[p] = 0xffffffffu;
  cluster.barrier_arrive();
  // ---- what happens to each request (every CTA works it out for itself)
  const int n_free = max(0, min(*a.n_free, a.capacity));
  const int per = (a.B + kForkThreads - 1) / kForkThreads;
  const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
  Counts3 sum = {0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    const int p = a.parents[b], own = a.kv_lens[b];
    const bool other = p >= 0 && p != b && p < a.B;
    const int len = other ? a.kv_lens[p] : p == b ? own : 0;
    const bool none = p < -1 || p >= a.B || (other && !fits(a, len));  // no request to go on from
    s.source[b] = none ? -2 : p;
    s.len[b] = len;
    s.old_at[b] = own;
    if (other && !none && (len & (page - 1)) != 0) ++sum.a;
  }
  Counts3 total;
  int wanted = block_scan3(sum, warp_sums, &total).a;  // pages asked for before this thread's requests
  sum = {0, 0, 0};
  for (int b = b0; b < b1; ++b) {
    const int p = s.source[b], len = s.len[b], own = s.old_at[b];
    const bool comes = p >= 0 && p != b;
    const bool part = comes && (len & (page - 1)) != 0;
    const bool ok = comes ? !part || wanted + 1 <= n_free : p != -2;
    s.source[b] = ok ? p : b;
    s.fresh[b] = ok && part ? wanted : -1;
    s.len[b] = ok ? len : own;
    if (part) ++wanted;
    s.old_at[b] = held_pages(a, own);
    s.take_at[b] = ok && comes ? held_pages(a, len) : 0;
    if (rank == 0) a.granted[b] = ok ? 1 : 0;
    sum.a += s.old_at[b];
    sum.b += s.take_at[b];
    sum.c += s.fresh[b] >= 0 ? 1 : 0;
  }
  const Counts3 before = block_scan3(sum, warp_sums, &total);
  {
    int x = before.a, y = before.b;
    for (int b = b0; b < b1; ++b) {
      const int n = s.old_at[b], m = s.take_at[b];
      s.old_at[b] = x;
      s.take_at[b] = y;
      x += n;
      y += m;
    }
  }
  if (tid == 0) {
    s.old_at[a.B] = total.a;
    s.take_at[a.B] = total.b;
  }
  const int taken = total.c;  // fresh pages: numbers 0 .. taken - 1 from the top of the stack
  const bool kept = total.a <= (long long)warps * kForkKept * 32 - warps;  // (the same for every warp)
  __syncthreads();
  cluster.barrier_wait();

  auto entry = [&](int r, int j) { return a.tables[(long long)r * a.table_stride + j]; };
  auto is_page = [&](int p) { return (unsigned)p < (unsigned)a.capacity; };
  // ---- 2: owners; what is taken over is set aside
  int mine[kForkKept];  // this lane's entries of requests that let them go; -1: none
#pragma unroll
  for (int i = 0; i < kForkKept; ++i) mine[i] = -1;
  const int run0 = (int)((long long)total.a * warp / warps);
  for_line(s.old_at, a.B, warp, warps, [&](int r, int j, int place) {
    if (r < 0) return;
    const int p = entry(r, j);
    if (!is_page(p)) return;
    if (s.source[r] == r) {
      a.owner[p] = 0;  // (no minimum is less)
    } else {
      atomicMin(a.owner + p, (unsigned)place + 1u);
#pragma unroll
      for (int i = 0; i < kForkKept; ++i)
        if ((place - run0) >> 5 == i) mine[i] = p;
    }
  });
  for_line(s.take_at, a.B, warp, warps, [&](int r, int j, int place) {
    if (r < 0) return;
    const int p = entry(s.source[r], j);
    const bool last = s.fresh[r] >= 0 && place + 1 == s.take_at[r + 1];
    if (last) {
      const int to = a.free_pages[n_free - 1 - s.fresh[r]];
      a.aside[place] = to;
      a.copies[s.fresh[r]] = make_int2(is_page(p) ? p : -1, is_page(to) ? to : -1);
    } else {
      a.aside[place] = p;
      if (is_page(p)) a.owner[p] = 0;
    }
  });
  cluster.sync();
  // ---- 3: how many come back in this warp's run
  auto comes_back = [&](int r, int j, int place) {
    if (r < 0 || s.source[r] == r) return -1;
    const int p = entry(r, j);
    return is_page(p) && a.owner[p] == (unsigned)place + 1u ? p : -1;
  };
  int back = 0;
  if (kept) {
    unsigned owner[kForkKept];
#pragma unroll
    for (int i = 0; i < kForkKept; ++i) owner[i] = mine[i] >= 0 ? a.owner[mine[i]] : 0u;
#pragma unroll
    for (int i = 0; i < kForkKept; ++i) {
      if (owner[i] != (unsigned)(run0 + 32 * i + lane) + 1u) mine[i] = -1;
      back += __popc(__ballot_sync(0xffffffffu, mine[i] >= 0));
    }
  } else {
    for_line(s.old_at, a.B, warp, warps,
             [&](int r, int j, int place) { back += __popc(__ballot_sync(0xffffffffu, comes_back(r, j, place) >= 0)); });
  }
  if (lane == 0) a.counts[warp] = back;
  cluster.sync();
  // ---- 4: onto the stack, in the line's order; then the rows
  int ahead = 0, all = 0;
  for (int w = lane; w < warps; w += 32) {
    const int n = a.counts[w];
    all += n;
    if (w < warp) ahead += n;
  }
  ahead = __reduce_add_sync(0xffffffffu, ahead);
  all = __reduce_add_sync(0xffffffffu, all);
  int height = n_free - taken + ahead;
  auto put = [&](int p) {
    const unsigned hit = __ballot_sync(0xffffffffu, p >= 0);
    const int at = height + __popc(hit & ((1u << lane) - 1u));
    if (p >= 0 && at < a.capacity) a.free_pages[at] = p;  // (a page on the stack twice is the caller's mistake)
    height += __popc(hit);
  };
  if (kept) {
#pragma unroll
    for (int i = 0; i < kForkKept; ++i) put(mine[i]);
  } else {
    for_line(s.old_at, a.B, warp, warps, [&](int r, int j, int place) { put(comes_back(r, j, place)); });
    cluster.sync();  // the rows have been read
  }
  for_line(s.take_at, a.B, warp, warps, [&](int r, int j, int place) {
    if (r >= 0) a.tables[(long long)r * a.table_stride + j] = a.aside[place];
  });
  if (rank == 0) {
    // (kv_out and n_free_out may be the inputs: every CTA has read those before it arrived at the barrier that ends pass 2)
    for (int b = tid; b < a.B; b += kForkThreads) a.kv_out[b] = s.len[b];
    if (tid == 0) {
      *a.n_free_out = min(a.capacity, n_free - taken + all);
      *a.n_copies = taken;
    }
  }
}

struct CopyArgs {
  const int2* copies;
  const int* n_copies;
  int n_pools;
  uint8_t* pool[LI4_FORK_POOLS];
  long long stride[LI4_FORK_POOLS];
  int pieces_at[LI4_FORK_POOLS + 1];  // pieces of kCopyBytes of a page in the pools before
  long long bytes[LI4_FORK_POOLS];
};

// A page's piece of kCopyBytes in a pool at a time.
__global__ void __launch_bounds__(kCopyThreads) paged_copy_kernel(const __grid_constant__ CopyArgs a) {
  pdl_launch_dependents();
  pdl_wait_primary();
  const int pieces = a.pieces_at[a.n_pools];
  const long long total = (long long)*a.n_copies * pieces;
  for (long long i = blockIdx.x; i < total; i += gridDim.x) {
    const int c = (int)(i / pieces), piece = (int)(i - (long long)c * pieces);
    int lo = 0, hi = a.n_pools;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.pieces_at[mid] <= piece) lo = mid;
      else hi = mid;
    }
    const int2 pages = a.copies[c];
    if (pages.x < 0 || pages.y < 0) continue;
    const long long at = (long long)(piece - a.pieces_at[lo]) * kCopyBytes;
    const int n = (int)(min((long long)kCopyBytes, a.bytes[lo] - at) / 16);
    const uint4* from = reinterpret_cast<const uint4*>(a.pool[lo] + pages.x * a.stride[lo] + at);
    uint4* to = reinterpret_cast<uint4*>(a.pool[lo] + pages.y * a.stride[lo] + at);
    uint4 v[kCopyBytes / 16 / kCopyThreads];
#pragma unroll
    for (int e = 0; e < kCopyBytes / 16 / kCopyThreads; ++e)
      if (e * kCopyThreads + (int)threadIdx.x < n) v[e] = from[e * kCopyThreads + threadIdx.x];
#pragma unroll
    for (int e = 0; e < kCopyBytes / 16 / kCopyThreads; ++e)
      if (e * kCopyThreads + (int)threadIdx.x < n) to[e * kCopyThreads + threadIdx.x] = v[e];
  }
}

template <typename KernelT, typename ArgsT>
static int launch_fork(KernelT kernel, const ArgsT& a, unsigned grid, int threads, size_t smem, int cluster,
                       cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, a), "paged_fork: kernel launch");
}

static size_t fork_shared_bytes(int64_t B) { return (size_t)(5 * B + 2) * sizeof(int); }

// Workspace: copies, owner, aside, counts and the number of copies.
struct ForkSpace {
  size_t owner, aside, counts, n_copies, bytes;
};
static ForkSpace fork_space(int64_t B, int64_t width, int64_t capacity) {
  ForkSpace s;
  s.owner = (size_t)B * sizeof(int2);
  s.aside = s.owner + (size_t)capacity * sizeof(unsigned);
  s.counts = s.aside + (size_t)B * width * sizeof(int);
  s.n_copies = s.counts + kForkCtas * kForkWarps * sizeof(int);
  s.bytes = s.n_copies + sizeof(int);
  return s;
}

// ---- memory that a call may not name twice
// rows of `bytes` bytes, `stride` apart
struct Region {
  const char* name;
  uintptr_t at;
  int64_t rows, stride, bytes;
};
static Region region(const char* name, const void* p, int64_t bytes, int64_t rows = 1, int64_t stride = 0) {
  return {name, reinterpret_cast<uintptr_t>(p), bytes > 0 ? rows : 0, stride, bytes};
}
static int64_t span(const Region& r) { return r.rows > 0 ? (r.rows - 1) * r.stride + r.bytes : 0; }

// Whether one of a's rows meets b's span.
static bool meet(const Region& a, const Region& b) {
  if (a.rows <= 0 || b.rows <= 0) return false;
  const int64_t off = (int64_t)(b.at - a.at), n = span(b);  // b from a's start
  if (off + n <= 0 || off >= span(a)) return false;
  if (off < 0 || a.rows == 1) return true;
  const int64_t row = off / a.stride;
  return off - row * a.stride < a.bytes || (row + 1 < a.rows && off + n > (row + 1) * a.stride);
}

// Whether a page of one pool lies over a page of another number of another pool: a copy into one would then change the
// other.  (The same pages named twice are copied twice.)  The ranges are sorted; those that meet have to be interleaved: of one
// stride, and modulo it apart or at the same page.
static bool pools_meet(void* const* pools, const int64_t* strides, const int64_t* bytes, int64_t n_pools, int64_t pages) {
  struct Pool {
    uintptr_t at;
    int64_t stride, bytes;
    uintptr_t end(int64_t n) const { return at + (uintptr_t)((n - 1) * stride + bytes); }
  };
  std::vector<Pool> all;
  all.reserve((size_t)n_pools);
  for (int64_t i = 0; i < n_pools; ++i)
    if (bytes[i] > 0) all.push_back({reinterpret_cast<uintptr_t>(pools[i]), strides[i], bytes[i]});
  std::sort(all.begin(), all.end(), [](const Pool& a, const Pool& b) { return a.at < b.at; });
  struct Piece {
    int64_t at, end, page;
  };
  std::vector<Piece> pieces;
  for (size_t i = 0, next; i < all.size(); i = next) {
    uintptr_t end = all[i].end(pages);
    for (next = i + 1; next < all.size() && all[next].at < end; ++next) {
      if (all[next].stride != all[i].stride) return true;
      end = std::max(end, all[next].end(pages));
    }
    if (next == i + 1) continue;
    // two strides' worth: every pool's page `page` of the first stride and the page after it in the second
    const int64_t stride = all[i].stride;
    pieces.clear();
    for (size_t k = i; k < next; ++k) {
      const int64_t off = (int64_t)(all[k].at - all[i].at), at = off % stride;
      for (int lap = 0; lap < 2; ++lap)
        pieces.push_back({at + lap * stride, at + lap * stride + all[k].bytes, lap - off / stride});
    }
    std::sort(pieces.begin(), pieces.end(), [](const Piece& a, const Piece& b) { return a.at < b.at; });
    Piece last = pieces[0];
    for (const Piece& p : pieces) {
      if (p.at < last.end && p.page != last.page) return true;
      if (p.end > last.end) last = p;
    }
  }
  return false;
}

}  // namespace li4

extern "C" size_t li4_paged_fork_workspace_bytes(int64_t n_requests, int64_t table_width, int64_t free_capacity) {
  if (n_requests <= 0 || n_requests > li4::kForkMaxRequests || table_width < 0 || free_capacity < 0 ||
      free_capacity > (1 << 30) || table_width > 0x7fffffffLL / n_requests)
    return 0;
  return li4::fork_space(n_requests, table_width, free_capacity).bytes;
}

extern "C" int li4_paged_fork(const int32_t* kv_lens, const int32_t* parents, int64_t n_requests, int32_t* block_tables,
                              int64_t table_stride, int64_t table_width, int32_t* free_pages, int64_t free_capacity,
                              const int32_t* n_free, int64_t page_size, int32_t* kv_lens_out, int32_t* n_free_out,
                              uint8_t* granted, void* const* pools, const int64_t* pool_strides,
                              const int64_t* pool_bytes, int64_t n_pools, void* workspace, size_t workspace_bytes,
                              void* stream) {
  using namespace li4;
  const char* what = "paged_fork";
  constexpr int64_t kMostBytes = 1LL << 60;  // (so that no span of a table or pool overflows)
  if (n_requests < 0 || table_width < 0 || free_capacity < 0 || table_stride < table_width || n_pools < 0 ||
      (n_requests > 1 && table_stride > kMostBytes / 4 / n_requests))
    return set_error(LI4_ERR_INVALID_ARG,
                     "%s: n_requests=%lld table_width=%lld table_stride=%lld free_capacity=%lld n_pools=%lld", what,
                     (long long)n_requests, (long long)table_width, (long long)table_stride, (long long)free_capacity,
                     (long long)n_pools);
  if (!is_pow2(page_size) || page_size < 8 || page_size > 1024)
    return set_error(LI4_ERR_UNSUPPORTED, "%s: page_size=%lld (a power of two from 8 to 1024)", what,
                     (long long)page_size);
  if (n_requests > kForkMaxRequests)
    return set_error(LI4_ERR_UNSUPPORTED, "%s: n_requests=%lld (at most %d)", what, (long long)n_requests,
                     kForkMaxRequests);
  if (free_capacity > (1 << 30) || (n_requests > 0 && table_width > 0x7fffffffLL / n_requests))
    return set_error(LI4_ERR_UNSUPPORTED, "%s: tables of %lld x %lld entries, %lld pages", what, (long long)n_requests,
                     (long long)table_width, (long long)free_capacity);
  if (!n_free || !n_free_out || (free_capacity > 0 && !free_pages) ||
      (n_requests > 0 && (!kv_lens || !parents || !kv_lens_out || !granted || (table_width > 0 && !block_tables))) ||
      (n_pools > 0 && (!pools || !pool_strides || !pool_bytes)))
    return set_error(LI4_ERR_INVALID_ARG, "%s: null pointer", what);
  for (int64_t i = 0; i < n_pools; ++i) {
    if ((!pools[i] && free_capacity > 0) || !aligned16(pools[i]) || pool_bytes[i] % 16 != 0 || pool_strides[i] % 16 != 0)
      return set_error(LI4_ERR_ALIGNMENT, "%s: pool %lld: pages must start on 16-byte boundaries, of a multiple of 16 bytes",
                       what, (long long)i);
    if (pool_bytes[i] < 0 || pool_bytes[i] > (1 << 30) || (pool_strides[i] < pool_bytes[i] && free_capacity > 1) ||
        (free_capacity > 1 && pool_strides[i] > kMostBytes / free_capacity))
      return set_error(LI4_ERR_INVALID_ARG, "%s: pool %lld: pages of %lld bytes, %lld apart", what, (long long)i,
                       (long long)pool_bytes[i], (long long)pool_strides[i]);
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (n_requests == 0) {
    if (n_free_out != n_free) {
      const int rc = check_cuda(cudaMemcpyAsync(n_free_out, n_free, sizeof(int32_t), cudaMemcpyDeviceToDevice, st),
                                "paged_fork: copy");
      if (rc != LI4_OK) return rc;
    }
    clear_error();
    return LI4_OK;
  }
  const ForkSpace space = fork_space(n_requests, table_width, free_capacity);
  if (!workspace || workspace_bytes < space.bytes || !aligned16(workspace))
    return set_error(LI4_ERR_WORKSPACE, "%s: %zu bytes of 16-byte aligned workspace needed, %zu given", what, space.bytes,
                     workspace_bytes);
  const Region tables = region("block_tables", block_tables, table_width * 4, n_requests, table_stride * 4);
  const Region written[5] = {tables, region("free_pages", free_pages, free_capacity * 4), region("kv_lens_out", kv_lens_out, n_requests * 4),
                             region("n_free_out", n_free_out, 4), region("granted", granted, n_requests)};
  const Region read[3] = {region("kv_lens", kv_lens, n_requests * 4), region("parents", parents, n_requests * 4),
                          region("n_free", n_free, 4)};
  for (int i = 0; i < 5; ++i) {
    for (int k = i + 1; k < 5; ++k)
      if (meet(written[i], written[k]))
        return set_error(LI4_ERR_INVALID_ARG, "%s: %s must not overlap %s", what, written[k].name, written[i].name);
    for (int k = 0; k < 3; ++k)
      if (meet(written[i], read[k]) && !(read[k].at == written[i].at && ((i == 2 && k == 0) || (i == 3 && k == 2))))
        return set_error(LI4_ERR_INVALID_ARG, "%s: %s must not overlap %s", what, written[i].name, read[k].name);
  }
  if (free_capacity > 0) {
    for (int64_t p = 0; p < n_pools; ++p) {
      const Region pool = region("a pool", pools[p], pool_bytes[p], free_capacity, pool_strides[p]);
      for (int i = 0; i < 8; ++i) {
        const Region& other = i < 5 ? written[i] : read[i - 5];
        if (meet(pool, other)) return set_error(LI4_ERR_INVALID_ARG, "%s: pool %lld must not overlap %s", what, (long long)p, other.name);
      }
    }
    try {
      if (pools_meet(pools, pool_strides, pool_bytes, n_pools, free_capacity))
        return set_error(LI4_ERR_INVALID_ARG, "%s: pages of one pool must not overlap other pages of another", what);
    } catch (...) {  // (no exception leaves a C function)
      return set_error(LI4_ERR_INVALID_ARG, "%s: no host memory for %lld pools", what, (long long)n_pools);
    }
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  ForkArgs a;
  a.kv_lens = kv_lens;
  a.parents = parents;
  a.tables = block_tables;
  a.free_pages = free_pages;
  a.n_free = n_free;
  a.table_stride = table_stride;
  a.B = (int)n_requests;
  a.width = (int)table_width;
  a.log_page = ilog2(page_size);
  a.capacity = (int)free_capacity;
  a.kv_out = kv_lens_out;
  a.n_free_out = n_free_out;
  a.granted = granted;
  a.copies = reinterpret_cast<int2*>(ws);
  a.owner = reinterpret_cast<unsigned*>(ws + space.owner);
  a.aside = reinterpret_cast<int*>(ws + space.aside);
  a.counts = reinterpret_cast<int*>(ws + space.counts);
  a.n_copies = reinterpret_cast<int*>(ws + space.n_copies);
  const size_t smem = fork_shared_bytes(n_requests);
  if (smem > 40 * 1024) {
    const int rc = check_cuda(cudaFuncSetAttribute(paged_fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)fork_shared_bytes(kForkMaxRequests)),
                              "paged_fork: shared memory limit");
    if (rc != LI4_OK) return rc;
  }
  int rc = launch_fork(paged_fork_kernel, a, kForkCtas, kForkThreads, smem, kForkCtas, st);
  CopyArgs c;
  c.copies = a.copies;
  c.n_copies = a.n_copies;
  for (int64_t p = 0; rc == LI4_OK && p < n_pools; p += LI4_FORK_POOLS) {
    c.n_pools = (int)(n_pools - p < LI4_FORK_POOLS ? n_pools - p : LI4_FORK_POOLS);
    c.pieces_at[0] = 0;
    for (int i = 0; i < c.n_pools; ++i) {
      c.pool[i] = static_cast<uint8_t*>(pools[p + i]);
      c.stride[i] = pool_strides[p + i];
      c.bytes[i] = pool_bytes[p + i];
      c.pieces_at[i + 1] = c.pieces_at[i] + (int)((pool_bytes[p + i] + kCopyBytes - 1) / kCopyBytes);
    }
    const int64_t most = n_requests * c.pieces_at[c.n_pools], fill = 8LL * current_sm_count();
    if (most > 0)
      rc = launch_fork(paged_copy_kernel, c, (unsigned)(most < fill ? most : fill), kCopyThreads, 0, 1, st);
  }
  if (rc == LI4_OK) clear_error();
  return rc;
}
