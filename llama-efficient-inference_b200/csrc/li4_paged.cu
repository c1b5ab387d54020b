// li4_paged.cu -- one serving step's bookkeeping over a paged KV cache, and the cache write, sm_100a.
//
// li4_paged_append: the requests' lengths -> pages for the new tokens, block tables, positions, slots.
// li4_rope_paged_write: RoPE on the packed queries and keys, keys and values into their slots.
#include <cooperative_groups.h>

#include "li4_common.cuh"
#include "li4_internal.h"

namespace li4 {

namespace cg = cooperative_groups;

__device__ unsigned g_paged_device_error;  // bit 7 of li4_device_errors

int paged_device_errors(unsigned* flags, bool reset) {
  int rc = check_cuda(cudaMemcpyFromSymbol(flags, g_paged_device_error, sizeof(unsigned)), "device_errors: paged");
  if (rc == LI4_OK && reset) {
    const unsigned zero = 0;
    rc = check_cuda(cudaMemcpyToSymbol(g_paged_device_error, &zero, sizeof(unsigned)), "device_errors: clearing");
  }
  return rc;
}

// ---------------------------------------------------------------------------
// Append.  Request b holds c_b tokens and gets n_b more: it needs ceil((c_b + n_b) / P) -
// ceil(c_b / P) fresh pages.  The fresh pages of the step are numbered in request order, then block
// order, and number k is the k-th from the top of the free stack, so an exclusive prefix sum of the
// needs places every page with no atomic and no order between threads.  Block j of a request is
// fresh exactly where its first token j P is one of the new ones, so the token at a block's start
// writes its table entry and every thread works on tokens alone.
//
// Each CTA of the launch's one cluster repeats the (cheap) prefix sums over the requests and then
// takes every C-th block of tokens; the cluster barrier stands between everyone's reads of the
// lengths and the first CTA's writes, so the outputs may be the inputs (kv_lens, n_free).
// Bound by latency: three dependent trips to L2 (lengths, free page or table entry, stores).
// ---------------------------------------------------------------------------
constexpr int kAppendMaxRequests = 8192;  // 12 bytes of shared memory each
constexpr int kAppendMaxLen = 1 << 30;

struct AppendArgs {
  const int* kv_lens;
  const int* new_lens;
  int* tables;
  const int* free_pages;
  const int* n_free;
  long long table_stride;
  int B, width, log_page, capacity, T;
  int max_len;     // no request grows past it
  int* cu;
  int* positions;
  long long* slots;
  int* kv_out;
  int* n_free_out;
  unsigned char* granted;
  int vector_out;  // positions and slots start on 16-byte boundaries
};

// Sums of 64 bits: the lengths are the caller's, and a wrong one must not wrap into a grant.
struct Sums {
  long long tokens, pages;
};
template <int THREADS>
__device__ __forceinline__ Sums block_scan2(Sums v, Sums* warp_sums, Sums* total) {  // exclusive, over the CTA
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Sums s = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long x = __shfl_up_sync(0xffffffffu, s.tokens, d), y = __shfl_up_sync(0xffffffffu, s.pages, d);
    if (lane >= d) {
      s.tokens += x;
      s.pages += y;
    }
  }
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  Sums base = {0, 0}, all = {0, 0};
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    const Sums p = warp_sums[w];
    if (w < warp) {
      base.tokens += p.tokens;
      base.pages += p.pages;
    }
    all.tokens += p.tokens;
    all.pages += p.pages;
  }
  *total = all;
  return {base.tokens + s.tokens - v.tokens, base.pages + s.pages - v.pages};
}

// The step of one request: its lengths, checked, and the fresh pages it asks for.
__device__ __forceinline__ bool append_request(const AppendArgs& a, int b, int* c, int* n, int* need) {
  const int page = 1 << a.log_page;
  *c = a.kv_lens[b];
  *n = a.new_lens[b];
  const bool sane = *c >= 0 && *n >= 0 && *c <= kAppendMaxLen - *n;
  if (!sane) {
    *n = max(0, min(*n, a.T));
    *need = 0;
    return false;
  }
  const int want = (*c + *n + page - 1) >> a.log_page, held = (*c + page - 1) >> a.log_page;
  const bool fits = want <= a.width && *c + *n <= a.max_len;
  *need = fits ? want - held : 0;
  return fits;
}

// TOK tokens in a row per thread: one search for the first, then on from request to request.
template <int THREADS, int TOK>
__global__ void __launch_bounds__(THREADS) paged_append_kernel(const __grid_constant__ AppendArgs a) {
  extern __shared__ int sm[];
  int* s_cu = sm;                // [B + 1] first token of each request
  int* s_ctx = s_cu + a.B + 1;   // [B] tokens held before the step
  int* s_rank = s_ctx + a.B;     // [B] number of the request's first fresh page; -1: refused
  __shared__ Sums warp_sums[THREADS / 32];
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, rank = (int)cluster.block_rank(), C = (int)cluster.num_blocks();
  const int page = 1 << a.log_page;
  pdl_launch_dependents();
  pdl_wait_primary();

  const int n_free = max(0, min(*a.n_free, a.capacity));
  const int per = (a.B + THREADS - 1) / THREADS;
  const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
  Sums sum = {0, 0};
  for (int b = b0; b < b1; ++b) {
    int c, n, need;
    append_request(a, b, &c, &n, &need);
    sum.tokens += n;
    sum.pages += need;
  }
  Sums total;
  Sums at = block_scan2<THREADS>(sum, warp_sums, &total);
  int taken = 0;
  for (int b = b0; b < b1; ++b) {
    int c, n, need;
    const bool fits = append_request(a, b, &c, &n, &need);
    // granted: the table is wide enough, the length allowed, the pages are there, the tokens are among the step's T
    const bool ok = fits && (need == 0 || at.pages + need <= n_free) && at.tokens + n <= a.T;
    s_cu[b] = (int)min(at.tokens, 0x7fffffffLL);
    s_ctx[b] = c;
    s_rank[b] = !ok ? -1 : need == 0 ? 0 : (int)at.pages;
    if (ok) taken += need;
    at.tokens += n;
    at.pages += need;
  }
  if (tid == 0) s_cu[a.B] = (int)min(total.tokens, 0x7fffffffLL);
  if (C > 1) cluster.sync();  // everyone has read the lengths and the stack's height
  else __syncthreads();
  if (rank == 0) {
    for (int b = tid; b <= a.B; b += THREADS) a.cu[b] = s_cu[b];
    for (int b = tid; b < a.B; b += THREADS) {
      const int n = s_cu[b + 1] - s_cu[b];
      a.granted[b] = s_rank[b] >= 0 ? 1 : 0;
      a.kv_out[b] = s_rank[b] >= 0 ? s_ctx[b] + n : s_ctx[b];
    }
    __syncthreads();
    block_scan2<THREADS>({0, taken}, warp_sums, &total);
    if (tid == 0) *a.n_free_out = n_free - (int)total.pages;
  }
  const int used = min(s_cu[a.B], a.T);
  const bool wide = a.vector_out != 0;
  for (int t0 = (rank * THREADS + tid) * TOK; t0 < a.T; t0 += C * THREADS * TOK) {
    int pos[TOK];
    long long slot[TOK];
#pragma unroll
    for (int i = 0; i < TOK; ++i) pos[i] = 0, slot[i] = -1;
    if (t0 < used) {
      int lo = 0, hi = a.B;  // the last request with cu <= t0 (requests of no tokens share their start)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= t0) lo = mid;
        else hi = mid;
      }
      const int* from[TOK];  // where the token's page stands
      bool ok[TOK], fresh[TOK];
#pragma unroll
      for (int i = 0; i < TOK; ++i) {
        const int t = t0 + i;
        ok[i] = t < used;
        from[i] = a.n_free;  // (not used where !ok)
        fresh[i] = false;
        if (!ok[i]) continue;
        while (s_cu[lo + 1] <= t) ++lo;
        const int c = s_ctx[lo], first = s_rank[lo];
        pos[i] = c + t - s_cu[lo];
        ok[i] = first >= 0;
        if (!ok[i]) continue;
        const int block = pos[i] >> a.log_page, held = (c + page - 1) >> a.log_page;
        int* entry = a.tables + (long long)lo * a.table_stride + block;
        fresh[i] = block >= held;
        from[i] = fresh[i] ? a.free_pages + (n_free - 1 - (first + block - held)) : entry;
        if (fresh[i] && (pos[i] & (page - 1)) == 0) *entry = *from[i];
      }
#pragma unroll
      for (int i = 0; i < TOK; ++i)
        if (ok[i]) slot[i] = ((long long)*from[i] << a.log_page) + (pos[i] & (page - 1));
    }
    if (TOK == 4 && wide && t0 + 4 <= a.T) {
      *reinterpret_cast<int4*>(a.positions + t0) = make_int4(pos[0], pos[1 % TOK], pos[2 % TOK], pos[3 % TOK]);
      *reinterpret_cast<longlong2*>(a.slots + t0) = make_longlong2(slot[0], slot[1 % TOK]);
      *reinterpret_cast<longlong2*>(a.slots + t0 + 2) = make_longlong2(slot[2 % TOK], slot[3 % TOK]);
    } else {
      for (int i = 0; i < TOK && t0 + i < a.T; ++i) {
        a.positions[t0 + i] = pos[i];
        a.slots[t0 + i] = slot[i];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// RoPE and cache write.  Pairs (x0, x1) = (x[2i], x[2i + 1]) turn by the table's angle of their
// token's position, (x0 c - x1 s, x0 s + x1 c) in fp32, rounded once; values are copied.  A thread
// owns 8 consecutive dims of one token: it reads the 4 + 4 table values once and walks over a group
// of the token's heads, so the table costs 1 / heads of the traffic.  Bound by HBM.
// ---------------------------------------------------------------------------
constexpr int kRopeThreads = 256;

struct RopeArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* q_out;
  uint16_t* k_out;  // may be null
  long long sqt, sqh, skt, skh, svt, svh, sqot, sqoh, skot, skoh;
  const float* cos;
  const float* sin;
  long long srope;
  const int* positions;
  const long long* slots;
  uint16_t* cache_k;
  uint16_t* cache_v;
  long long sckp, sckr, sckh, scvp, scvr, scvh;
  long long num_slots;
  int T, H, Hkv, chunks, log_page, max_pos, heads_per_group;
};

template <typename T2>
struct Pair;
template <>
struct Pair<__half2> {
  static __device__ __forceinline__ float2 load(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
  static __device__ __forceinline__ uint32_t store(float x, float y) {
    __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
template <>
struct Pair<__nv_bfloat162> {
  static __device__ __forceinline__ float2 load(uint32_t u) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
  }
  static __device__ __forceinline__ uint32_t store(float x, float y) {
    __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};

template <typename T2>
__device__ __forceinline__ uint4 turn8(uint4 x, const float4& c, const float4& s) {
  const float2 a = Pair<T2>::load(x.x), b = Pair<T2>::load(x.y), d = Pair<T2>::load(x.z), e = Pair<T2>::load(x.w);
  return make_uint4(Pair<T2>::store(a.x * c.x - a.y * s.x, a.x * s.x + a.y * c.x),
                    Pair<T2>::store(b.x * c.y - b.y * s.y, b.x * s.y + b.y * c.y),
                    Pair<T2>::store(d.x * c.z - d.y * s.z, d.x * s.z + d.y * c.z),
                    Pair<T2>::store(e.x * c.w - e.y * s.w, e.x * s.w + e.y * c.w));
}

template <typename F>
__device__ __forceinline__ void for_heads(int h0, int h1, const uint16_t* src, long long stride, F&& put) {
  for (int h = h0; h < h1; h += 4) {
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (h + i < h1) x[i] = *reinterpret_cast<const uint4*>(src + (long long)(h + i) * stride);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (h + i < h1) put(h + i, x[i]);
  }
}

template <typename T2>
__global__ void __launch_bounds__(kRopeThreads) rope_paged_write_kernel(const __grid_constant__ RopeArgs a) {
  pdl_launch_dependents();
  pdl_wait_primary();
  const long long i = (long long)blockIdx.x * kRopeThreads + threadIdx.x;
  const long long t = i / a.chunks;
  if (t >= a.T) return;
  const int d = (int)(i - t * a.chunks) * 8;
  int pos = a.positions[t];
  const long long slot = a.slots[t];
  // (a token that is skipped may stand anywhere: li4_paged_append refuses a request at the table's end like any other)
  if (slot >= a.num_slots || (slot >= 0 && (pos < 0 || pos >= a.max_pos))) atomicOr(&g_paged_device_error, 128u);
  pos = max(0, min(pos, a.max_pos - 1));
  const bool keep = slot >= 0 && slot < a.num_slots;
  const long long page = keep ? slot >> a.log_page : 0, row = keep ? slot & ((1 << a.log_page) - 1) : 0;
  const float4 c = *reinterpret_cast<const float4*>(a.cos + (long long)pos * a.srope + d / 2);
  const float4 s = *reinterpret_cast<const float4*>(a.sin + (long long)pos * a.srope + d / 2);
  const int h0 = blockIdx.y * a.heads_per_group, h1 = min(a.H + 2 * a.Hkv, h0 + a.heads_per_group);
  uint16_t* ck = a.cache_k + page * a.sckp + row * a.sckr + d;
  uint16_t* cv = a.cache_v + page * a.scvp + row * a.scvr + d;
  // four heads at a time: their loads are under way together (one at a time, 16381 tokens took 95 us instead of 75)
  for_heads(h0, min(h1, a.H), a.q + t * a.sqt + d, a.sqh, [&](int h, uint4 x) {
    *reinterpret_cast<uint4*>(a.q_out + t * a.sqot + (long long)h * a.sqoh + d) = turn8<T2>(x, c, s);
  });
  for_heads(max(h0 - a.H, 0), min(h1 - a.H, a.Hkv), a.k + t * a.skt + d, a.skh, [&](int h, uint4 x) {
    const uint4 y = turn8<T2>(x, c, s);
    if (a.k_out) *reinterpret_cast<uint4*>(a.k_out + t * a.skot + (long long)h * a.skoh + d) = y;
    if (keep) *reinterpret_cast<uint4*>(ck + (long long)h * a.sckh) = y;
  });
  if (keep)
    for_heads(max(h0 - a.H - a.Hkv, 0), h1 - a.H - a.Hkv, a.v + t * a.svt + d, a.svh,
              [&](int h, uint4 x) { *reinterpret_cast<uint4*>(cv + (long long)h * a.scvh) = x; });
}

template <typename KernelT, typename ArgsT>
static int launch_pdl(KernelT kernel, const ArgsT& a, dim3 grid, int threads, size_t smem, int cluster,
                      cudaStream_t stream, const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
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
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, a), what);
}

template <int THREADS, int TOK>
static int launch_append(const AppendArgs& a, int cluster, cudaStream_t stream) {
  const size_t smem = (3 * (size_t)a.B + 1) * sizeof(int);
  if (smem > 40 * 1024) {
    const int rc = check_cuda(cudaFuncSetAttribute(paged_append_kernel<THREADS, TOK>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)((3 * kAppendMaxRequests + 1) * sizeof(int))),
                              "paged_append: shared memory limit");
    if (rc != LI4_OK) return rc;
  }
  return launch_pdl(paged_append_kernel<THREADS, TOK>, a, dim3((unsigned)cluster), THREADS, smem, cluster, stream,
                    "paged_append: kernel launch");
}

}  // namespace li4

extern "C" int li4_paged_append(const int32_t* kv_lens, const int32_t* new_lens, int64_t n_requests,
                                int32_t* block_tables, int64_t table_stride, int64_t table_width,
                                const int32_t* free_pages, int64_t free_capacity, const int32_t* n_free,
                                int64_t page_size, int64_t n_tokens, int32_t* cu_seqlens, int32_t* positions,
                                int64_t* slots, int32_t* kv_lens_out, int32_t* n_free_out, uint8_t* granted,
                                void* stream) {
  return li4_paged_append_within(kv_lens, new_lens, n_requests, block_tables, table_stride, table_width, free_pages,
                                 free_capacity, n_free, page_size, n_tokens, li4::kAppendMaxLen, cu_seqlens, positions,
                                 slots, kv_lens_out, n_free_out, granted, stream);
}

extern "C" int li4_paged_append_within(const int32_t* kv_lens, const int32_t* new_lens, int64_t n_requests,
                                       int32_t* block_tables, int64_t table_stride, int64_t table_width,
                                       const int32_t* free_pages, int64_t free_capacity, const int32_t* n_free,
                                       int64_t page_size, int64_t n_tokens, int64_t max_len, int32_t* cu_seqlens,
                                       int32_t* positions, int64_t* slots, int32_t* kv_lens_out, int32_t* n_free_out,
                                       uint8_t* granted, void* stream) {
  using namespace li4;
  if (n_requests < 0 || table_width < 0 || free_capacity < 0 || n_tokens < 0 || table_stride < table_width)
    return set_error(LI4_ERR_INVALID_ARG,
                     "paged_append: n_requests=%lld table_width=%lld table_stride=%lld free_capacity=%lld n_tokens=%lld",
                     (long long)n_requests, (long long)table_width, (long long)table_stride, (long long)free_capacity,
                     (long long)n_tokens);
  if (!is_pow2(page_size) || page_size < 8 || page_size > 1024)
    return set_error(LI4_ERR_UNSUPPORTED, "paged_append: page_size=%lld (a power of two from 8 to 1024)",
                     (long long)page_size);
  if (n_requests > kAppendMaxRequests)
    return set_error(LI4_ERR_UNSUPPORTED, "paged_append: n_requests=%lld (at most %d)", (long long)n_requests,
                     kAppendMaxRequests);
  if (max_len < 0) return set_error(LI4_ERR_INVALID_ARG, "paged_append: max_len=%lld", (long long)max_len);
  if (n_tokens > kAppendMaxLen || free_capacity > kAppendMaxLen || table_width > kAppendMaxLen)
    return set_error(LI4_ERR_INVALID_ARG, "paged_append: sizes above 2^30");
  if (!n_free || !cu_seqlens || !n_free_out ||
      (n_requests > 0 && (!kv_lens || !new_lens || !kv_lens_out || !granted)) ||
      (n_tokens > 0 && (!positions || !slots)) || (n_requests > 0 && table_width > 0 && !block_tables) ||
      (free_capacity > 0 && !free_pages))
    return set_error(LI4_ERR_INVALID_ARG, "paged_append: null pointer");
  AppendArgs a;
  a.kv_lens = kv_lens;
  a.new_lens = new_lens;
  a.tables = block_tables;
  a.free_pages = free_pages;
  a.n_free = n_free;
  a.table_stride = table_stride;
  a.B = (int)n_requests;
  a.width = (int)table_width;
  a.log_page = ilog2(page_size);
  a.capacity = (int)free_capacity;
  a.T = (int)n_tokens;
  a.max_len = (int)(max_len < kAppendMaxLen ? max_len : kAppendMaxLen);
  a.cu = cu_seqlens;
  a.positions = positions;
  a.slots = reinterpret_cast<long long*>(slots);
  a.kv_out = kv_lens_out;
  a.n_free_out = n_free_out;
  a.granted = granted;
  a.vector_out = aligned16(positions) && aligned16(slots);
  // few tokens: one CTA, a token per thread; many: a cluster of eight, four per thread.  The one / the other, us: 64
  // requests of a token 2.9 / 4.1, 512 tokens of 64 requests 3.5 / 3.9, of 512 requests 4.2 / 4.9, 1000 of 64 requests
  // 5.9 / 4.5, 1024 of 1024 requests 6.2 / 5.7, 2000 of 256 8.1 / 4.7, 16000 of 256 52 / 4.8, 65000 of 256 183 / 9.1
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = n_tokens <= 512 ? launch_append<256, 1>(a, 1, st) : launch_append<512, 4>(a, 8, st);
  if (rc == LI4_OK) clear_error();
  return rc;
}

extern "C" int li4_rope_paged_write(const void* q, const void* k, const void* v, int dtype, int64_t n_tokens,
                                    int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, const int64_t* strides,
                                    const float* rope_cos, const float* rope_sin, int64_t rope_stride,
                                    int64_t max_pos, const int32_t* positions, const int64_t* slots, void* q_out,
                                    void* k_out, void* cache_k, void* cache_v, int64_t num_pages, int64_t page_size,
                                    void* stream) {
  using namespace li4;
  if (dtype != LI4_F16 && dtype != LI4_BF16)
    return set_error(LI4_ERR_UNSUPPORTED, "rope_paged_write: dtype %d (LI4_F16 or LI4_BF16)", dtype);
  if (n_tokens < 0 || n_heads < 0 || n_kv_heads < 0 || num_pages < 0 || max_pos < 0 || n_tokens > (1 << 30) ||
      n_heads + 2 * n_kv_heads > 65535 || max_pos > (1 << 30))
    return set_error(LI4_ERR_INVALID_ARG, "rope_paged_write: n_tokens=%lld n_heads=%lld n_kv_heads=%lld num_pages=%lld "
                     "max_pos=%lld", (long long)n_tokens, (long long)n_heads, (long long)n_kv_heads,
                     (long long)num_pages, (long long)max_pos);
  if (head_dim < 8 || head_dim > 256 || head_dim % 8 != 0)
    return set_error(LI4_ERR_UNSUPPORTED, "rope_paged_write: head_dim=%lld (a multiple of 8 up to 256)",
                     (long long)head_dim);
  if (!is_pow2(page_size) || page_size < 8 || page_size > 1024)
    return set_error(LI4_ERR_UNSUPPORTED, "rope_paged_write: page_size=%lld (a power of two from 8 to 1024)",
                     (long long)page_size);
  if (n_tokens == 0 || n_heads + n_kv_heads == 0) {
    clear_error();
    return LI4_OK;
  }
  if (max_pos < 1)
    return set_error(LI4_ERR_INVALID_ARG, "rope_paged_write: max_pos=%lld (tokens need a table row)",
                     (long long)max_pos);
  if (!strides || !rope_cos || !rope_sin || !positions || !slots || (n_heads > 0 && (!q || !q_out)) ||
      (n_kv_heads > 0 && (!k || !v)) || (n_kv_heads > 0 && num_pages > 0 && (!cache_k || !cache_v)))
    return set_error(LI4_ERR_INVALID_ARG, "rope_paged_write: null pointer");
  bool aligned = aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(k_out) &&
                 aligned16(cache_k) && aligned16(cache_v) && aligned16(rope_cos) && aligned16(rope_sin) &&
                 rope_stride % 4 == 0;
  for (int i = 0; i < 16; ++i) aligned = aligned && strides[i] % 8 == 0;
  if (!aligned)
    return set_error(LI4_ERR_ALIGNMENT, "rope_paged_write: every row must start on a 16-byte boundary");
  if (rope_stride < head_dim / 2)
    return set_error(LI4_ERR_INVALID_ARG, "rope_paged_write: table rows of %lld for head_dim %lld",
                     (long long)rope_stride, (long long)head_dim);
  RopeArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_out = static_cast<uint16_t*>(k_out);
  a.sqt = strides[0], a.sqh = strides[1], a.skt = strides[2], a.skh = strides[3], a.svt = strides[4],
  a.svh = strides[5], a.sqot = strides[6], a.sqoh = strides[7], a.skot = strides[8], a.skoh = strides[9];
  a.sckp = strides[10], a.sckr = strides[11], a.sckh = strides[12], a.scvp = strides[13], a.scvr = strides[14],
  a.scvh = strides[15];
  a.cos = rope_cos;
  a.sin = rope_sin;
  a.srope = rope_stride;
  a.positions = positions;
  a.slots = reinterpret_cast<const long long*>(slots);
  a.cache_k = static_cast<uint16_t*>(cache_k);
  a.cache_v = static_cast<uint16_t*>(cache_v);
  a.log_page = ilog2(page_size);
  a.num_slots = num_pages << a.log_page;
  a.T = (int)n_tokens;
  a.H = (int)n_heads;
  a.Hkv = (int)n_kv_heads;
  a.chunks = (int)(head_dim / 8);
  a.max_pos = (int)max_pos;
  // heads per thread: all of them when the tokens alone fill the GPU, else as few as keeps it busy
  const int heads = a.H + 2 * a.Hkv;
  const long long blocks = ((long long)a.T * a.chunks + kRopeThreads - 1) / kRopeThreads;
  const long long want = 4LL * current_sm_count();
  long long groups = blocks >= want ? 1 : (want + blocks - 1) / blocks;
  if (groups > heads) groups = heads;
  a.heads_per_group = (int)((heads + groups - 1) / groups);
  groups = (heads + a.heads_per_group - 1) / a.heads_per_group;
  const dim3 grid((unsigned)blocks, (unsigned)groups, 1);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int rc = dtype == LI4_F16
                     ? launch_pdl(rope_paged_write_kernel<__half2>, a, grid, kRopeThreads, 0, 1, s,
                                  "rope_paged_write: kernel launch")
                     : launch_pdl(rope_paged_write_kernel<__nv_bfloat162>, a, grid, kRopeThreads, 0, 1, s,
                                  "rope_paged_write: kernel launch");
  if (rc == LI4_OK) clear_error();
  return rc;
}
