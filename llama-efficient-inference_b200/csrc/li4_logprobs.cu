// li4_logprobs.cu -- log probabilities of given tokens, entropy and the likeliest tokens of rows of logits, sm_100a.
//
// With t_j = (x_j - b) log2(e) for a base b, the largest value, S = sum 2^t_j and W = sum 2^t_j t_j give
//   log p_j = x_j - b - ln 2 log2 S,   entropy = ln 2 (log2 S - W / S)
// in one pass: a thread's base moves with its largest value, once per tile of 32 values, and sums with different bases join as
// S' = f S, W' = f (W + d S), d = (b - b') log2(e), f = 2^d.
//
// The likeliest tokens: the threads are cut into 32 groups, and the top-th largest of the groups' maxima so far bounds
// the top-th largest value of the row from below.  Values that reach the bound are set aside: of a row of V
// values in random order some 32 ln(32 / (32 - top)) by the first tile and fewer by every later one (20 of 128256: about a
// hundred).  Their order decides at the end: 64-bit keys of (value's order, inverted index), ranked by counting.
// A bound may be old: it only has to be one.  A row whose values rise or are equal can set aside more than there is room
// for; its likeliest are then found one after the other, a pass over the row each.
//
// A cluster of 1, 2, 4 or 8 CTAs takes a row.  Bound by the bytes of the logits where there are many rows, by two trips to memory and
// the cluster's join where there are few.
#include <cooperative_groups.h>

#include "li4_common.cuh"
#include "li4_internal.h"

namespace li4 {

namespace cg = cooperative_groups;

constexpr int kLogThreads = 256;
constexpr int kLogWarps = kLogThreads / 32;
constexpr int kLogValues = 32;   // of a thread in a tile
constexpr int kLogTile = kLogThreads * kLogValues;
constexpr int kLogAside = 2048;  // keys set aside per CTA
constexpr int kMaxTop = LI4_MAX_TOP;
constexpr int kLogCluster = 8;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct LogArgs {
  const void* logits;
  long long stride;
  int cols, top;
  const long long* tokens;  // null: no log probabilities of given tokens
  float* logprobs;
  float* entropy;           // null: none
  long long* top_ids;
  float* top_logprobs;
};

template <typename T>
__device__ __forceinline__ float logit(T x);
template <>
__device__ __forceinline__ float logit<float>(float x) { return x; }
template <>
__device__ __forceinline__ float logit<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float logit<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float maxn(float a, float b) {  // NaN where one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Larger value, then lower index, first; NaN above all.
__device__ __forceinline__ unsigned long long key_of(float x, int index) {
  unsigned u = __float_as_uint(x + 0.f);  // (-0 becomes 0)
  u = x != x ? 0xffffffffu : u & 0x80000000u ? ~u : u | 0x80000000u;
  return (unsigned long long)u << 32 | (0xffffffffu - (unsigned)index);
}
__device__ __forceinline__ float value_of(unsigned long long key) {
  const unsigned u = (unsigned)(key >> 32);
  return u == 0xffffffffu ? NAN : __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int index_of(unsigned long long key) { return (int)(0xffffffffu - (unsigned)key); }

// t is held at -2^14, where 2^t = 0: 0 t stays 0, however far the values lie apart.
__device__ __forceinline__ float t_of(float x, float b) { return maxn((x - b) * kLog2e, -16384.f); }

struct Sums {
  float b, s, w;  // base, sum 2^t, sum 2^t t
};
__device__ __forceinline__ Sums join(const Sums& x, const Sums& y) {
  const float b = fmaxf(x.b, y.b);
  // (a base of -infinity: nothing but -infinity seen, sums of 0)
  const float dx = x.b == -INFINITY ? 0.f : t_of(x.b, b), dy = y.b == -INFINITY ? 0.f : t_of(y.b, b);
  const float fx = ex2(dx), fy = ex2(dy);
  return {b, fx * x.s + fy * y.s, fx * (x.w + dx * x.s) + fy * (y.w + dy * y.s)};
}

// The bound: values x with !(x <= bound) are set aside.  The top-th largest of 32 maxima less one step (equal values
// belong to those set aside), or -infinity itself.
__device__ __forceinline__ float bound_of(float group_max, int top) {
  const int lane = threadIdx.x & 31;
  int above = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float v = __shfl_sync(0xffffffffu, group_max, i);
    above += v > group_max || (v == group_max && i < lane) ? 1 : 0;
  }
  const unsigned at = __ballot_sync(0xffffffffu, above == top - 1);
  const float x = __shfl_sync(0xffffffffu, group_max, __ffs(at) - 1);
  return x == -INFINITY ? x : nextafterf(x, -INFINITY);
}

template <typename T>
__global__ void __launch_bounds__(kLogThreads, 4) token_logprobs_kernel(const __grid_constant__ LogArgs a) {
  constexpr int VEC = 16 / sizeof(T), LOADS = kLogValues / VEC;
  __shared__ unsigned long long s_aside[kLogAside];
  __shared__ unsigned long long s_top[kMaxTop];                 // the CTA's likeliest, in order
  __shared__ unsigned long long s_all[kLogCluster * kMaxTop];   // rank 0: every CTA's
  __shared__ unsigned long long s_best[kLogWarps];
  __shared__ float s_group[32];
  __shared__ Sums s_sums[kLogWarps];
  __shared__ Sums s_row;        // the CTA's
  __shared__ float s_bound;
  __shared__ int s_n;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)cluster.block_rank(), C = (int)cluster.num_blocks();
  const long long r = blockIdx.x / C;
  const int V = a.cols, top = a.top;
  pdl_launch_dependents();
  pdl_wait_primary();

  const T* row = static_cast<const T*>(a.logits) + r * a.stride;
  // vector v of the row: values VEC v - off .. VEC v - off + VEC - 1, on 16-byte boundaries
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
  const int vectors = (int)(((long long)V + off + VEC - 1) / VEC);
  const int v0 = (int)((long long)vectors * rank / C), v1 = (int)((long long)vectors * (rank + 1) / C);
  if (tid == 0) s_n = 0;

  Sums sum = {-INFINITY, 0.f, 0.f};
  float group_max = -INFINITY, bound = -INFINITY;
  bool first = true;
  for (int t0 = v0; t0 < v1; t0 += kLogThreads * LOADS) {
    float x[kLogValues];
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      const int v = t0 + l * kLogThreads + tid;
      const long long e0 = (long long)v * VEC - off;
      if (v < v1 && e0 >= 0 && e0 + VEC <= V) {
        const uint4 raw = *reinterpret_cast<const uint4*>(row + e0);
        const T* p = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[l * VEC + e] = logit<T>(p[e]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          x[l * VEC + e] = v < v1 && e0 + e >= 0 && e0 + e < V ? logit<T>(row[e0 + e]) : -INFINITY;
      }
    }
    float m = x[0];
#pragma unroll
    for (int e = 1; e < kLogValues; ++e) m = fmaxf(m, x[e]);
    if (m > sum.b) {
      const float d = sum.b == -INFINITY ? 0.f : t_of(sum.b, m), f = ex2(d);
      sum.w = f * (sum.w + d * sum.s);
      sum.s *= f;
      sum.b = m;
    }
    const float base = sum.b == -INFINITY ? 0.f : sum.b;
    float s = 0.f, w = 0.f;
#pragma unroll
    for (int e = 0; e < kLogValues; ++e) {
      const float t = t_of(x[e], base);
      const float p = ex2(t);
      s += p;
      w = fmaf(p, t, w);
    }
    sum.s += s;
    sum.w += w;
    if (top > 0) {
      // groups of 8 threads
      group_max = fmaxf(group_max, m);
      float g = group_max;
#pragma unroll
      for (int d = 1; d < 8; d *= 2) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, d));
      if ((lane & 7) == 0) *const_cast<volatile float*>(&s_group[tid / 8]) = g;
      if (first) {
        __syncthreads();
        bound = bound_of(s_group[lane], top);
        if (tid == 0) *const_cast<volatile float*>(&s_bound) = bound;
        __syncthreads();
      } else {
        bound = *const_cast<volatile float*>(&s_bound);
        if (warp == 0) {  // (the other groups' maxima may be of this tile or the last: a bound either way)
          bound = bound_of(*const_cast<volatile float*>(&s_group[lane]), top);
          if (lane == 0) *const_cast<volatile float*>(&s_bound) = bound;
        }
      }
      first = false;
      if (!(m <= bound) || s != s) {
#pragma unroll
        for (int e = 0; e < kLogValues; ++e)
          if (!(x[e] <= bound)) {
            const int at = atomicAdd(&s_n, 1);
            const long long index = (long long)(t0 + e / VEC * kLogThreads + tid) * VEC - off + e % VEC;
            if (at < kLogAside) s_aside[at] = key_of(x[e], (int)index);
          }
      }
    }
  }
#pragma unroll
  for (int d = 1; d < 32; d *= 2)
    sum = join(sum, {__shfl_xor_sync(0xffffffffu, sum.b, d), __shfl_xor_sync(0xffffffffu, sum.s, d),
                     __shfl_xor_sync(0xffffffffu, sum.w, d)});
  if (lane == 0) s_sums[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kLogWarps; ++w) sum = join(sum, s_sums[w]);
    s_row = sum;
  }
  // ---- the CTA's likeliest, in order; places that no value fills have key 0
  if (top > 0) {
    const int n = s_n;
    if (tid < kMaxTop) s_top[tid] = 0;
    __syncthreads();
    if (n <= kLogAside) {
      for (int i = tid; i < n; i += kLogThreads) {
        const unsigned long long key = s_aside[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += s_aside[j] > key ? 1 : 0;
        if (above < top) s_top[above] = key;
      }
    } else {
      unsigned long long last = ~0ull;
      for (int i = 0; i < top; ++i) {
        unsigned long long best = 0;
        for (long long e = (long long)v0 * VEC - off + tid; e < (long long)v1 * VEC - off; e += kLogThreads) {
          if (e < 0 || e >= V) continue;
          const unsigned long long key = key_of(logit<T>(row[e]), (int)e);
          if (key < last && key > best) best = key;
        }
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
          const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, d);
          best = other > best ? other : best;
        }
        if (lane == 0) s_best[warp] = best;
        __syncthreads();
        for (int w = 0; w < kLogWarps; ++w) best = s_best[w] > best ? s_best[w] : best;
        if (tid == 0) s_top[i] = best;
        last = best;
        __syncthreads();
      }
    }
  }
  cluster.sync();
  // ---- the row's
  if (rank == 0) {
    if (tid < C * kMaxTop && top > 0)
      s_all[tid] = tid % kMaxTop < top ? cluster.map_shared_rank(s_top, tid / kMaxTop)[tid % kMaxTop] : 0ull;
    Sums all = s_row;
    for (int c = 1; c < C; ++c) all = join(all, *cluster.map_shared_rank(&s_row, c));
    const float l2 = all.b == -INFINITY ? NAN : log2f(all.s), base = all.b;
    __syncthreads();
    auto logprob = [&](float x) { return (x - base) - kLn2 * l2; };
    if (top > 0) {
      const unsigned long long key = tid < C * kMaxTop ? s_all[tid] : 0;
      int above = 0, values = 0;
      for (int j = 0; j < C * kMaxTop; ++j) {
        above += s_all[j] > key ? 1 : 0;
        values += s_all[j] != 0 ? 1 : 0;
      }
      if (key != 0 && above < top) {
        a.top_ids[r * top + above] = index_of(key);
        a.top_logprobs[r * top + above] = logprob(value_of(key));
      }
      // fewer than top values above -infinity: the lowest indices among the rest, which lie below 2 top
      if (values < top && tid < 32) {
        int place = values;
        for (int e0 = 0; e0 < V && place < top; e0 += 32) {
          const bool low = e0 + lane < V && logit<T>(row[e0 + lane]) == -INFINITY;
          const unsigned hit = __ballot_sync(0xffffffffu, low);
          const int at = place + __popc(hit & ((1u << lane) - 1u));
          if (low && at < top) {
            a.top_ids[r * top + at] = e0 + lane;
            a.top_logprobs[r * top + at] = logprob(-INFINITY);
          }
          place += __popc(hit);
        }
      }
    }
    if (tid == 0) {
      if (a.tokens) {
        const long long token = a.tokens[r];
        a.logprobs[r] = token >= 0 && token < V ? logprob(logit<T>(row[token])) : NAN;
      }
      if (a.entropy) a.entropy[r] = kLn2 * (l2 - all.w / all.s);
    }
  }
  cluster.sync();  // (the shared memory of every CTA is read until here)
}

template <typename T>
static int launch_logprobs(const LogArgs& a, int64_t rows, int cluster, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cluster), 1, 1);
  cfg.blockDim = dim3(kLogThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return check_cuda(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, a), "token_logprobs: kernel launch");
}

}  // namespace li4

extern "C" int li4_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t cols, int64_t stride,
                                  const int64_t* tokens, int64_t top, float* logprobs, float* entropy,
                                  int64_t* top_ids, float* top_logprobs, void* stream) {
  using namespace li4;
  const char* what = "token_logprobs";
  if (dtype != LI4_F16 && dtype != LI4_BF16 && dtype != LI4_F32)
    return set_error(LI4_ERR_UNSUPPORTED, "%s: dtype %d (LI4_F16, LI4_BF16 or LI4_F32)", what, dtype);
  if (rows < 0 || cols < 1 || cols > (1 << 30) || rows > (1 << 27) || stride < 0 || (rows > 1 && stride < cols))
    return set_error(LI4_ERR_INVALID_ARG, "%s: rows=%lld cols=%lld stride=%lld", what, (long long)rows, (long long)cols,
                     (long long)stride);
  if (top < 0 || top > kMaxTop || top > cols)
    return set_error(LI4_ERR_UNSUPPORTED, "%s: top=%lld of %lld (at most %d)", what, (long long)top, (long long)cols,
                     kMaxTop);
  if (rows == 0) {
    clear_error();
    return LI4_OK;
  }
  if (!logits || (tokens != nullptr) != (logprobs != nullptr) || (top > 0 && (!top_ids || !top_logprobs)))
    return set_error(LI4_ERR_INVALID_ARG, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == LI4_F32 ? 4 : 2) != 0)
    return set_error(LI4_ERR_ALIGNMENT, "%s: logits are not aligned to their type", what);
  LogArgs a;
  a.logits = logits;
  a.stride = stride;
  a.cols = (int)cols;
  a.top = (int)top;
  a.tokens = reinterpret_cast<const long long*>(tokens);
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_ids = reinterpret_cast<long long*>(top_ids);
  a.top_logprobs = top_logprobs;
  // CTAs per row: as many as keep the SMs busy, a tile each at least
  int c = 1;
  while (c < kLogCluster && rows * c <= 2LL * current_sm_count() && cols / (2 * c) >= kLogTile) c *= 2;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = dtype == LI4_F32   ? launch_logprobs<float>(a, rows, c, st)
                 : dtype == LI4_F16 ? launch_logprobs<__half>(a, rows, c, st)
                                    : launch_logprobs<__nv_bfloat16>(a, rows, c, st);
  if (rc == LI4_OK) clear_error();
  return rc;
}
