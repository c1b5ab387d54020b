// li4_logprobs.cu -- log probabilities of given tokens, entropy and the likeliest tokens of rows of logits, sm_100a.
//
// With t_j = (x_j - b) log2(e) for a base b near the largest value, S = sum 2^t_j and W = sum 2^t_j t_j give
//   log p_j = x_j - b - ln 2 log2 S,   entropy = ln 2 (log2 S - W / S)
// in one pass: a thread's base follows its largest value, at a distance of up to 4, and sums with different bases join as
// S' = f S, W' = f (W + d S), d = (b - b') log2(e), f = 2^d.
//
// The likeliest tokens: a thread keeps the largest values of its two best tiles, which tiles these were, and the largest of its
// other tiles.  At the end, of each warp's 32 largest values the j-th, and of these the c-th largest among the warps, j c >= top, bounds
// the top-th largest of all from below.  The few threads whose largest reaches the bound read that tile again, and the
// second (a warp reads all tiles of a thread where a third reaches it) and set such values aside; 64-bit keys of (value's order, inverted index) give their
// order, ranked by counting.  (Values set aside tile by tile, against a bound that grows: 2047 rows of 128256 fp16 values, 8
// likeliest, 148 us, one fp32 row, 20 likeliest, 12.2 us.)  A row whose values are equal can have more of them than there is
// room for; its likeliest are then found one after the other, a pass over the row each.  So rows with fewer allowed tokens than
// likeliest asked for want -infinity in the other places, not the type's lowest value (2047 fp16 rows with three tokens
// allowed, 8 / 32 likeliest: 150 / 151 us with -infinity, 7200 / 27000 us with the lowest value; one row 8 / 10 and 64 / 193).
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
// Of a type's values: 16-byte loads of a thread under way at a time, how many such steps make a tile.  16 values a step for 16-bit
// types (2047 rows of 128256 values, 8 likeliest: fp16 122 us, of four loads a step 131; bf16 127 and 209).  A tile of two steps
// halves the bookkeeping, but with the loads as they are now tiles of one step would do for 16-bit types too (117 and 110 us);
// fp32 rows want them (one row, 20 likeliest: 10.3 us, with tiles of two steps 12.3 us).  Four CTAs per SM, five for bf16 (127
// us instead of 148).
__host__ __device__ constexpr int log_loads(int bytes) { return bytes == 4 ? 4 : 2; }
__host__ __device__ constexpr int log_steps(int bytes) { return bytes == 4 ? 1 : 2; }
constexpr int kLogStep = kLogThreads * 16;  // values of a step
constexpr int kLogAside = 2048;  // keys set aside per CTA
constexpr int kMaxTop = LI4_MAX_TOP;
constexpr int kLogCluster = 8;
constexpr float kLag = 4.f;  // how far a thread's base may lag behind its largest value: 2^t <= e^4
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

// Two fp32 lanes at once.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float max_of3(float a, float b, float c) {  // (drops NaN)
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ Sums join(const Sums& x, const Sums& y) {
  const float b = fmaxf(x.b, y.b);
  // (a base of -infinity: nothing but -infinity seen, sums of 0)
  const float dx = x.b == -INFINITY ? 0.f : t_of(x.b, b), dy = y.b == -INFINITY ? 0.f : t_of(y.b, b);
  const float fx = ex2(dx), fy = ex2(dy);
  return {b, fx * x.s + fy * y.s, fx * (x.w + dx * x.s) + fy * (y.w + dy * y.s)};
}

// The j-th largest of a warp's values (j from 1 to 4), on every lane.
__device__ __forceinline__ float warp_largest(float x, int j) {
  const int lane = threadIdx.x & 31;
  if (j == 1) {
#pragma unroll
    for (int d = 1; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
  }
#pragma unroll
  for (int k = 2; k <= 32; k *= 2)  // a sorting network, the largest on lane 0
#pragma unroll
    for (int d = k / 2; d > 0; d /= 2) {
      const float y = __shfl_xor_sync(0xffffffffu, x, d);
      x = ((lane & d) == 0) == ((lane & k) == 0) ? fmaxf(x, y) : fminf(x, y);
    }
  return __shfl_sync(0xffffffffu, x, j - 1);
}

// Values x with !(x <= bound) are set aside.  The c-th largest of the warps' values less one step (equal values belong to
// those set aside), or -infinity itself.
__device__ __forceinline__ float bound_of(const float* of_warp, int c) {
  const float x = of_warp[threadIdx.x % kLogWarps];
  int above = 0;
#pragma unroll
  for (int w = 0; w < kLogWarps; ++w) {
    const float y = __shfl_sync(0xffffffffu, x, w);
    above += y > x || (y == x && w < (int)threadIdx.x % kLogWarps) ? 1 : 0;
  }
  const unsigned at = __ballot_sync(0xffffffffu, above == c - 1);
  const float v = __shfl_sync(0xffffffffu, x, __ffs(at) - 1);
  const unsigned u = __float_as_uint(v + 0.f);  // one step down: towards 0 above it, away from it below
  return v == -INFINITY ? v : __uint_as_float(v > 0.f ? u - 1 : u == 0 ? 0x80000001u : u + 1);
}

// Sixteen bytes of logits: their largest value (NaN dropped), pair e of them.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static __device__ __forceinline__ float largest(const uint4& r) {
    return max_of3(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), __uint_as_float(r.z), __uint_as_float(r.w));
  }
  static __device__ __forceinline__ float2 two(const uint4& r, int e) {
    return e == 0 ? make_float2(__uint_as_float(r.x), __uint_as_float(r.y)) : make_float2(__uint_as_float(r.z), __uint_as_float(r.w));
  }
};
__device__ __forceinline__ uint32_t word(const uint4& r, int e) { return e == 0 ? r.x : e == 1 ? r.y : e == 2 ? r.z : r.w; }
template <>
struct Vec<__half> {
  static __device__ __forceinline__ float largest(const uint4& r) {
    const __half2 m = __hmax2(__hmax2(u32_as_h2(r.x), u32_as_h2(r.y)), __hmax2(u32_as_h2(r.z), u32_as_h2(r.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ float2 two(const uint4& r, int e) { return __half22float2(u32_as_h2(word(r, e))); }
};
template <>
struct Vec<__nv_bfloat16> {
  static __device__ __forceinline__ __nv_bfloat162 b2(uint32_t u) { return *reinterpret_cast<const __nv_bfloat162*>(&u); }
  static __device__ __forceinline__ float largest(const uint4& r) {
    const __nv_bfloat162 m = __hmax2(__hmax2(b2(r.x), b2(r.y)), __hmax2(b2(r.z), b2(r.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ float2 two(const uint4& r, int e) {
    const uint32_t w = word(r, e);  // (a bf16 is the high half of its fp32)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
};

// Joins a Sums of each of the lowest N lanes, on lane 0.
template <int N>
__device__ __forceinline__ Sums join_lanes(Sums x) {
#pragma unroll
  for (int d = 1; d < N; d *= 2)
    x = join(x, {__shfl_xor_sync(0xffffffffu, x.b, d), __shfl_xor_sync(0xffffffffu, x.s, d), __shfl_xor_sync(0xffffffffu, x.w, d)});
  return x;
}

template <typename T>
__global__ void __launch_bounds__(kLogThreads, __is_same(T, __nv_bfloat16) ? 5 : 4) token_logprobs_kernel(const __grid_constant__ LogArgs a) {
  constexpr int VEC = 16 / sizeof(T), kLogLoads = log_loads(sizeof(T)), STEP = kLogThreads * kLogLoads;
  constexpr int STEPS = log_steps(sizeof(T)), TILE = STEPS * STEP;
  __shared__ __align__(16) unsigned long long s_aside[kLogAside];
  __shared__ __align__(16) unsigned long long s_top[kMaxTop];                // the CTA's likeliest, in order
  __shared__ __align__(16) unsigned long long s_all[kLogCluster * kMaxTop];  // rank 0: every CTA's
  __shared__ unsigned long long s_best[kLogWarps];
  __shared__ float s_warp[kLogWarps];  // each warp's j-th largest
  __shared__ Sums s_sums[kLogWarps];
  __shared__ Sums s_row;               // the CTA's
  __shared__ int s_n;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)cluster.block_rank(), C = (int)cluster.num_blocks();
  const long long r = blockIdx.x / C;
  const int V = a.cols, top = a.top;
  const int j = (top + kLogWarps - 1) / kLogWarps, c = j > 0 ? (top + j - 1) / j : 0;
  pdl_launch_dependents();
  if (tid == 0) s_n = 0;  // (counted in after a barrier)
  pdl_wait_primary();

  const T* row = static_cast<const T*>(a.logits) + r * a.stride;
  // vector v of the row: values VEC v - off .. VEC v - off + VEC - 1, on 16-byte boundaries
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
  const uint4* vec = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row) & ~uintptr_t(15));
  const int vectors = (int)(((long long)V + off + VEC - 1) / VEC);
  const int v0 = (int)((long long)vectors * rank / C), v1 = (int)((long long)vectors * (rank + 1) / C);
  // vectors that lie wholly in the row, of this CTA
  const int c0 = max(v0, off > 0 ? 1 : 0), c1 = min(v1, (int)(((long long)V + off) / VEC));
  auto clean = [&](int t0) { return t0 >= c0 && t0 + STEP <= c1; };

  float most = -INFINITY, second = -INFINITY, other = -INFINITY;  // of the thread's tiles: the two best, the best of the rest
  int most_at = v0, second_at = v0;
  uint4 raw[kLogLoads], next[kLogLoads];
  auto load = [&](uint4* to, int t0) {
#pragma unroll
    for (int l = 0; l < kLogLoads; ++l) to[l] = __ldcg(vec + t0 + l * kLogThreads + tid);
  };
  if (clean(v0)) load(next, v0);
  uint64_t run_s = 0, run_w = 0;  // pairs of sums against base b
  float b = -INFINITY, nb = 0.f;  // the base, which may lag behind the largest value by kLag; minus it, or 0
  for (int t0 = v0; t0 < v1; t0 += TILE) {
    float best = -INFINITY;
#pragma unroll
    for (int h = 0; h < STEPS; ++h) {
      const int at = t0 + h * STEP;
      if (at >= v1) break;
      if (clean(at)) {
#pragma unroll
        for (int l = 0; l < kLogLoads; ++l) raw[l] = next[l];
      } else {
        constexpr uint32_t LOW = sizeof(T) == 4 ? 0xff800000u : __is_same(T, __half) ? 0xfc00fc00u : 0xff80ff80u;  // -infinity
#pragma unroll
        for (int l = 0; l < kLogLoads; ++l) {
          const int v = at + l * kLogThreads + tid;
          raw[l] = make_uint4(LOW, LOW, LOW, LOW);
          if (v >= c0 && v < c1) {
            raw[l] = __ldcg(vec + v);
          } else if (v < v1) {  // a vector that the row's end cuts, value by value; -infinity beside them
            uint32_t u[4] = {LOW, LOW, LOW, LOW};
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const long long at = (long long)v * VEC - off + e;
              if (at < 0 || at >= V) continue;
              if constexpr (sizeof(T) == 4) u[e] = reinterpret_cast<const uint32_t*>(row)[at];
              else u[e >> 1] = __byte_perm(u[e >> 1], reinterpret_cast<const uint16_t*>(row)[at], e & 1 ? 0x5410 : 0x3254);
            }
            raw[l] = make_uint4(u[0], u[1], u[2], u[3]);
          }
        }
      }
      if (at + STEP < v1 && clean(at + STEP)) load(next, at + STEP);
      float m = Vec<T>::largest(raw[0]);
#pragma unroll
      for (int l = 1; l < kLogLoads; ++l) m = fmaxf(m, Vec<T>::largest(raw[l]));
      best = fmaxf(best, m);
      if (m - kLag > b) {
        const float d = b == -INFINITY ? 0.f : t_of(b, m), f = ex2(d);
        const float2 ss = halves(run_s), ww = halves(run_w);
        run_s = pair(f * ss.x, f * ss.y);
        run_w = pair(f * fmaf(d, ss.x, ww.x), f * fmaf(d, ss.y, ww.y));
        b = m;
        nb = -m;
      }
      const uint64_t nb2 = pair(nb, nb), l2e = pair(kLog2e, kLog2e);
      uint64_t s2 = 0, w2 = 0;
#pragma unroll
      for (int l = 0; l < kLogLoads; ++l)
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) {
          const float2 x = Vec<T>::two(raw[l], e);
          const uint64_t t = mul_pair(add_pair(pair(x.x, x.y), nb2), l2e);
          const float2 tf = halves(t);
          const uint64_t p = pair(ex2(tf.x), ex2(tf.y));
          s2 = add_pair(s2, p);
          w2 = fma_pair(p, t, w2);
        }
      const float2 ww = halves(w2);
      if (!(ww.x + ww.y == ww.x + ww.y)) {  // 0 x -infinity: values of probability 0 add 0 (a NaN stays one)
        float w = 0.f;
#pragma unroll
        for (int l = 0; l < kLogLoads; ++l)
#pragma unroll
          for (int e = 0; e < VEC / 2; ++e) {
            const float2 x = Vec<T>::two(raw[l], e);
            const float t = t_of(x.x, -nb), u = t_of(x.y, -nb);
            w = fmaf(ex2(u), u, fmaf(ex2(t), t, w));
          }
        w2 = pair(w, 0.f);
      }
      run_s = add_pair(run_s, s2);
      run_w = add_pair(run_w, w2);
    }
    other = fmaxf(other, fminf(best, second));
    if (best > second) {
      const bool first = best > most;
      second_at = first ? most_at : t0;
      second = first ? most : best;
      most_at = first ? t0 : most_at;
      most = first ? best : most;
    }
  }
  const float2 ss = halves(run_s), ww = halves(run_w);
  Sums sum = {b, ss.x + ss.y, ww.x + ww.y};
  const bool nan = sum.s != sum.s;  // (or an infinity: either way every value is looked at)
  sum = join_lanes<32>(sum);
  if (lane == 0) s_sums[warp] = sum;
  if (top > 0) {
    const float g = warp_largest(most, j);
    if (lane == 0) s_warp[warp] = g;
    if (tid < kMaxTop) s_top[tid] = 0;
  }
  __syncthreads();
  if (warp == kLogWarps - 1) {
    sum = join_lanes<kLogWarps>(s_sums[lane % kLogWarps]);
    if (lane == 0) s_row = sum;
  }
  // ---- the CTA's likeliest, in order; places that no value fills have key 0
  if (top > 0) {
    const float bound = bound_of(s_warp, c);
    // sets aside what reaches the bound of the values of thread `who` in the tile at t0
    auto take = [&](int t0, int who) {
      unsigned mine = 0;  // a bit per value
#pragma unroll
      for (int l = 0; l < STEPS * kLogLoads; ++l) {
        const int v = t0 + l * kLogThreads + who;
        const long long e0 = (long long)v * VEC - off;
        if (v >= c0 && v < c1) {
          const uint4 again = __ldcg(vec + v);
#pragma unroll
          for (int e = 0; e < VEC; e += 2) {
            const float2 x = Vec<T>::two(again, e / 2);
            mine |= (x.x <= bound ? 0u : 1u << (l * VEC + e)) | (x.y <= bound ? 0u : 2u << (l * VEC + e));
          }
        } else if (v < v1) {
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (e0 + e >= 0 && e0 + e < V && !(logit<T>(row[e0 + e]) <= bound)) mine |= 1u << (l * VEC + e);
        }
      }
      if (mine != 0) {
        int at = atomicAdd(&s_n, __popc(mine));
        for (; mine != 0; mine &= mine - 1, ++at) {
          const int b = __ffs(mine) - 1;
          const long long index = (long long)(t0 + b / VEC * kLogThreads + who) * VEC - off + b % VEC;
          if (at < kLogAside) s_aside[at] = key_of(logit<T>(row[index]), (int)index);
        }
      }
    };
    const int tiles = (v1 - v0 + TILE - 1) / TILE;
    if (nan) {
      for (int i = 0; i < tiles; ++i) take(v0 + i * TILE, tid);
    } else if (most > bound && !(other > bound)) {
      take(most_at, tid);
      if (second > bound) take(second_at, tid);
    }
    // a thread whose third tile reaches the bound: the warp reads all of that thread's, a tile per lane
    for (unsigned whole = __ballot_sync(0xffffffffu, !nan && other > bound); whole != 0; whole &= whole - 1)
      for (int i = lane; i < tiles; i += 32) take(v0 + i * TILE, warp * 32 + __ffs(whole) - 1);
    __syncthreads();
    const int n = s_n;
    if (n <= kLogAside) {
      for (int i = tid; i < n; i += kLogThreads) {
        const unsigned long long key = s_aside[i];
        int above = 0, k = 0;
#pragma unroll 4
        for (; k + 2 <= n; k += 2) {
          const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(s_aside + k);
          above += (two.x > key ? 1 : 0) + (two.y > key ? 1 : 0);
        }
        if (k < n) above += s_aside[k] > key ? 1 : 0;
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
  if (C > 1) cluster.sync();
  else __syncthreads();
  // ---- the row's
  if (rank == 0) {
    if (tid < C * top) s_all[tid] = cluster.map_shared_rank(s_top, tid / top)[tid % top];
    if (C > 1 && warp == kLogWarps - 1) {
      sum = join_lanes<kLogCluster>(lane < C ? *cluster.map_shared_rank(&s_row, lane) : Sums{-INFINITY, 0.f, 0.f});
      if (lane == 0) s_sums[0] = sum;
    }
    __syncthreads();
    const Sums all = C > 1 ? s_sums[0] : s_row;
    const float l2 = all.b == -INFINITY ? NAN : log2f(all.s), base = all.b;
    auto logprob = [&](float x) { return (x - base) - kLn2 * l2; };
    if (top > 0) {
      const unsigned long long key = tid < C * top ? s_all[tid] : 0;
      const int values = __syncthreads_count(key != 0);
      int above = 0;
      if (C == 1) above = tid;
      else if (key != 0)
#pragma unroll 4
        for (int k = 0; k < C * top; ++k) above += s_all[k] > key ? 1 : 0;
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
  if (C > 1) cluster.sync();  // (the shared memory of every CTA is read until here)
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
  // CTAs per row: as many as keep the SMs busy, a step's values each at least (64 fp32 rows of 128256, 5 likeliest: one
  // CTA each 25.8 us, 2 17.6, 4 14.5, 8 13.5; without the likeliest 23.0, 14.5, 11.4, 9.7)
  int c = 1;
  while (c < kLogCluster && rows * c <= 2LL * current_sm_count() && cols / (2 * c) >= kLogStep) c *= 2;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = dtype == LI4_F32   ? launch_logprobs<float>(a, rows, c, st)
                 : dtype == LI4_F16 ? launch_logprobs<__half>(a, rows, c, st)
                                    : launch_logprobs<__nv_bfloat16>(a, rows, c, st);
  if (rc == LI4_OK) clear_error();
  return rc;
}
