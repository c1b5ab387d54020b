// li4_attention_args.cuh -- what the packed-sequence attention kernels share: arguments, the packed
// rows of a KV head, where a key's rows lie, the exact redo of a row (sm_100a).
#pragma once

#include "li4_common.cuh"
#include "li4_internal.h"

namespace li4 {

// Queries [T, H, d] of B sequences one after another (cu); sequence b's keys are its own packed rows
// (prompt) or the first kv_lens[b] rows its block table names (paged).  Query i of a sequence of n
// queries and L keys sees keys 0 .. L - n + i.
struct SeqAttnArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  long long sqt, sqh, sot, soh;    // element strides: token, head
  long long skp, skt, skh;         // page (paged only), row, KV head
  long long svp, svt, svh;
  const int* cu;
  const int* kv_lens;              // paged only
  const int* tables;               // paged only
  long long table_stride;
  int table_width, num_pages, log_page;
  int B, T, Hkv, rep, hd;
  float scale_log2;                // softmax scale times log2(e)
  int small_rows, big_rows;        // this launch takes sequences of small_rows < n * rep <= big_rows
  int grid;                        // CTAs that share the work
  long long max_keys;              // no sequence has more, as far as the host knows
  float* part;                     // partial results of split items (see li4_seq_attention.cu)
};

// One sequence as this launch sees it (n = 0: not this launch's).
struct Seq {
  int start, n, len;
};

template <bool PAGED>
__device__ __forceinline__ Seq load_seq(const SeqAttnArgs& a, int b) {
  Seq s;
  s.start = max(0, min(a.cu[b], a.T));
  const int end = max(s.start, min(a.cu[b + 1], a.T));
  s.n = end - s.start;
  if constexpr (PAGED) {
    const long long room = (long long)a.table_width << a.log_page;
    s.len = (int)max(0LL, min((long long)a.kv_lens[b], room));
  } else {
    s.len = s.n;
  }
  const long long rows = (long long)s.n * a.rep;
  if (rows <= a.small_rows || rows > a.big_rows) s.n = 0;
  return s;
}

// Element offset of key row j (K and V), or -1 where the block table names no page of the cache (such
// rows read as zeros).
template <bool PAGED>
__device__ __forceinline__ bool key_offsets(const SeqAttnArgs& a, int b, const Seq& s, int j, long long* ko,
                                            long long* vo) {
  if constexpr (PAGED) {
    const int page = a.tables[(long long)b * a.table_stride + (j >> a.log_page)];
    const int row = j & ((1 << a.log_page) - 1);
    *ko = (long long)page * a.skp + (long long)row * a.skt;
    *vo = (long long)page * a.svp + (long long)row * a.svt;
    return (unsigned)page < (unsigned)a.num_pages;
  } else {
    *ko = (long long)(s.start + j) * a.skt;
    *vo = (long long)(s.start + j) * a.svt;
    return true;
  }
}

// ---- 16-bit types ----
template <typename T>
struct Type16;
template <>
struct Type16<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<__half2*>(&u));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint16_t one(float x) { return __half_as_ushort(__float2half_rn(x)); }
};
template <>
struct Type16<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint16_t one(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// One output row again, by one warp, over the keys the row sees among [k0, k1) only: sum_j
// exp2(s_j - m) v_j for dims lane + 32 i in o[i].  The tensor-core tiles multiply a masked key's zero
// probability by its value, so a NaN or infinity in a value that the row must not see reaches the row;
// rows that come out not finite are redone here, where masked keys are never read.
template <typename T, bool PAGED, int D>
__device__ __noinline__ void redo_row(const SeqAttnArgs& a, int b, const Seq s, int kvh, int row, int k0, int k1, float m,
                                      float* o) {
  const int lane = threadIdx.x & 31;
  const int token = row / a.rep, head = kvh * a.rep + row % a.rep;
  const uint16_t* q = a.q + (long long)(s.start + token) * a.sqt + (long long)head * a.sqh;
  const int last = min(k1 - 1, s.len - s.n + token);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
  for (int j0 = k0; j0 <= last; j0 += 32) {
    const int j = j0 + lane;
    long long ko = 0, vo = 0;
    bool have = false;
    float p = 0.f;
    if (j <= last) {
      have = key_offsets<PAGED>(a, b, s, j, &ko, &vo);
      float dot = 0.f;
      if (have) {
        const uint16_t* k = a.k + ko + (long long)kvh * a.skh;
        for (int d = 0; d < a.hd; d += 2) {
          const float2 x = Type16<T>::unpack(*reinterpret_cast<const uint32_t*>(q + d));
          const float2 y = Type16<T>::unpack(*reinterpret_cast<const uint32_t*>(k + d));
          dot += x.x * y.x + x.y * y.y;
        }
      }
      p = exp2_fast(dot * a.scale_log2 - m);
    }
    const int count = min(32, last + 1 - j0);
    for (int c = 0; c < count; ++c) {
      const float pc = __shfl_sync(0xffffffffu, p, c);
      const long long off = __shfl_sync(0xffffffffu, vo, c);
      if (!__shfl_sync(0xffffffffu, (int)have, c)) continue;
      const uint16_t* v = a.v + off + (long long)kvh * a.svh;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int d = lane + 32 * i;
        if (d < a.hd) o[i] += pc * Type16<T>::unpack((uint32_t)v[d]).x;
      }
    }
  }
}

// ---- launches shared by the entry points ----
int launch_seq_attention(const SeqAttnArgs& a, bool paged, int dtype, int max_rows, cudaStream_t stream);
int launch_tile_attention(const SeqAttnArgs& a, bool paged, int dtype, cudaStream_t stream);
size_t tile_attention_part_bytes(int hd, int rep, int64_t tokens, int64_t kv_heads, int64_t max_keys, int sm);
size_t seq_attention_part_bytes(int hd, int max_rows, int sm);

}  // namespace li4
