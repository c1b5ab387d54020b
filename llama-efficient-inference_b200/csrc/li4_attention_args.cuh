// li4_attention_args.cuh -- what the packed-sequence attention kernels share: arguments, the packed
// rows of a KV head (sm_100a).
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

// ---- 16-bit types ----
template <typename T>
struct Type16;
template <>
struct Type16<__half> {
  static __device__ __forceinline__ bool not_finite(uint16_t x) { return (x & 0x7fffu) >= 0x7c00u; }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<__half2*>(&u));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
template <>
struct Type16<__nv_bfloat16> {
  static __device__ __forceinline__ bool not_finite(uint16_t x) { return (x & 0x7fffu) >= 0x7f80u; }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// ---- launches shared by the entry points ----
int launch_seq_attention(const SeqAttnArgs& a, bool paged, int dtype, int max_rows, cudaStream_t stream);
int launch_tile_attention(const SeqAttnArgs& a, bool paged, int dtype, cudaStream_t stream);
size_t tile_attention_part_bytes(int hd, int rep, int64_t tokens, int64_t kv_heads, int64_t max_keys, int sm);
size_t seq_attention_part_bytes(int hd, int max_rows, int sm);

}  // namespace li4
