// li4_tile_attention.cu -- attention of packed sequences with many rows per KV head, on the 5th-generation
// tensor cores (tcgen05), sm_100a.
//
// The rows of an item are those of li4_seq_attention.cu: the rep query heads of a KV head over
// consecutive queries, row = query * rep + head.  An item is two tiles of up to 128 rows (128 / rep whole
// queries each) of one sequence and KV head; the two tiles share every key and value tile, and while one
// tile's softmax runs on the arithmetic units the other's products run on the tensor cores.
//
//   warp 8  (TMA)   queries once, then key and value tiles of 128 rows through a ring of slots; a paged
//                   tile is one copy per page and 64 dims (the page's rows land at their place of the tile)
//   warp 9  (MMA)   S_i = Q_i K^T (M 128, N 128 keys) into tensor memory, O_i += P_i V (A = P_i from tensor
//                   memory, N = dims, V as it lies: N-major) accumulated there over the whole item
//   warps 0-3, 4-7  softmax of tile 0, 1: a thread owns a row (tensor-memory lane) and needs no exchange;
//                   P in the 16-bit type replaces S in its columns
//
// The running maximum moves lazily: probabilities are taken against a maximum that may lag up to 2^8
// behind (P <= 256 fits both 16-bit types, the sum is fp32), so the accumulated output is rescaled only
// when a row's maximum grows by more than that -- rarely after the first tiles.
// Every mbarrier wait is bounded: one that runs out sets bit 8 of li4_device_errors; every role then
// leaves its loop, copies and MMAs in flight are waited for (bounded) and the tensor memory is freed.
#include <cuda.h>

#include <mutex>
#include <utility>
#include <vector>

#include "li4_attention_args.cuh"
#include "li4_gemv_device.cuh"

namespace li4 {

__device__ unsigned g_tile_device_error;  // bit 8 of li4_device_errors

int tile_device_errors(unsigned* flags, bool reset) {
  int rc = check_cuda(cudaMemcpyFromSymbol(flags, g_tile_device_error, sizeof(unsigned)), "device_errors: attention");
  if (rc == LI4_OK && reset) {
    const unsigned zero = 0;
    rc = check_cuda(cudaMemcpyToSymbol(g_tile_device_error, &zero, sizeof(unsigned)), "device_errors: clearing");
  }
  return rc;
}

constexpr int kTileRows = 128;       // rows of a tile: tensor-memory lanes
constexpr int kTileKeys = 128;       // keys of a step
constexpr int kTileThreads = 384;    // 8 softmax warps, the TMA warp, the MMA warp, 2 that only fill their group
constexpr int kTmaWarp = 8, kMmaWarp = 9;
constexpr unsigned kTileWaitLimit = 1u << 24;  // polls
constexpr float kLazyLog2 = 8.f;     // how far the maximum in use may lag, in powers of two

__host__ __device__ constexpr int tile_slots(int D) { return D == 64 ? 8 : 4; }
__host__ __device__ constexpr int tile_bytes(int D) { return 128 * D * 2; }  // a tile of queries, keys or values
__host__ __device__ constexpr int tile_smem_bytes(int D) { return 1024 + (2 + tile_slots(D)) * tile_bytes(D) + 512; }

#ifndef POLY
#define POLY 0x8888
#endif
constexpr unsigned kPolyPairs = POLY;  // which of 16 pairs of probabilities the polynomial takes

struct TileArgs {
  SeqAttnArgs s;
  int tokens_per_tile;  // whole queries of a tile: 128 / rep
  int box_rows;         // key rows of one copy
};

// ---- mbarriers, tensor memory ----
__device__ __forceinline__ bool tile_wait(uint64_t* bar, unsigned parity) {
  for (unsigned i = 0; i < kTileWaitLimit; ++i)
    if (mbar_test_wait(bar, parity)) return true;
  atomicOr(&g_tile_device_error, 256u);
  return false;
}
__device__ __forceinline__ bool tile_wait2(uint64_t* bar, unsigned parity, uint64_t* bar2, unsigned parity2) {
  for (unsigned i = 0; i < kTileWaitLimit; ++i) {
    const bool a = mbar_test_wait(bar, parity), b = mbar_test_wait(bar2, parity2);
    if (a && b) return true;
  }
  atomicOr(&g_tile_device_error, 256u);
  return false;
}
// A converged warp: tests, or waits; every lane returns the same.
__device__ __forceinline__ bool tile_test_warp(uint64_t* bar, unsigned parity) {
  return __all_sync(0xffffffffu, mbar_test_wait(bar, parity));
}
__device__ __forceinline__ bool tile_wait_warp(uint64_t* bar, unsigned parity) {
  for (unsigned i = 0; i < kTileWaitLimit; ++i)
    if (tile_test_warp(bar, parity)) return true;
  if ((threadIdx.x & 31) == 0) atomicOr(&g_tile_device_error, 256u);
  return false;
}

__device__ __forceinline__ void tma_load4(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z,
                                          int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          dst),
      "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// One thread of a converged warp.  Issuing through elect.sync (not a lane test) tells the compiler that one thread is
// active; under `lane == 0` each tcgen05.mma took about 100 cycles to issue (8192-token prompts at 128 dims: 601 us
// against 513).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}

// Shared-memory operand, 128-byte swizzle (see int4_gemm_kernel): K-major rows of 64 values, 8-row groups
// 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)1u << 16 | (uint64_t)(1024u >> 4) << 32 | (uint64_t)1u << 46 |
         (uint64_t)2u << 61;
}
// The same rows read along the other axis (N-major operand: a row is one k, its 64 values are 64 n): the
// next 64 n are `chunk` bytes on (leading offset), the next 8 k 1024 bytes (stride offset).
__device__ __forceinline__ uint64_t desc_n_major(uint32_t addr, uint32_t chunk) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)(chunk >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 |
         (uint64_t)1u << 46 | (uint64_t)2u << 61;
}
// Instruction descriptor, kind::f16: fp32 accumulator, A and B of one type (0 fp16, 1 bf16), B N-major or not.
__host__ __device__ constexpr uint32_t tile_idesc(int n, int type, int b_n_major) {
  return (1u << 4) | ((uint32_t)type << 7) | ((uint32_t)type << 10) | ((uint32_t)b_n_major << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}

// 32 columns of the warp's 32 lanes; the values count once tmem_ld_wait has named them.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                 "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]),
                 "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]),
                 "+f"(v[30]), "+f"(v[31])::"memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const float* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"f"(v[0]),
      "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]),
      "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]),
      "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]),
      "f"(v[29]), "f"(v[30]), "f"(v[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(
          v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(addr)
      : "memory");
}
// Two fp32 lanes at once (the packed forms halve the issue slots of the softmax's multiply-adds and sums).
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float* x, float* y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(*x), "=f"(*y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x and 2^y for x, y <= 64 on the multiply-add pipe.  The 16-per-cycle exponential unit bounds the softmax, so part of
// its exponentials are taken here: x = n + f with n the nearest integer (added to 1.5 * 2^23, which leaves n in the low
// bits), 2^f on [-1/2, 1/2] by a polynomial with value 1 at 0 fitted for the least largest relative error
// (degree 5: 9.2e-8; 1.7e-7 evaluated in fp32, the size of the unit's own error), n added to the exponent bits.  x is
// held at -127, where the sum of bits is exactly zero: a masked score gives probability 0.  NaN passes the bound; its
// bits end up as a huge value that the 16-bit type turns into an infinity.
__device__ __forceinline__ void exp2_pair(uint64_t v, float* x, float* y) {
  unpack2(v, x, y);
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(*x));  // -127
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(*y));
  v = pack2(*x, *y);
  const uint64_t t = add2(v, pack2(12582912.f, 12582912.f));
  const uint64_t n = add2(t, pack2(-12582912.f, -12582912.f));
  const uint64_t f = fma2(n, pack2(-1.f, -1.f), v);
  uint64_t p = pack2(0x1.5bba14p-10f, 0x1.5bba14p-10f);
  p = fma2(p, f, pack2(0x1.3cea88p-7f, 0x1.3cea88p-7f));
  p = fma2(p, f, pack2(0x1.c6b752p-5f, 0x1.c6b752p-5f));
  p = fma2(p, f, pack2(0x1.ebf9bcp-3f, 0x1.ebf9bcp-3f));
  p = fma2(p, f, pack2(0x1.62e42ap-1f, 0x1.62e42ap-1f));
  p = fma2(p, f, pack2(1.f, 1.f));
  float tx, ty, px, py;
  unpack2(t, &tx, &ty);
  unpack2(p, &px, &py);
  *x = __uint_as_float(__float_as_uint(px) + (__float_as_uint(tx) << 23));
  *y = __uint_as_float(__float_as_uint(py) + (__float_as_uint(ty) << 23));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Item `index` of the launch: sequences in order, inside a sequence the later (longer) pairs of tiles first, KV
// heads innermost.  One warp; every lane returns the same.
struct TileItem {
  int b, pair, kvh;  // b = -1: no such item
};
template <bool PAGED>
__device__ __forceinline__ TileItem find_item(const TileArgs& a, int index) {
  const int lane = threadIdx.x & 31;
  const int per_pair = 2 * a.tokens_per_tile;
  TileItem it = {-1, 0, 0};
  for (int b0 = 0; b0 < a.s.B; b0 += 32) {
    int items = 0, pairs = 0;
    if (b0 + lane < a.s.B) {
      pairs = (load_seq<PAGED>(a.s, b0 + lane).n + per_pair - 1) / per_pair;
      items = pairs * a.s.Hkv;
    }
    int incl = items;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, index < incl);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const int rel = index - __shfl_sync(0xffffffffu, incl - items, src);
      pairs = __shfl_sync(0xffffffffu, pairs, src);
      it.b = b0 + src;
      it.pair = pairs - 1 - rel / a.s.Hkv;
      it.kvh = rel % a.s.Hkv;
      return it;
    }
    index -= __shfl_sync(0xffffffffu, incl, 31);
  }
  return it;
}

template <typename T, int D, bool PAGED>
__global__ void __launch_bounds__(kTileThreads, 1)
    tile_attention_kernel(const __grid_constant__ TileArgs a, const __grid_constant__ CUtensorMap map_q,
                          const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  constexpr int NS = tile_slots(D), TB = tile_bytes(D), SUB = D / 64;
  constexpr int TYPE = sizeof(T) == 2 && __is_same(T, __half) ? 0 : 1;
  // Tensor-memory columns: S_i at 128 i, O_i at 256 + D i.  At 64 dims there is room for P_i beside them (64 columns
  // each), so S_i of the next step is computed as soon as the softmax has read the last one; at 128 dims P_i lies in
  // S_i's first 64 columns and the next S_i follows P_i V.
  constexpr bool EARLY = D == 64;
  constexpr uint32_t S_COL = 0, O_COL = 256, P_COL = EARLY ? 384 : 0, P_STEP = EARLY ? 64 : 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + 2 * TB;
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(ring + NS * TB);
  uint64_t* kv_empty = kv_full + NS;
  uint64_t* q_full = kv_empty + NS;
  uint64_t* s_full = q_full + 1;   // [2] S_i written
  uint64_t* p_full = s_full + 2;   // [2][2] half of P_i written (4 warps), O_i rescaled before the first
  uint64_t* o_done = p_full + 4;   // [2] the last P_i V finished
  uint64_t* s_free = o_done + 2;   // [2] S_i read (4 warps); 64 dims only
  uint64_t* v_tail = s_free + 2;   // the last value tile's missing rows are zeros
  uint64_t* drained = v_tail + 1;  // the product warp gave up and its MMAs have finished
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drained + 1);
  TileItem* s_item = reinterpret_cast<TileItem*>(tmem_holder + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  pdl_wait_primary();
  if (warp == 0) {
    const TileItem it = find_item<PAGED>(a, (int)blockIdx.x);
    if (lane == 0) *s_item = it;
  }
  if (tid == 32) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&s_free[i], 4);
    }
    mbar_init(v_tail, 1);
    mbar_init(drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  const TileItem item = *s_item;
  if (item.b < 0) return;
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_holder)),
                 "n"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const Seq s = load_seq<PAGED>(a.s, item.b);
  const int TPT = a.tokens_per_tile;
  const int tok0 = item.pair * 2 * TPT;  // first query of tile 0
  // steps of each tile: up to the last key its last query sees
  int steps[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int first = tok0 + i * TPT, last = min(s.n, first + TPT) - 1;
    const int keys = first < s.n ? max(0, s.len - s.n + last + 1) : 0;
    steps[i] = (keys + kTileKeys - 1) / kTileKeys;
  }
  const int nk = max(steps[0], steps[1]);
  // place of key tile j and value tile j in the ring's order: the order in which the products take them
  auto key_at = [](int j) { return !EARLY ? 2 * j : j == 0 ? 0 : 2 * j - 1; };
  auto value_at = [nk](int j) { return !EARLY || j == nk - 1 ? 2 * j + 1 : 2 * j + 2; };
  // the sequence's last tile: only the keys it has, whole groups of 16; rows past the end are made zeros (what lies
  // there may be anything, and 0 x NaN is NaN)
  const int tail_rows = min(kTileKeys, s.len - (nk - 1) * kTileKeys), tail_groups = (tail_rows + 15) / 16;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  bool ok = true;

  // 384 threads x 168 registers at the launch: the softmax's two groups take 208 each, the third keeps 80
  // (2 x 128 x 208 + 128 x 80 <= 384 x 168)
  if (warp >= kTmaWarp) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
  if (warp == kTmaWarp) {
    // ---- copies
    if (lane == 0 && nk > 0) {
      // a tile whose queries all lie past the tensor is not loaded (its rows are not used)
      const int tiles = steps[1] > 0 ? 2 : 1;
      mbar_arrive_expect_tx(q_full, tiles * SUB * TPT * a.s.rep * 128);
      for (int i = 0; i < tiles; ++i)
        for (int c = 0; c < SUB; ++c)
          tma_load4(smem_addr(smem + i * TB + c * (TB / SUB)), &map_q, q_full, c * 64, 0, item.kvh,
                    s.start + tok0 + i * TPT);
    }
    int n = 0;  // tiles issued
    for (; n < 2 * nk && ok; ++n) {
      // tile n of the ring's order
      const bool value = !EARLY ? n & 1 : n == 2 * nk - 1 || (n > 0 && !(n & 1));
      const int j = !EARLY ? n / 2 : n == 2 * nk - 1 ? nk - 1 : value ? n / 2 - 1 : (n + 1) / 2;
      const int key0 = j * kTileKeys;
      const int rows = min(kTileKeys, s.len - key0);
      int row = s.start + key0, page = 0;
      bool mine = lane == 0;
      int boxes = 1;
      if constexpr (PAGED) {
        boxes = (rows + a.box_rows - 1) / a.box_rows;
        mine = lane < boxes;
        const int key = key0 + lane * a.box_rows;
        row = key & ((1 << a.s.log_page) - 1);
        // an entry outside the cache is a coordinate outside the tensor: zeros
        if (mine) page = a.s.tables[(long long)item.b * a.s.table_stride + (key >> a.s.log_page)];
      }
      const int slot = n % NS;
      if (n >= NS) ok = tile_wait_warp(&kv_empty[slot], ((n / NS) - 1) & 1);
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&kv_full[slot], boxes * a.box_rows * SUB * 128);
      __syncwarp();
      if (mine)
        for (int c = 0; c < SUB; ++c)
          tma_load4(smem_addr(ring + slot * TB + c * (TB / SUB)) + lane * a.box_rows * 128, value ? &map_v : &map_k,
                    &kv_full[slot], c * 64, row, item.kvh, page);
    }
    if (ok && nk > 0 && tail_rows < tail_groups * 16) {
      const int last = 2 * nk - 1, slot = last % NS;
      ok = tile_wait_warp(&kv_full[slot], (last / NS) & 1);
      for (int e = lane; ok && e < (tail_groups * 16 - tail_rows) * SUB * 8; e += 32) {
        const int r = tail_rows + e / (SUB * 8), c = e % (SUB * 8);
        *reinterpret_cast<uint4*>(ring + slot * TB + (c >> 3) * (TB / SUB) + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(v_tail);
    }
    if (!ok)  // copies in flight land before the memory goes
      for (int i = max(0, n - NS); i < n; ++i) tile_wait_warp(&kv_full[i % NS], (i / NS) & 1);
  } else if (warp == kMmaWarp) {
    // ---- products: one elected thread, tile 0 then tile 1 (a warp per tile was slower: their products then share the
    // tensor cores and both finish late).  Any barrier read costs it 160-220 cycles and several at once hardly more, so
    // what a group of products needs is tested together.
    constexpr uint32_t IDESC_S = tile_idesc(kTileKeys, TYPE, 0), IDESC_O = tile_idesc(D, TYPE, 1);
    const uint64_t q_desc = desc_k_major(smem_addr(smem)), k_desc = desc_k_major(smem_addr(ring)),
                   v_desc = desc_n_major(smem_addr(ring), TB / SUB);
    auto full = [&](int n) { return &kv_full[n % NS]; };
    auto phase = [&](int n) { return (unsigned)(n / NS) & 1u; };
    auto scores = [&](int i, int j) {  // S_i of step j
      const uint64_t qd = q_desc + i * (TB >> 4), kd = k_desc + key_at(j) % NS * (TB >> 4);
#pragma unroll
      for (int c = 0; c < SUB; ++c)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_ss(tmem + S_COL + i * 128, qd + ((c * (TB / SUB) + kk * 32) >> 4), kd + ((c * (TB / SUB) + kk * 32) >> 4),
                 IDESC_S, c + kk > 0);
      tc_commit(&s_full[i]);
    };
    auto outputs = [&](int i, int j, int h) {  // half h (64 keys) of P_i V of step j
      const uint64_t vd = v_desc + value_at(j) % NS * (TB >> 4) + h * 512;
      const uint32_t o = tmem + O_COL + i * D, pr = tmem + P_COL + i * P_STEP + h * 32;
      if (j < nk - 1 || tail_groups == 8) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) mma_ts(o, pr + kk * 8, vd + kk * 128, IDESC_O, j + h + kk > 0);
      } else {
#pragma unroll 1
        for (int kk = 0; kk < 4 && 4 * h + kk < tail_groups; ++kk)
          mma_ts(o, pr + kk * 8, vd + kk * 128, IDESC_O, j + h + kk > 0);
      }
    };
    if (elect_one() && nk > 0) {
      ok = tile_wait2(q_full, 0, full(0), 0);
      if (ok) {
        tc_fence_after();
        if (steps[0] > 0) scores(0, 0);
        if (steps[1] > 0) scores(1, 0);
        tc_commit(&kv_empty[0]);
      }
      if (nk == 1 && ok && tail_rows < tail_groups * 16) ok = tile_wait(v_tail, 0);
#pragma unroll 1
      for (int j = 0; j < nk && ok; ++j) {
        const int kn = j + 1 < nk ? key_at(j + 1) : 0, vn = value_at(j);  // (kn 0: a tile that is long there)
        if (j > 0 && j == nk - 1 && tail_rows < tail_groups * 16) ok = tile_wait(v_tail, 0);
        if constexpr (EARLY) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (ok && j + 1 < steps[i]) {
              ok = tile_wait2(&s_free[i], j & 1, full(kn), phase(kn));
              if (!ok) break;
              tc_fence_after();
              scores(i, j + 1);
            }
          if (j + 1 < nk) tc_commit(&kv_empty[kn % NS]);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (ok && j < steps[i]) {
              ok = tile_wait2(&p_full[2 * i], j & 1, full(vn), phase(vn));
              if (!ok) break;
              tc_fence_after();
              outputs(i, j, 0);
              ok = tile_wait(&p_full[2 * i + 1], j & 1);
              if (!ok) break;
              tc_fence_after();
              outputs(i, j, 1);
              tc_commit(&o_done[i]);
            }
          tc_commit(&kv_empty[vn % NS]);
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (ok && j < steps[i]) {
              ok = tile_wait2(&p_full[2 * i], j & 1, full(vn), phase(vn));
              if (!ok) break;
              tc_fence_after();
              outputs(i, j, 0);
              ok = j + 1 < nk ? tile_wait2(&p_full[2 * i + 1], j & 1, full(kn), phase(kn)) : tile_wait(&p_full[2 * i + 1], j & 1);
              if (!ok) break;
              tc_fence_after();
              outputs(i, j, 1);
              tc_commit(&o_done[i]);
              if (j + 1 < steps[i]) scores(i, j + 1);
            }
          tc_commit(&kv_empty[vn % NS]);
          if (j + 1 < nk) tc_commit(&kv_empty[kn % NS]);
        }
      }
      if (!ok) {  // MMAs in flight finish before the memory goes
        tc_commit(drained);
        tile_wait(drained, 0);
      }
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax of tile i: this thread's row
    const int i = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const int tok = tok0 + i * TPT + row / a.s.rep;
    const bool valid = row < TPT * a.s.rep && tok < s.n;
    const int lim = valid ? s.len - s.n + tok : -1;            // last key the row sees
    const int first_lim = s.len - s.n + tok0 + i * TPT;        // the tile's first row's
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + S_COL + i * 128, o_at = tmem + lanes + O_COL + i * D,
                   p_at = tmem + lanes + P_COL + i * P_STEP;
    const float c = a.s.scale_log2;
    float m = -INFINITY, base = 0.f, l = 0.f;  // maximum in use (raw score), m * c or 0, sum against it
    const int my_steps = i == 0 ? steps[0] : steps[1];
    bool s_here = false;
    for (int j = 0; j < my_steps && ok; ++j) {
      if (!s_here) ok = tile_wait_warp(&s_full[i], j & 1);
      if (!ok) break;
      tc_fence_after();
      float x[128];
#pragma unroll
      for (int g = 0; g < 4; ++g) tmem_ld32(s_at + g * 32, x + g * 32);
#pragma unroll
      for (int g = 0; g < 4; ++g) tmem_ld_wait(x + g * 32);
      if constexpr (EARLY) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[i]);
      }
      // (asked here, used after the maximum: the answer takes a while)
      const bool o_here = !EARLY || j == 0 || mbar_test_wait(&o_done[i], (j - 1) & 1);
      const int key0 = j * kTileKeys;
      if (key0 + kTileKeys - 1 > first_lim) {
        const int rel = lim - key0;
#pragma unroll
        for (int e = 0; e < 128; ++e)
          if (e > rel) x[e] = -INFINITY;
      }
      float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int e = 4; e < 124; e += 8) {
#pragma unroll
        for (int w = 0; w < 4; ++w) mx[w] = max3(mx[w], x[e + w], x[e + 4 + w]);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) mx[w] = fmaxf(mx[w], x[124 + w]);
      const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
      // (the difference is NaN for two infinities of one sign: no move)
      if (__any_sync(0xffffffffu, (top - m) * c > kLazyLog2)) {
        const float mn = fmaxf(m, top);
        const float nb = mn == -INFINITY ? 0.f : mn * c;
        const float f = exp2_fast(m * c - nb);
        l = m == -INFINITY ? 0.f : l * f;
        if (j > 0) {
          ok = tile_wait_warp(&o_done[i], (j - 1) & 1);
          if (!ok) break;
          tc_fence_after();
          const float fo = m == -INFINITY ? 0.f : f;
#pragma unroll 1
          for (int g = 0; g < D / 32; ++g) {
            float o[32];
            tmem_ld32(o_at + g * 32, o);
            tmem_ld_wait(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= fo;
            tmem_st32(o_at + g * 32, o);
          }
        }
        m = mn;
        base = nb;
      }
      if constexpr (EARLY) {  // the last P_i V has read P_i
        if (!__all_sync(0xffffffffu, o_here)) ok = tile_wait_warp(&o_done[i], (j - 1) & 1);
        if (!ok) break;
        tc_fence_after();
      }
      const uint64_t cc = pack2(c, c), nb2 = pack2(-base, -base);
      uint64_t sum0 = 0, sum1 = 0;  // pairs of zeros
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int g = 2 * h; g < 2 * h + 2; ++g) {
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float p0, p1;
            const uint64_t t = fma2(pack2(x[g * 32 + 2 * e], x[g * 32 + 2 * e + 1]), cc, nb2);
            if ((kPolyPairs >> e) & 1) {
              exp2_pair(t, &p0, &p1);
            } else {
              unpack2(t, &p0, &p1);
              p0 = exp2_fast(p0);
              p1 = exp2_fast(p1);
            }
            uint64_t& sum = e & 1 ? sum1 : sum0;
            sum = add2(sum, pack2(p0, p1));
            p[e] = Type16<T>::pack(p0, p1);
          }
          tmem_st16(p_at + g * 16, p);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * i + h]);
        if (h == 0) s_here = EARLY && j + 1 < my_steps && mbar_test_wait(&s_full[i], (j + 1) & 1);
      }
      s_here = __all_sync(0xffffffffu, s_here);
      float s0, s1;
      unpack2(add2(sum0, sum1), &s0, &s1);
      l += s0 + s1;
    }
    // ---- the row's output
    if (my_steps > 0 && ok) {
      ok = tile_wait_warp(&o_done[i], (my_steps - 1) & 1);
      tc_fence_after();
    }
    if (ok) {
      const bool none = lim < 0;
      const float inv = 1.f / l;
      uint16_t* out = a.s.out + (long long)(s.start + tok) * a.s.sot +
                      (long long)(item.kvh * a.s.rep + row % a.s.rep) * a.s.soh;
      float odd = 0.f;  // becomes NaN with the first output that is not finite
      if (my_steps > 0) {
#pragma unroll 1
        for (int g = 0; g < D / 32; ++g) {
          float o[32];
          tmem_ld32(o_at + g * 32, o);
          tmem_ld_wait(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) odd = fmaf(o[e], 0.f, odd);
          if (valid) {
#pragma unroll
            for (int v = 0; v < 4; ++v)
              if (g * 32 + v * 8 < a.s.hd) {
                uint4 w;
                w.x = Type16<T>::pack(o[v * 8] * inv, o[v * 8 + 1] * inv);
                w.y = Type16<T>::pack(o[v * 8 + 2] * inv, o[v * 8 + 3] * inv);
                w.z = Type16<T>::pack(o[v * 8 + 4] * inv, o[v * 8 + 5] * inv);
                w.w = Type16<T>::pack(o[v * 8 + 6] * inv, o[v * 8 + 7] * inv);
                *reinterpret_cast<uint4*>(out + g * 32 + v * 8) = none ? make_uint4(0, 0, 0, 0) : w;
              }
          }
        }
      } else if (valid) {
        for (int d = 0; d < a.s.hd; d += 8) *reinterpret_cast<uint4*>(out + d) = make_uint4(0, 0, 0, 0);
      }
      unsigned again = __ballot_sync(0xffffffffu, valid && !none && isfinite(l) && !(odd == 0.f));
      while (again) {
        const int src = __ffs(again) - 1;
        again &= again - 1;
        const float mb = __shfl_sync(0xffffffffu, base, src), ll = __shfl_sync(0xffffffffu, l, src);
        const int pr = (tok0 + i * TPT) * a.s.rep + (warp & 3) * 32 + src;
        float o[D / 32];
        redo_row<T, PAGED, D>(a.s, item.b, s, item.kvh, pr, 0, s.len, mb, o);
        const int rt = pr / a.s.rep;
        uint16_t* ro = a.s.out + (long long)(s.start + rt) * a.s.sot + (long long)(item.kvh * a.s.rep + pr % a.s.rep) * a.s.soh;
        for (int e = 0; e < D / 32; ++e)
          if (lane + 32 * e < a.s.hd) ro[lane + 32 * e] = Type16<T>::one(o[e] / ll);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
  }
}

// ---- tensor maps ----
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult st;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &st) != cudaSuccess ||
        st != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// [w][z][y][d] with element strides sy, sz, sw; boxes of 64 values x by rows of y and bw of w, 128-byte swizzle.
static int make_map(CUtensorMap* map, int dtype, const void* base, int64_t d, int64_t y, int64_t sy, int64_t z,
                    int64_t sz, int64_t w, int64_t sw, int by, int bw) {
  const EncodeTiled fn = encode_tiled();
  if (!fn) return set_error(LI4_ERR_CUDA, "attention: the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)y, (cuuint64_t)z, (cuuint64_t)w};
  // the stride of a dimension of one element is never used: any valid value
  const cuuint64_t strides[3] = {(cuuint64_t)(y > 1 ? 2 * sy : 16), (cuuint64_t)(z > 1 ? 2 * sz : 16),
                                 (cuuint64_t)(w > 1 ? 2 * sw : 16)};
  const cuuint32_t box[4] = {64, (cuuint32_t)by, 1, (cuuint32_t)bw}, one[4] = {1, 1, 1, 1};
  const CUresult rc = fn(map, dtype == LI4_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                         const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return set_error(LI4_ERR_CUDA, "attention: cuTensorMapEncodeTiled failed (%d)", (int)rc);
  return LI4_OK;
}

template <typename T, int D, bool PAGED>
static int launch_tile(const TileArgs& a, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                       unsigned grid, cudaStream_t stream) {
  static std::mutex mu;
  static std::vector<int> done_dev;  // of this kernel
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    bool seen = false;
    for (int d : done_dev) seen |= (d == dev);
    if (!seen) {
      const int rc = check_cuda(cudaFuncSetAttribute(tile_attention_kernel<T, D, PAGED>,
                                                     cudaFuncAttributeMaxDynamicSharedMemorySize, tile_smem_bytes(D)),
                                "attention: shared memory limit");
      if (rc != LI4_OK) return rc;
      done_dev.push_back(dev);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(kTileThreads, 1, 1);
  cfg.dynamicSmemBytes = tile_smem_bytes(D);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, tile_attention_kernel<T, D, PAGED>, a, q, k, v),
                    "attention: kernel launch");
}

int launch_tile_attention(const SeqAttnArgs& args, bool paged, int dtype, cudaStream_t stream) {
  TileArgs a;
  a.s = args;
  const int rep = args.rep, page = 1 << args.log_page;
  a.tokens_per_tile = kTileRows / rep;
  a.box_rows = paged ? (page < kTileKeys ? page : kTileKeys) : kTileKeys;
  CUtensorMap q, k, v;
  // queries [token][KV head][head of the group][d]: a box is the rep rows of tokens_per_tile tokens
  int rc = make_map(&q, dtype, args.q, args.hd, rep, args.sqh, args.Hkv, args.sqh * rep, args.T, args.sqt, rep,
                    a.tokens_per_tile);
  const int64_t y = paged ? page : args.T, w = paged ? args.num_pages : 1;
  if (rc == LI4_OK)
    rc = make_map(&k, dtype, args.k, args.hd, y, args.skt, args.Hkv, args.skh, w, args.skp, a.box_rows, 1);
  if (rc == LI4_OK)
    rc = make_map(&v, dtype, args.v, args.hd, y, args.svt, args.Hkv, args.svh, w, args.svp, a.box_rows, 1);
  if (rc != LI4_OK) return rc;
  const int64_t pairs = args.T / (2 * a.tokens_per_tile) + args.B;  // at least the sequences' pairs of tiles
  const int64_t grid = pairs * args.Hkv;
  if (grid > 0x7fffffff) return set_error(LI4_ERR_UNSUPPORTED, "attention: too many items");
  const unsigned g = (unsigned)grid;
  const bool half = dtype == LI4_F16;
  if (args.hd <= 64) {
    if (paged) return half ? launch_tile<__half, 64, true>(a, q, k, v, g, stream) : launch_tile<__nv_bfloat16, 64, true>(a, q, k, v, g, stream);
    return half ? launch_tile<__half, 64, false>(a, q, k, v, g, stream) : launch_tile<__nv_bfloat16, 64, false>(a, q, k, v, g, stream);
  }
  if (paged) return half ? launch_tile<__half, 128, true>(a, q, k, v, g, stream) : launch_tile<__nv_bfloat16, 128, true>(a, q, k, v, g, stream);
  return half ? launch_tile<__half, 128, false>(a, q, k, v, g, stream) : launch_tile<__nv_bfloat16, 128, false>(a, q, k, v, g, stream);
}

}  // namespace li4
