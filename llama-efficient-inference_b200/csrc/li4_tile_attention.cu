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
//                   writes P in the 16-bit type
//   warp 10         the CTA's next item, when the present one nears its end
// Over a cache in 4 bits a fourth group of warps, 12 to 15, unpacks a quarter each of every key and value tile into its
// slot instead; warp 8 copies the queries alone.
//
// Prompts of 8192 tokens (32 / 8 heads, fp16), 128 dims: 463 us in a burst (1.19 PFLOP/s, 0.72 of cuBLAS's burst rate);
// call after call for seconds 530 us (1.04 PFLOP/s, 0.75 of its sustained rate), as the power limit brings the clock to
// 1.5 GHz: 0.82 million cycles either way.  64 dims: 370 us, bound by the softmax's issue and latency.  A NaN in the
// first value, which runs every CTA's first two items twice: 775 and 574 us.
//
// The running maximum moves lazily: probabilities are taken against a maximum that may lag up to 2^8
// behind (P <= 256 fits both 16-bit types, the sum is fp32), so the accumulated output is rescaled only
// when a row's maximum grows by more than that -- rarely after the first tiles.
//
// A masked key's probability is zero, but zero times a NaN or an infinity is NaN: a value that a row must not see can
// reach it through the last few key tiles of an item, where some keys are hidden from some rows.  A CTA that meets an
// output that is not finite therefore runs that item again, and its later ones from the start, with care (a role's
// code exists twice where that spares the usual pass time): the copying warp takes the values that are not finite out
// of those tiles before the products may have them and notes where in each dim the first +inf, -inf or NaN stood, and a
// row that sees that key gets it added at the end (what is not finite does not depend on its weight in a sum).  At most
// two items of a CTA run twice, whatever the context.
// Every mbarrier wait is bounded: one that runs out sets bit 8 of li4_device_errors.  The copying warp then issues
// nothing more (a barrier whose bytes are still to come must not be armed twice), the other roles run to the end of
// their item without waiting, copies and MMAs in flight are waited for (bounded) and the tensor memory is freed.
#include <cuda.h>

#include <atomic>
#include <mutex>
#include <type_traits>
#include <utility>
#include <vector>

#include "li4_attention_args.cuh"
#include "li4_gemv_device.cuh"
#include "li4_int4_pages.cuh"

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
constexpr int kTileThreads = 384;    // 8 softmax warps, the TMA, MMA and item warps, one that only fills its group
constexpr int kTmaWarp = 8, kMmaWarp = 9, kUnpackWarp = 12;
constexpr int kTile4Threads = 512;   // over a cache in 4 bits: and 4 unpacking warps
constexpr unsigned kTileWaitLimit = 1u << 24;  // polls, about half a second; and for each key tile that an item may have,
constexpr unsigned kTileWaitStep = 1u << 8;    // as some waits last an item (a step of 2900 cycles is some 60 polls)
constexpr int kTileMinSteps = 8;     // key tiles below which a range is not cut
constexpr int kUnseen = 0x7fffffff;   // no key
constexpr float kLazyLog2 = 8.f;     // how far the maximum in use may lag, in powers of two

__host__ __device__ constexpr int tile_slots(int D) { return D == 64 ? 8 : 4; }
__host__ __device__ constexpr int tile_bytes(int D) { return 128 * D * 2; }  // a tile of queries, keys or values
__host__ __device__ constexpr int tile_smem_bytes(int D) { return 1024 + (2 + tile_slots(D)) * tile_bytes(D) + 512 + 16 * D; }

// Which of 16 pairs of probabilities the polynomial takes (8192 tokens at 64 dims: none 387 us, 2 378 us, 4 360 us,
// 5 370 us; at 128 dims, where the products and the power limit bound, 459, 456, 460, 466 us).
constexpr unsigned kPolyPairs = 0x8888;

struct TileArgs {
  SeqAttnArgs s;
  int tokens_per_tile;  // whole queries of a tile: 128 / rep
  int part_slots;       // items whose partial results fit the workspace (0: keys are not split)
  int box_rows;         // key rows of one copy
  unsigned wait_limit;  // polls of a wait
};

// Over a cache in 4 bits (Q4): k, v and box_rows are not used.
struct Tile4Args : TileArgs {
  li4_int4_pages k4, v4;
};
template <typename ArgsT>
constexpr bool kTileInt4 = __is_same(ArgsT, Tile4Args);

// ---- mbarriers, tensor memory ----
// A converged warp waits for a phase, at most `limit` polls; a wait that runs out leaves limit = 1, which makes every later
// wait of the warp give up at once: the roles then run to their ends on whatever is there, no role misses another's
// arrival, and the warp reports at the end.  (Written as one PTX loop for a whole warp: a ready barrier costs 63 cycles,
// against 120 in a branch of one thread and 150 with a check after it.)
__device__ __forceinline__ void tile_wait(uint64_t* bar, unsigned parity, unsigned& limit) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, %0;\n"
      "LAB_WAIT:\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra LAB_DONE;\n\t"
      "sub.u32 n, n, 1;\n\tsetp.ne.u32 q, n, 0;\n\t@q bra LAB_WAIT;\n\tmov.u32 %0, 1;\nLAB_DONE:\n\t}"
      : "+r"(limit)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
}
// Both of two barriers (two tests together cost hardly more than one).
__device__ __forceinline__ void tile_wait2(uint64_t* bar, unsigned parity, uint64_t* bar2, unsigned parity2,
                                           unsigned& limit) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, %0;\n"
      "LAB_WAIT:\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 q, [%3], %4;\n\tand.pred p, p, q;\n\t@p bra LAB_DONE;\n\t"
      "sub.u32 n, n, 1;\n\tsetp.ne.u32 q, n, 0;\n\t@q bra LAB_WAIT;\n\tmov.u32 %0, 1;\nLAB_DONE:\n\t}"
      : "+r"(limit)
      : "r"(smem_addr(bar)), "r"(parity), "r"(smem_addr(bar2)), "r"(parity2)
      : "memory");
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
// (the high word of both forms below: stride offset 1024, version 1, 128-byte swizzle)
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_k_major(uint32_t addr) { return ((addr >> 4) & 0x3FFFu) | 1u << 16; }
// The same rows read along the other axis (N-major operand: a row is one k, its 64 values are 64 n): the
// next 64 n are `chunk` bytes on (leading offset), the next 8 k 1024 bytes (stride offset).
__device__ __forceinline__ uint32_t desc_n_major(uint32_t addr, uint32_t chunk) {
  return ((addr >> 4) & 0x3FFFu) | (chunk >> 4) << 16;
}
// Instruction descriptor, kind::f16: fp32 accumulator, A and B of one type (0 fp16, 1 bf16), B N-major or not.
__host__ __device__ constexpr uint32_t tile_idesc(int n, int type, int b_n_major) {
  return (1u << 4) | ((uint32_t)type << 7) | ((uint32_t)type << 10) | ((uint32_t)b_n_major << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTileRows >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "r"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tmov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "r"(kDescHigh)
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
// bits), 2^f on [-1/2, 1/2] by a polynomial with value 1 at 0, its coefficients from a linear program
// for the least largest relative error on Chebyshev nodes, then rounded to fp32 (degree 5: 1.09e-7 in exact arithmetic,
// 1.7e-7 evaluated in fp32, the size of the unit's own error), n added to the exponent bits.  x is
// held at -127, where the sum of bits is exactly zero: a masked score gives probability 0.  NaN passes the bound and its
// bits end up as the largest finite value; the row's maximum is NaN then, which makes its sum NaN.
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
// (NaN where one of them is)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The launch's items: sequences in order, inside a sequence the later (longer) pairs of tiles first, then the KV heads,
// the ranges of keys innermost.  One warp; every lane returns the same.
struct TileWork {
  int b;              // sequence; -1: no such item
  int kvh;
  int start, n, len;  // the sequence (Seq)
  int tok0;           // first query of tile 0
  int first;          // first key tile of the item's range
  int steps[2];       // key tiles of each tile of rows: up to the last key its last query sees
  int part;           // the item's place among the partial results; -1: it has all its keys
};

// Ranges of keys per (pair of tiles, KV head): more than one where these alone leave SMs idle.
template <bool PAGED>
__device__ __forceinline__ int item_splits(const TileArgs& a) {
  if (a.part_slots == 0) return 1;
  const int lane = threadIdx.x & 31, per_pair = 2 * a.tokens_per_tile;
  int pairs = 0, len = 0;
  for (int b = lane; b < a.s.B; b += 32) {
    const Seq s = load_seq<PAGED>(a.s, b);
    pairs += (s.n + per_pair - 1) / per_pair;
    if (s.n > 0) len = max(len, s.len);
  }
  pairs = __reduce_add_sync(0xffffffffu, pairs);
  len = __reduce_max_sync(0xffffffffu, len);
  const int most = (len + kTileMinSteps * kTileKeys - 1) / (kTileMinSteps * kTileKeys);
  return max(1, min(most, a.part_slots / max(1, pairs * a.s.Hkv)));
}

template <bool PAGED>
__device__ __forceinline__ TileWork find_item(const TileArgs& a, int index, int splits) {
  const int lane = threadIdx.x & 31;
  const int per_pair = 2 * a.tokens_per_tile, number = index;
  TileWork w = {};
  w.b = -1;
  for (int b0 = 0; b0 < a.s.B; b0 += 32) {
    int items = 0, pairs = 0;
    Seq s = {0, 0, 0};
    if (b0 + lane < a.s.B) {
      s = load_seq<PAGED>(a.s, b0 + lane);
      pairs = (s.n + per_pair - 1) / per_pair;
      items = pairs * a.s.Hkv * splits;
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
      w.b = b0 + src;
      w.part = splits > 1 ? number : -1;
      w.start = __shfl_sync(0xffffffffu, s.start, src);
      w.n = __shfl_sync(0xffffffffu, s.n, src);
      w.len = __shfl_sync(0xffffffffu, s.len, src);
      const int head = rel / splits, split = rel - head * splits;
      w.kvh = head % a.s.Hkv;
      w.tok0 = (pairs - 1 - head / a.s.Hkv) * per_pair;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int first = w.tok0 + i * a.tokens_per_tile, last = min(w.n, first + a.tokens_per_tile) - 1;
        const int keys = first < w.n ? max(0, w.len - w.n + last + 1) : 0;
        w.steps[i] = (keys + kTileKeys - 1) / kTileKeys;
      }
      const int all = max(w.steps[0], w.steps[1]), per = max(kTileMinSteps, (all + splits - 1) / splits);
      w.first = min(all, split * per);
      const int end = min(all, w.first + per);
      w.steps[0] = max(0, min(w.steps[0], end) - w.first);
      w.steps[1] = max(0, min(w.steps[1], end) - w.first);
      return w;
    }
    index -= __shfl_sync(0xffffffffu, incl, 31);
  }
  return w;
}

// Cluster launch control: asks for a CTA of this launch that has not started yet; its index arrives in `reply` on `bar`.
__device__ __forceinline__ void ask_next(uint32_t reply, uint64_t* bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(reply),
      "r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ int read_next(uint32_t reply) {  // -1: none is left
  int x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 lo, hi;\n\t.reg .b128 h;\n\t"
      "ld.shared.v2.b64 {lo, hi}, [%1];\n\tmov.b128 h, {lo, hi};\n\tmov.b32 %0, -1;\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n\t}"
      : "=r"(x)
      : "r"(reply)
      : "memory");
  return x;
}

// One item's partial results: 2 x 128 rows of D outputs, four dims of all rows after four dims of all rows (a warp's lanes
// are rows), then (exponent base, sum) per row.
__host__ __device__ constexpr size_t tile_part_floats(int D) { return (size_t)2 * kTileRows * (D + 2); }
__device__ __forceinline__ size_t tile_part_at(int row, int d) { return ((size_t)(d >> 2) * 2 * kTileRows + row) * 4 + (d & 3); }

// Takes what is not finite out of rows [from, to) of a value tile (the warp's lanes are rows) and notes, per dim, the first
// key with +inf or NaN and the first with -inf or NaN: `first` is [2][D].
template <typename T, int D>
__device__ __noinline__ void take_out(uint8_t* tile, int from, int to, int key0, int* first) {
  constexpr uint16_t INF = __is_same(T, __half) ? 0x7c00 : 0x7f80;
  for (int r = from + (threadIdx.x & 31); r < to; r += 32) {
#pragma unroll 1
    for (int c = 0; c < D / 8; ++c) {  // the chunk of dims 8 c .. 8 c + 7: at c ^ r of its row (128-byte swizzle)
      uint4* at = reinterpret_cast<uint4*>(tile + (c >> 3) * (tile_bytes(D) * 64 / D) + r * 128 + ((c ^ r) & 7) * 16);
      const uint4 v = *at;
      uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint16_t x = (uint16_t)(u[e >> 1] >> (e & 1) * 16);
        if ((x & 0x7fff) < INF) continue;
        if (x != (INF | 0x8000)) atomicMin(first + 8 * c + e, key0 + r);
        if (x != INF) atomicMin(first + D + 8 * c + e, key0 + r);
        u[e >> 1] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
        *at = make_uint4(u[0], u[1], u[2], u[3]);
      }
    }
  }
}

// Adds what was taken out to the outputs of the warp's rows (lane's row sees keys up to last).
template <int D>
__device__ __noinline__ void put_back(uint32_t o_at, const int* first, int last) {
#pragma unroll 1
  for (int g = 0; g < D / 32; ++g) {
    float o[32];
    tmem_ld32(o_at + g * 32, o);
    tmem_ld_wait(o);
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      if (last >= first[g * 32 + e]) o[e] += INFINITY;
      if (last >= first[g * 32 + e + D]) o[e] -= INFINITY;
    }
    tmem_st32(o_at + g * 32, o);
  }
  tmem_st_wait();
}

// ---- a cache in 4 bits: a quarter of a tile (32 rows) by a warp, a row per lane: one address per row, and 8 neighbouring
// lanes store to all eight 16-byte places of swizzled rows.  A lane's row of the next key and of the next value tile waits in
// shared memory of its own (2048 tokens over 8000 at 128 dims: two lanes per row, an address and a shuffle for each turn
// of 16 rows 741 us, rows kept in registers 461 us, like this 369 us; the 16-bit cache 270 us).
__host__ __device__ constexpr int row4_bytes(int D) { return D / 2 + D / kGroup4 * 4; }
__host__ __device__ constexpr int rows4_bytes(int D) { return 2 * kTileKeys * row4_bytes(D); }  // of the four warps

// The page of key `key`, -1 past the end.  (Whether it lies in the cache is asked where it is used: the answer of the
// table takes a trip to L2.)
__device__ __forceinline__ int row_page4(const SeqAttnArgs& a, const TileWork& w, int key) {
  int page = -1;
  if (key < w.len) page = a.tables[(long long)w.b * a.table_stride + (key >> a.log_page)];
  return page;
}

// Asks for the row of this lane's key; what does not exist becomes zero codes and parameters, which make zeros.  to: the
// warp's rows, 16-byte pieces of codes of all lanes after one another, then their parameters; kvh: the item's KV head.
template <int D>
__device__ __forceinline__ void load_row4(uint32_t to, const SeqAttnArgs& a, const li4_int4_pages& pages, int kvh, int page,
                                          int key) {
  const int lane = threadIdx.x & 31, row = key & ((1 << a.log_page) - 1);
  const bool ok = (unsigned)page < (unsigned)a.num_pages;
  const uint8_t* c = static_cast<const uint8_t*>(pages.codes) + page * pages.stride_cp + row * pages.stride_ct + kvh * pages.stride_ch;
  const uint32_t* p = static_cast<const uint32_t*>(pages.params) + page * pages.stride_pp + row * pages.stride_pt + kvh * pages.stride_ph;
  if (!ok) {  // (addresses are not read then)
    c = reinterpret_cast<const uint8_t*>(a.q);
    p = reinterpret_cast<const uint32_t*>(a.q);
  }
#pragma unroll
  for (int g = 0; g < D / 32; ++g) {
    const bool have = ok && g * kGroup4 < a.hd;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + g * 512 + lane * 16), "l"(have ? c + g * 16 : c),
                 "r"(have ? 16 : 0)
                 : "memory");
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + 16 * D + g * 128 + lane * 4), "l"(have ? p + g : p),
                 "r"(have ? 4 : 0)
                 : "memory");
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

// The row's values to row r of the tile.
template <typename T, int D>
__device__ __forceinline__ void store_row4(const uint8_t* from, uint8_t* tile, int r) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int g = 0; g < D / 32; ++g) {
    const uint4 c = *reinterpret_cast<const uint4*>(from + g * 512 + lane * 16);
    const uint32_t p = *reinterpret_cast<const uint32_t*>(from + 16 * D + g * 128 + lane * 4);
    uint8_t* at = tile + (g >> 1) * (tile_bytes(D) * 64 / D) + r * 128;
    const uint32_t s2 = both_low(p), m2 = both_high(p);
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t u[4];
      values8<T>(w[e], s2, m2, u);
      *reinterpret_cast<uint4*>(at + (((4 * (g & 1) + e) ^ (r & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
}

template <typename T, int D, bool PAGED, typename ArgsT>
__global__ void __launch_bounds__(kTileInt4<ArgsT> ? kTile4Threads : kTileThreads, 1)
    tile_attention_kernel(const __grid_constant__ ArgsT a, const __grid_constant__ CUtensorMap map_q,
                          const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  constexpr int NS = tile_slots(D), TB = tile_bytes(D), SUB = D / 64;
  constexpr bool Q4 = kTileInt4<ArgsT>;
  constexpr int TYPE = __is_same(T, __half) ? 0 : 1;
  // Tensor-memory columns: S_i at 128 i, O_i at 256 + D i.  At 64 dims there is room for P_i beside them (64 columns
  // each), so S_i of the next step is computed as soon as the softmax has read the last one; at 128 dims P_i lies in
  // S_i's first 64 columns and the next S_i follows P_i V.
  constexpr bool EARLY = D == 64;
  constexpr uint32_t S_COL = 0, O_COL = 256, P_COL = EARLY ? 384 : 0, P_STEP = EARLY ? 64 : 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + 2 * TB;
  uint8_t* reply = ring + NS * TB;       // 16 bytes
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(reply + 16);
  uint64_t* kv_empty = kv_full + NS;
  uint64_t* q_full = kv_empty + NS;
  uint64_t* q_empty = q_full + 1;        // the item's last scores have read the queries
  uint64_t* s_full = q_empty + 1;        // [2] S_i written
  uint64_t* p_full = s_full + 2;         // [2][2] half of P_i written (4 warps), O_i rescaled before the first
  uint64_t* o_done = p_full + 4;         // [2] the last P_i V finished
  uint64_t* s_free = o_done + 2;         // [2] S_i read (4 warps); 64 dims only
  uint64_t* v_tail = s_free + 2;         // the last value tile's rows are there, its missing rows not yet zeros
  uint64_t* drained = v_tail + 1;        // a wait ran out: the MMAs issued so far have finished
  uint64_t* work_full = drained + 1;     // [2] work[i] names an item
  uint64_t* work_empty = work_full + 2;  // [2] the working warps have read it (Q4: 14 of them)
  uint64_t* replied = work_empty + 2;    // the reply is there
  uint64_t* ending = replied + 1;        // the products are near the item's end
  uint64_t* taken_out = ending + 1;      // [2] an item's infinities and NaNs are noted (items taken with care alone)
  uint64_t* noted = taken_out + 2;       // Q4: the notes of an item taken with care are clear
  uint64_t* notes_read = noted + 1;      // [2] the 8 softmax warps have read an item's notes
  TileWork* work = reinterpret_cast<TileWork*>(notes_read + 2);  // [2]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(work + 2);
  volatile int* again = reinterpret_cast<int*>(tmem_holder + 1);  // [2] by item parity: one to run again
  volatile int* gave_up = again + 2;             // [2] a wait of the usual pass, of the one with care ran out
  int* first_bad = const_cast<int*>(again) + 4;  // [2][2][D] of items taken with care: see take_out
  static_assert(16 + (2 * NS + 25) * 8 + 2 * sizeof(TileWork) + 20 <= 512, "what lies behind the tiles fits");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&kv_full[i], Q4 ? 4 : 1);
      mbar_init(&kv_empty[i], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&work_full[i], 1);
      mbar_init(&work_empty[i], Q4 ? 14 : 10);
    }
    mbar_init(v_tail, 1);
    mbar_init(drained, 1);
    mbar_init(replied, 1);
    mbar_init(ending, 1);
    mbar_init(&taken_out[0], Q4 ? 4 : 1);
    mbar_init(&taken_out[1], Q4 ? 4 : 1);
    if (Q4) mbar_init(noted, 1);
    mbar_init(&notes_read[0], 8);
    mbar_init(&notes_read[1], 8);
    again[0] = again[1] = gave_up[0] = gave_up[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_holder)),
                 "n"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait_primary();
  const uint32_t tmem = *tmem_holder;
  const int TPT = a.tokens_per_tile;
  unsigned limit = a.wait_limit;

  // Place of key tile j and value tile j in an item's order of the ring: the order in which the products take them.
  auto key_at = [](int j) { return !EARLY ? 2 * j : j == 0 ? 0 : 2 * j - 1; };
  auto value_at = [](int j, int nk) { return !EARLY || j == nk - 1 ? 2 * j + 1 : 2 * j + 2; };
  // A wait of this warp has run out.  (All lanes of a wait test one word in one instruction, so they agree.)
  auto ran_out = [&]() { return __any_sync(0xffffffffu, limit == 1) != 0; };
  // The working warps' next item (this CTA's k-th); b = -1 ends.
  auto next_work = [&](int k) {
    tile_wait(&work_full[k & 1], (k >> 1) & 1, limit);
    TileWork w = work[k & 1];
    if (ran_out()) w.b = -1;
    if (lane == 0) mbar_arrive(&work_empty[k & 1]);
    return w;
  };
  // The end of the usual pass, where every warp meets.  True: a pass with care follows.
  auto go_again = [&]() {
    if (ran_out() && lane == 0) gave_up[0] = 1;
    tc_fence_before();
    __syncthreads();
    return gave_up[0] == 0 && again[0] + again[1] > 0;
  };
  auto end_care = [&]() {
    if (ran_out() && lane == 0) gave_up[1] = 1;
    tc_fence_before();
    __syncthreads();
  };
  // The item's first key tile with a key that some row of it must not see.
  auto masked_from = [](const TileWork& w) {
    return max(0, (max(0, w.len - w.n + w.tok0 + 1) >> 7) - w.first);
  };
  // Keys of the item's last key tile; P V takes them in groups of 16, and rows of the last group past the end are made
  // zeros (what lies there may be anything, and 0 x NaN is NaN).
  auto tail_rows_of = [](const TileWork& w, int nk) { return min(kTileKeys, w.len - (w.first + nk - 1) * kTileKeys); };

  // 384 threads x 168 registers at the launch: the softmax's two groups take 208 each, the third keeps 80
  // (2 x 128 x 208 + 128 x 80 <= 384 x 168)
  // Q4: 512 threads x 128 at the launch: 192 each for the softmax, 48 for the third group, 80 for the unpacking warps
  // (2 x 128 x 192 + 128 x 48 + 128 x 80 = 512 x 128; 192 / 64 / 64: 2048 tokens over 8000 at 128 dims 555 us instead of 461)
  if (Q4 && warp >= kUnpackWarp) {
    if constexpr (Q4) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
      // ---- this warp's quarter of the key and value tiles
      const int row0 = (warp - kUnpackWarp) * (kTileKeys / 4);
      uint8_t* const rows = reinterpret_cast<uint8_t*>(reply) + 512 + 16 * D + (warp - kUnpackWarp) * 64 * row4_bytes(D);  // keys', values'
      int k = 0;
      unsigned base = 0;
      for (bool care = false;; care = true) {
        unsigned cares = 0;
        for (;;) {
          const TileWork w = next_work(k++);
          if (w.b < 0) break;
          const int nk = max(w.steps[0], w.steps[1]);
          if (nk == 0) continue;
          const int key0 = w.first * kTileKeys + row0 + lane;  // this lane's key of key tile 0
          int page = row_page4(a.s, w, key0), page_v = page;
          load_row4<D>(smem_addr(rows), a.s, a.k4, w.kvh, page, key0);
          load_row4<D>(smem_addr(rows + 32 * row4_bytes(D)), a.s, a.v4, w.kvh, page, key0);
          page = row_page4(a.s, w, key0 + kTileKeys);  // pages of the key tile that is asked for next
          const int care_from = care ? masked_from(w) : nk;
          int* bad = first_bad + (cares & 1) * 2 * D;
          if (care) tile_wait(noted, cares & 1, limit);
          unsigned g = base;
          // one tile into the ring; its row of the same kind of tile a step on is asked for at once
          auto put = [&](bool value, int j, int page_next) {
            const unsigned slot = g % NS;
            uint8_t* const tile = ring + slot * TB;
            uint8_t* const mine = rows + (value ? 32 * row4_bytes(D) : 0);
            if (g >= NS) tile_wait(&kv_empty[slot], ((g / NS) - 1) & 1, limit);
            ++g;
            // (the row was the last request but one, or the last: the second key tile's and the last value tile's, 64 dims)
            if (EARLY && j == (value ? nk - 1 : 1)) asm volatile("cp.async.wait_group 0;" ::: "memory");
            else asm volatile("cp.async.wait_group 1;" ::: "memory");
            if (ran_out()) return;
            store_row4<T, D>(mine, tile, row0 + lane);
            load_row4<D>(smem_addr(mine), a.s, value ? a.v4 : a.k4, w.kvh, page_next, key0 + (j + 1) * kTileKeys);
            if (value && j >= care_from) {
              __syncwarp();
              take_out<T, D>(tile, row0, row0 + kTileKeys / 4, (w.first + j) * kTileKeys, bad);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&kv_full[slot]);
          };
#pragma unroll 1
          for (int j = 0; j < nk; ++j) {
            put(false, j, page);
            if (EARLY && j > 0) put(true, j - 1, page_v);
            page_v = page;  // of key tile j + 1
            page = row_page4(a.s, w, key0 + (j + 2) * kTileKeys);
            if (!EARLY) put(true, j, page_v);
          }
          if (EARLY) put(true, nk - 1, -1);
          asm volatile("cp.async.wait_group 0;" ::: "memory");
          if (care) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&taken_out[cares & 1]);
            ++cares;
          }
          base += 2 * nk;
        }
        if (care) {
          end_care();
          break;
        }
        if (!go_again()) break;
      }
    }
  } else if (warp >= kTmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Q4 ? 48 : 80));
    if (Q4 && warp == kTmaWarp) {
      // ---- queries
      int k = 0;
      unsigned qn = 0;
      for (bool care = false;; care = true) {
        unsigned cares = 0;
        for (;;) {
          const TileWork w = next_work(k++);
          if (w.b < 0) break;
          if (max(w.steps[0], w.steps[1]) == 0) continue;
          if (qn > 0) tile_wait(q_empty, (qn - 1) & 1, limit);
          if (lane == 0 && limit != 1) {
            const int lo = w.steps[0] > 0 ? 0 : 1, hi = w.steps[1] > 0 ? 2 : 1;
            mbar_arrive_expect_tx(q_full, (hi - lo) * SUB * TPT * a.s.rep * 128);
            for (int i = lo; i < hi; ++i)
              for (int c = 0; c < SUB; ++c)
                tma_load4(smem_addr(smem + i * TB + c * (TB / SUB)), &map_q, q_full, c * 64, 0, w.kvh,
                          w.start + w.tok0 + i * TPT);
          }
          if (!ran_out()) ++qn;
          if (care) {
            if (cares > 1) tile_wait(&notes_read[cares & 1], ((cares >> 1) - 1) & 1, limit);
            for (int e = lane; e < 2 * D; e += 32) first_bad[(cares & 1) * 2 * D + e] = kUnseen;
            __syncwarp();
            if (lane == 0) mbar_arrive(noted);
            ++cares;
          }
        }
        if (ran_out() && qn > 0) {  // the copies land before the memory goes
          unsigned more = kTileWaitLimit;
          tile_wait(q_full, (qn - 1) & 1, more);
        }
        if (care) {
          end_care();
          break;
        }
        if (!go_again()) break;
      }
    } else if (warp == kTmaWarp) {
      // ---- copies
      int k = 0;
      unsigned base = 0, issued = 0, qn = 0, tails = 0;  // ring tiles of earlier items, all issued; queries; mended tiles
      auto pass = [&](const bool with_care) {
        unsigned cares = 0;
        for (;;) {
          const TileWork w = next_work(k++);
          if (w.b < 0) break;
          const int nk = max(w.steps[0], w.steps[1]);
          if (nk == 0) continue;
          if (qn > 0) tile_wait(q_empty, (qn - 1) & 1, limit);
          ++qn;
          // (once a wait has run out nothing is armed or loaded any more)
          if (lane == 0 && limit != 1) {
            // a tile whose queries all lie past the sequence, or that sees no key of the range, is not loaded
            const int lo = w.steps[0] > 0 ? 0 : 1, hi = w.steps[1] > 0 ? 2 : 1;
            mbar_arrive_expect_tx(q_full, (hi - lo) * SUB * TPT * a.s.rep * 128);
            for (int i = lo; i < hi; ++i)
              for (int c = 0; c < SUB; ++c)
                tma_load4(smem_addr(smem + i * TB + c * (TB / SUB)), &map_q, q_full, c * 64, 0, w.kvh,
                          w.start + w.tok0 + i * TPT);
          }
          const int tail = tail_rows_of(w, nk), end = (tail + 15) / 16 * 16;
          const int care_from = with_care ? masked_from(w) : nk;
          int* bad = first_bad + (cares & 1) * 2 * D;
          if (with_care) {
            if (cares > 1) tile_wait(&notes_read[cares & 1], ((cares >> 1) - 1) & 1, limit);
            for (int e = lane; e < 2 * D; e += 32) bad[e] = kUnseen;
            __syncwarp();
          }
          for (int n = 0; n < 2 * nk; ++n) {
            const bool value = !EARLY ? n & 1 : n == 2 * nk - 1 || (n > 0 && !(n & 1));
            const int j = !EARLY ? n / 2 : n == 2 * nk - 1 ? nk - 1 : value ? n / 2 - 1 : (n + 1) / 2;
            const int key0 = (w.first + j) * kTileKeys;
            int row = w.start + key0, page = 0;
            bool mine = lane == 0;
            int boxes = 1;
            if constexpr (PAGED) {
              boxes = (min(kTileKeys, w.len - key0) + a.box_rows - 1) / a.box_rows;
              mine = lane < boxes;
              const int key = key0 + lane * a.box_rows;
              row = key & ((1 << a.s.log_page) - 1);
              // an entry outside the cache is a coordinate outside the tensor: zeros
              if (mine) page = a.s.tables[(long long)w.b * a.s.table_stride + (key >> a.s.log_page)];
            }
            // the last value tile with missing rows, and with care each that has hidden keys, arrives on a barrier of its
            // own and counts as full once its rows are mended
            const bool mend = (n == 2 * nk - 1 && tail < end) || (value && j >= care_from);
            const unsigned g = base + n, slot = g % NS;
            uint64_t* bar = mend ? v_tail : &kv_full[slot];
            if (g >= NS) tile_wait(&kv_empty[slot], ((g / NS) - 1) & 1, limit);
            if (lane == 0 && limit != 1) mbar_arrive_expect_tx(bar, boxes * a.box_rows * SUB * 128);
            __syncwarp();
            if (mine && limit != 1)
              for (int c = 0; c < SUB; ++c)
                tma_load4(smem_addr(ring + slot * TB + c * (TB / SUB)) + lane * a.box_rows * 128, value ? &map_v : &map_k,
                          bar, c * 64, row, w.kvh, page);
            if (mend) {
              tile_wait(v_tail, tails++ & 1, limit);
              for (int e = n < 2 * nk - 1 ? kTileKeys * SUB * 8 : lane; e < (end - tail) * SUB * 8; e += 32) {
                const int r = tail + e / (SUB * 8), c = e % (SUB * 8);
                *reinterpret_cast<uint4*>(ring + slot * TB + (c >> 3) * (TB / SUB) + r * 128 + (c & 7) * 16) =
                    make_uint4(0, 0, 0, 0);
              }
              if (with_care) take_out<T, D>(ring + slot * TB, 0, n < 2 * nk - 1 ? kTileKeys : tail, key0, bad);
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
              if (lane == 0 && limit != 1) mbar_arrive(&kv_full[slot]);
            }
            if (limit != 1) issued = g + 1;  // (a tile that goes to v_tail counts once it has been mended)
          }
          if (with_care) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&taken_out[cares & 1]);
            ++cares;
          }
          base += 2 * nk;
        }
        if (ran_out()) {  // copies in flight land before the memory goes
          unsigned more;
          for (unsigned i = issued > NS ? issued - NS : 0; i < issued; ++i)
            tile_wait(&kv_full[i % NS], (i / NS) & 1, more = kTileWaitLimit);
          if (qn > 0) tile_wait(q_full, (qn - 1) & 1, more = kTileWaitLimit);
          if (tails > 0) tile_wait(v_tail, (tails - 1) & 1, more = kTileWaitLimit);
        }
      };
      // Its code twice at 64 dims (16 prompts of 15001 tokens 180 us, 184 with one), once at 128 dims (a chunk of 512 beside
      // 31 requests 83.6 us, 87 with two: more code to fetch between the other kernels' launches).
      if constexpr (D == 64) {
        pass(false);
        if (go_again()) {
          pass(true);
          end_care();
        }
      } else {
        for (bool care = false;; care = true) {
          pass(care);
          if (care) {
            end_care();
            break;
          }
          if (!go_again()) break;
        }
      }
    } else if (warp == kMmaWarp) {
      // ---- products, tile 0 then tile 1 (a warp per tile was slower: their products then share the tensor cores and
      // both finish late).  The warp waits together; one thread issues a group of products.
      constexpr uint32_t IDESC_S = tile_idesc(kTileKeys, TYPE, 0), IDESC_O = tile_idesc(D, TYPE, 1);
      const uint32_t q_desc = desc_k_major(smem_addr(smem)), k_desc = desc_k_major(smem_addr(ring)),
                     v_desc = desc_n_major(smem_addr(ring), TB / SUB);
      // (Nothing is issued once a wait has run out: a freed slot is loaded again, so what frees it must have seen its last
      // load land.)
      unsigned base = 0, qn = 0, done0 = 0, done1 = 0;  // of earlier items: ring tiles, query loads, steps
      int k = 0;
      for (int passes = 1;; ++passes) {
        for (;;) {
          const TileWork w = next_work(k++);
          if (w.b < 0) {
            if (lane == 0) mbar_arrive(ending);
            break;
          }
          const int nk = max(w.steps[0], w.steps[1]);
          if (nk == 0) {
            if (lane == 0) mbar_arrive(ending);
            continue;
          }
          const int tail_groups = (tail_rows_of(w, nk) + 15) / 16;
          auto full = [&](unsigned n) { return &kv_full[(base + n) % NS]; };
          auto phase = [&](unsigned n) { return (base + n) / NS & 1u; };
          auto scores = [&](int i, unsigned slot) {  // S_i against the key tile in a slot
            const uint32_t qd = q_desc + i * (TB >> 4), kd = k_desc + slot * (TB >> 4);
  #pragma unroll
            for (int c = 0; c < SUB; ++c)
  #pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_ss(tmem + S_COL + i * 128, qd + ((c * (TB / SUB) + kk * 32) >> 4),
                       kd + ((c * (TB / SUB) + kk * 32) >> 4), IDESC_S, c + kk > 0);
            tc_commit(&s_full[i]);
          };
          // keys 64 h .. 64 h + 64 of P_i V with the value tile in a slot
          auto outputs = [&](int i, unsigned slot, int h, bool first, int groups) {
            const uint32_t vd = v_desc + slot * (TB >> 4) + h * 512;
            const uint32_t o = tmem + O_COL + i * D, pr = tmem + P_COL + i * P_STEP + h * 32;
            if (groups == 8) {
  #pragma unroll
              for (int kk = 0; kk < 4; ++kk) mma_ts(o, pr + kk * 8, vd + kk * 128, IDESC_O, !first || h + kk > 0);
            } else {
  #pragma unroll 1
              for (int kk = 0; kk < 4 && 4 * h + kk < groups; ++kk)
                mma_ts(o, pr + kk * 8, vd + kk * 128, IDESC_O, !first || h + kk > 0);
            }
          };
          tile_wait2(q_full, qn & 1, full(0), phase(0), limit);
          if (EARLY && done0 > 0 && w.steps[0] > 0) tile_wait(&s_free[0], (done0 - 1) & 1, limit);
          if (EARLY && done1 > 0 && w.steps[1] > 0) tile_wait(&s_free[1], (done1 - 1) & 1, limit);
          tc_fence_after();
          if (elect_one() && limit != 1) {
            if (w.steps[0] > 0) scores(0, base % NS);
            if (w.steps[1] > 0) scores(1, base % NS);
            tc_commit(&kv_empty[base % NS]);
            if (nk == 1) tc_commit(q_empty);
          }
  #pragma unroll 1
          for (int j = 0; j < nk; ++j) {
            if (j == max(0, nk - 3) && lane == 0) mbar_arrive(ending);
            const unsigned kn = key_at(j + 1), vn = value_at(j, nk);
            const unsigned kslot = (base + kn) % NS, vslot = (base + vn) % NS;
            const int groups = j == nk - 1 ? tail_groups : 8;
            const bool more0 = j + 1 < w.steps[0], more1 = j + 1 < w.steps[1];
            if constexpr (EARLY) {
              // the next scores of both tiles, then the step's P V of each
              if (j + 1 < nk) {
                tile_wait(full(kn), phase(kn), limit);
                if (more0 && more1) tile_wait2(&s_free[0], (done0 + j) & 1, &s_free[1], (done1 + j) & 1, limit);
                else if (more0) tile_wait(&s_free[0], (done0 + j) & 1, limit);
                else tile_wait(&s_free[1], (done1 + j) & 1, limit);
                tc_fence_after();
                if (elect_one() && limit != 1) {
                  if (more0) scores(0, kslot);
                  if (more1) scores(1, kslot);
                  tc_commit(&kv_empty[kslot]);
                  if (j + 1 == nk - 1) tc_commit(q_empty);
                }
              }
  #pragma unroll
              for (int i = 0; i < 2; ++i)
                if (j < w.steps[i]) {
                  const unsigned par = ((i ? done1 : done0) + j) & 1;
                  tile_wait2(&p_full[2 * i + 1], par, full(vn), phase(vn), limit);
                  tc_fence_after();
                  if (elect_one() && limit != 1) {
                    outputs(i, vslot, 0, j == 0, groups);
                    outputs(i, vslot, 1, j == 0, groups);
                    tc_commit(&o_done[i]);
                    if (i == 1 || j >= w.steps[1]) tc_commit(&kv_empty[vslot]);
                  }
                }
            } else {
              // each tile's P V, as its halves come, then its next scores
  #pragma unroll
              for (int i = 0; i < 2; ++i)
                if (j < w.steps[i]) {
                  const unsigned par = ((i ? done1 : done0) + j) & 1;
                  tile_wait2(&p_full[2 * i], par, full(vn), phase(vn), limit);
                  tc_fence_after();
                  if (elect_one() && limit != 1) outputs(i, vslot, 0, j == 0, groups);
                  const bool more = i ? more1 : more0;
                  if (more) tile_wait2(&p_full[2 * i + 1], par, full(kn), phase(kn), limit);
                  else tile_wait(&p_full[2 * i + 1], par, limit);
                  tc_fence_after();
                  if (elect_one() && limit != 1) {
                    outputs(i, vslot, 1, j == 0, groups);
                    tc_commit(&o_done[i]);
                    if (i == 1 || j >= w.steps[1]) tc_commit(&kv_empty[vslot]);
                    if (more) scores(i, kslot);
                    if (more && (i == 1 || !more1)) {
                      tc_commit(&kv_empty[kslot]);
                      if (j + 1 == nk - 1) tc_commit(q_empty);
                    }
                  }
                }
            }
          }
          ++qn;
          base += 2 * nk;
          done0 += w.steps[0];
          done1 += w.steps[1];
        }
        if (passes == 2) {
          end_care();
          break;
        }
        if (!go_again()) break;
      }
    } else if (warp == kTmaWarp + 2) {
      // ---- items: the CTA's own, then those of CTAs that have not started.  Heavy items come first in a launch and the
      // next is taken three steps before the present one ends, so the SMs finish together whatever the lengths are
      // (taken at the present one's start, a prompt of 2048 tokens at 64 dims ran 42 us instead of 33)
      const int splits = item_splits<PAGED>(a);
      int index = (int)blockIdx.x, k = 0, asked = 0, held[2] = {-1, -1};
      auto pass = [&](auto care) {
        constexpr bool CARE = decltype(care)::value;
        for (;; ++k) {
          TileWork w;
          w.b = -1;
          int at = -1;
          if constexpr (CARE) {
            for (int i = 0; i < 2 && at < 0; ++i)
              if (again[i] != 0) at = held[i], held[i] = -1;
          }
          const bool repeat = at >= 0;
          if (!repeat) at = index;
          // (an output that is not finite ends the usual pass: it has come from one of the last two items)
          if (at >= 0 && (CARE || !__any_sync(0xffffffffu, again[0] + again[1] > 0))) w = find_item<PAGED>(a, at, splits);
          if (!CARE && w.b >= 0) held[k & 1] = at;
          if (lane == 0) {
            work[k & 1] = w;
            mbar_arrive(&work_full[k & 1]);
          }
          if (w.b < 0 || ran_out()) break;
          tile_wait2(&work_empty[k & 1], (k >> 1) & 1, ending, k & 1, limit);
          if (ran_out()) break;
          if (repeat) continue;
          if (lane == 0) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the last reply has been read
            mbar_arrive_expect_tx(replied, 16);
            ask_next(smem_addr(reply), replied);
          }
          __syncwarp();
          tile_wait(replied, asked & 1, limit);
          if (ran_out()) {  // (the reply is still to land: once more before the memory goes)
            unsigned more = kTileWaitLimit;
            tile_wait(replied, asked & 1, more);
            break;
          }
          ++asked;
          index = read_next(smem_addr(reply));
          __syncwarp();
        }
      };
      pass(std::false_type{});
      if (go_again()) {
        ++k;
        pass(std::true_type{});
        end_care();
      }
    } else if (go_again()) {
      end_care();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Q4 ? 192 : 208));
    // ---- softmax of tile i: this thread's row
    const int i = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + S_COL + i * 128, o_at = tmem + lanes + O_COL + i * D,
                   p_at = tmem + lanes + P_COL + i * P_STEP;
    const float c = a.s.scale_log2;
    const int row_tok = row / a.s.rep, row_head = row - row_tok * a.s.rep;
    int k = 0, done = 0;  // steps of earlier items
    auto pass = [&](auto care) {
      constexpr bool CARE = decltype(care)::value;
      unsigned cares = 0;
      for (;; ++k) {
        // (the item stays in work[k & 1] until this warp has asked for the next: read again where it is needed)
        tile_wait(&work_full[k & 1], (k >> 1) & 1, limit);
        const volatile TileWork& item = work[k & 1];
        const int first = item.first, my_steps = item.b < 0 || ran_out() ? -1 : item.steps[i];
        const int first_tok = item.tok0 + i * TPT, hidden = item.len - item.n;
        const bool valid = row < TPT * a.s.rep && first_tok + row_tok < item.n;
        const int lim = valid ? hidden + first_tok + row_tok : -1;  // last key the row sees
        const int first_lim = hidden + first_tok;                   // the tile's first row's
        __syncwarp();
        if (lane == 0) mbar_arrive(&work_empty[k & 1]);
        if (my_steps < 0) break;
        float m = -INFINITY, base = 0.f, l = 0.f;  // maximum in use (raw score), m * c or 0, sum against it
        bool s_here = false;
        for (int j = 0; j < my_steps; ++j) {
          if (!s_here) tile_wait(&s_full[i], (done + j) & 1, limit);
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
          const int key0 = (first + j) * kTileKeys;
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
            for (int v = 0; v < 4; ++v) mx[v] = max3(mx[v], x[e + v], x[e + 4 + v]);
          }
  #pragma unroll
          for (int v = 0; v < 4; ++v) mx[v] = max2(mx[v], x[124 + v]);
          // (asked here, used a little later: the answer takes a while)
          [[maybe_unused]] const bool o_here = !EARLY || j == 0 || mbar_test_wait(&o_done[i], (done + j - 1) & 1);
          const float top = max2(max3(mx[0], mx[1], mx[2]), mx[3]);
          // (the difference is NaN for two infinities of one sign and beside a NaN score: no move.  A tile's rows past its
          // queries hold other requests' queries or what shared memory held before: they have no say in when the others'
          // sums are rounded anew)
          if (__any_sync(0xffffffffu, lim >= 0 && (top - m) * c > kLazyLog2)) {
            const float mn = fmaxf(m, top);
            const float nb = mn == -INFINITY ? 0.f : mn * c;
            const float f = m == -INFINITY ? 0.f : exp2_fast(m * c - nb);
            l *= f;  // (0 so far, or NaN, where nothing finite has been seen)
            if (j > 0) {
              tile_wait(&o_done[i], (done + j - 1) & 1, limit);
              tc_fence_after();
  #pragma unroll 1
              for (int g = 0; g < D / 32; ++g) {
                float o[32];
                tmem_ld32(o_at + g * 32, o);
                tmem_ld_wait(o);
  #pragma unroll
                for (int e = 0; e < 32; ++e) o[e] *= f;
                tmem_st32(o_at + g * 32, o);
              }
            }
            m = mn;
            base = nb;
          }
          if constexpr (EARLY) {  // the last P_i V has read P_i
            if (!__all_sync(0xffffffffu, o_here)) tile_wait(&o_done[i], (done + j - 1) & 1, limit);
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
              if (g == 2) s_here = EARLY && j + 1 < my_steps && mbar_test_wait(&s_full[i], (done + j + 1) & 1);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[2 * i + h]);
          }
          s_here = __all_sync(0xffffffffu, s_here);
          float s0, s1;
          unpack2(add2(sum0, sum1), &s0, &s1);
          // a NaN score, or an infinite one (its exponent is infinity - infinity), makes the row NaN
          l = top < INFINITY ? l + (s0 + s1) : NAN;
        }
        // ---- the row's output, or its part of it
        done += my_steps;
        if (my_steps > 0) {
          tile_wait(&o_done[i], (done - 1) & 1, limit);
          tc_fence_after();
        }
        const int tok = first_tok + row_tok, part_at = item.part;
        const bool whole = part_at < 0;
        const bool none = lim < 0;
        const float inv = 1.f / l;
        uint16_t* out = a.s.out + (long long)(item.start + tok) * a.s.sot + (long long)(item.kvh * a.s.rep + row_head) * a.s.soh;
        float* part = a.s.part + tile_part_floats(D) * (whole ? 0 : part_at);
        if (CARE && max(item.steps[0], item.steps[1]) > 0) {
          tile_wait(&taken_out[cares & 1], cares >> 1 & 1, limit);
          if (my_steps > 0) put_back<D>(o_at, first_bad + (cares & 1) * 2 * D, lim);
          __syncwarp();
          if (lane == 0) mbar_arrive(&notes_read[cares & 1]);
          ++cares;
        }
        // a row's outputs go out a 32-byte sector at a time where they start on one (16 prompts of 15001 tokens together:
        // 180 us, 184 with 16-byte stores)
        const bool sectors = __all_sync(0xffffffffu, (reinterpret_cast<uintptr_t>(out) & 31u) == 0);
        float odd = 0.f;  // becomes NaN with the first output that is not finite
        if (my_steps > 0) {
  #pragma unroll 1
          for (int g = 0; g < D / 32; ++g) {
            float o[32];
            tmem_ld32(o_at + g * 32, o);
            tmem_ld_wait(o);
  #pragma unroll
            for (int e = 0; e < 32; ++e) odd = fmaf(o[e], 0.f, odd);
            if (valid && whole) {
  #pragma unroll
              for (int v = 0; v < 2; ++v) {  // 16 dims: a sector
                uint32_t u[8];
  #pragma unroll
                for (int e = 0; e < 8; ++e)
                  u[e] = none ? 0u : Type16<T>::pack(o[v * 16 + 2 * e] * inv, o[v * 16 + 2 * e + 1] * inv);
                uint16_t* to = out + g * 32 + v * 16;
                if (sectors && g * 32 + v * 16 + 16 <= a.s.hd) {
                  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(u[0]), "r"(u[1]),
                               "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                               : "memory");
                } else {
                  if (g * 32 + v * 16 < a.s.hd) *reinterpret_cast<uint4*>(to) = make_uint4(u[0], u[1], u[2], u[3]);
                  if (g * 32 + v * 16 + 8 < a.s.hd) *reinterpret_cast<uint4*>(to + 8) = make_uint4(u[4], u[5], u[6], u[7]);
                }
              }
            } else if (valid) {
  #pragma unroll
              for (int v = 0; v < 8; ++v)
                *reinterpret_cast<float4*>(part + tile_part_at(i * kTileRows + row, g * 32 + v * 4)) =
                    make_float4(o[v * 4], o[v * 4 + 1], o[v * 4 + 2], o[v * 4 + 3]);
            }
            __syncwarp();  // (the next load takes the whole warp)
          }
        } else if (valid && whole) {
          for (int d = 0; d < a.s.hd; d += 8) *reinterpret_cast<uint4*>(out + d) = make_uint4(0, 0, 0, 0);
        }
        float2* ml = reinterpret_cast<float2*>(part + (size_t)2 * kTileRows * D) + i * kTileRows;
        if (!whole && valid) ml[row] = m == -INFINITY ? make_float2(-INFINITY, l) : make_float2(base, l);
        // an output that is not finite though the row's sum is: it may come from values that the row must not see
        if (!CARE && valid && !none && my_steps > 0 && isfinite(l) && !(odd == 0.f)) again[k & 1] = 1;
        __syncwarp();
      }
    };
    pass(std::false_type{});
    if (go_again()) {
      ++k;
      pass(std::true_type{});
      end_care();
    }
  }
  if (ran_out() && lane == 0) atomicOr(&g_tile_device_error, 256u);
  if (warp == kMmaWarp) {
    if (gave_up[0] + gave_up[1] > 0) {  // MMAs in flight finish before the memory goes
      unsigned more = kTileWaitLimit;
      if (elect_one()) tc_commit(drained);
      tile_wait(drained, 0, more);
    }
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
  }
}

// Joins the ranges of keys of an item, 32 of its rows per CTA; returns at once where the launch did not split.
template <typename T, int D, bool PAGED, typename ArgsT>
__global__ void __launch_bounds__(256) tile_join_kernel(const __grid_constant__ ArgsT a) {
  __shared__ TileWork s_work;
  __shared__ int s_splits;
  pdl_launch_dependents();
  pdl_wait_primary();
  if (threadIdx.x < 32) {
    const int splits = item_splits<PAGED>(a);
    TileWork w;
    w.b = -1;
    if (splits > 1) w = find_item<PAGED>(a, (int)blockIdx.x * splits, splits);
    if (threadIdx.x == 0) {
      s_work = w;
      s_splits = splits;
    }
  }
  __syncthreads();
  const TileWork w = s_work;
  if (w.b < 0) return;
  const int splits = s_splits;
  const int r = blockIdx.y * 32 + (threadIdx.x & 31), i = r >> 7, row = r & 127;  // a lane is a row, a warp some dims
  constexpr int W = D / 8;
  const int d0 = (threadIdx.x >> 5) * W;
  const int row_tok = row / a.s.rep, tok = w.tok0 + i * a.tokens_per_tile + row_tok;
  if (row >= a.tokens_per_tile * a.s.rep || tok >= w.n || d0 >= a.s.hd) return;
  const float* part = a.s.part + tile_part_floats(D) * ((size_t)blockIdx.x * splits);
  float M = -INFINITY;
  for (int p = 0; p < splits; ++p)
    M = fmaxf(M, __ldcg(part + p * tile_part_floats(D) + (size_t)2 * kTileRows * D + r * 2));
  float L = 0.f, o[W];
#pragma unroll
  for (int e = 0; e < W; ++e) o[e] = 0.f;
  for (int p = 0; p < splits; ++p) {
    const float* q = part + p * tile_part_floats(D);
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(q + (size_t)2 * kTileRows * D) + r);
    if (ml.x == -INFINITY && ml.y == 0.f) continue;  // saw no key: its outputs were not written
    const float f = exp2_fast(ml.x - M);
    L += f * ml.y;
#pragma unroll
    for (int e = 0; e < W; e += 4) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(q + tile_part_at(r, d0 + e)));
      o[e] += f * v.x;
      o[e + 1] += f * v.y;
      o[e + 2] += f * v.z;
      o[e + 3] += f * v.w;
    }
  }
  const bool none = w.len - w.n + tok < 0;
  const float inv = 1.f / L;
  uint16_t* out = a.s.out + (long long)(w.start + tok) * a.s.sot +
                  (long long)(w.kvh * a.s.rep + row - row_tok * a.s.rep) * a.s.soh + d0;
#pragma unroll
  for (int e = 0; e < W; e += 8) {
    if (d0 + e >= a.s.hd) break;
    uint4 u;
    u.x = Type16<T>::pack(o[e] * inv, o[e + 1] * inv);
    u.y = Type16<T>::pack(o[e + 2] * inv, o[e + 3] * inv);
    u.z = Type16<T>::pack(o[e + 4] * inv, o[e + 5] * inv);
    u.w = Type16<T>::pack(o[e + 6] * inv, o[e + 7] * inv);
    *reinterpret_cast<uint4*>(out + e) = none ? make_uint4(0, 0, 0, 0) : u;
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

template <typename T, int D, bool PAGED, typename ArgsT>
static int launch_tile(const ArgsT& a, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                       unsigned grid, cudaStream_t stream) {
  const int smem = tile_smem_bytes(D) + (kTileInt4<ArgsT> ? rows4_bytes(D) : 0);
  static std::mutex mu;
  static std::vector<int> done_dev;  // of this kernel
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    bool seen = false;
    for (int d : done_dev) seen |= (d == dev);
    if (!seen) {
      const int rc = check_cuda(cudaFuncSetAttribute(tile_attention_kernel<T, D, PAGED, ArgsT>,
                                                     cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                                "attention: shared memory limit");
      if (rc != LI4_OK) return rc;
      done_dev.push_back(dev);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(kTileInt4<ArgsT> ? kTile4Threads : kTileThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int rc = check_cuda(cudaLaunchKernelEx(&cfg, tile_attention_kernel<T, D, PAGED, ArgsT>, a, q, k, v),
                      "attention: kernel launch");
  if (rc != LI4_OK || a.part_slots == 0) return rc;
  cfg.gridDim = dim3((unsigned)a.part_slots / 2, 2 * kTileRows / 32, 1);  // (a split item has two parts at least)
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = 0;
  return check_cuda(cudaLaunchKernelEx(&cfg, tile_join_kernel<T, D, PAGED, ArgsT>, a), "attention: kernel launch");
}

// Items whose partial results the workspace has room for: one per SM, where the pairs of tiles that the tokens alone
// make do not fill the SMs and some sequence may have enough keys to cut.  (Up to two per SM, a chunk of 512 tokens beside
// 31 decoding requests took 113 us instead of 100, one of 128 tokens over 32000 keys 74 instead of 67.)
static int tile_part_slots(int rep, int64_t tokens, int64_t kv_heads, int64_t max_keys, int sm) {
  const int64_t pairs = tokens / (2 * (kTileRows / rep));
  return pairs * kv_heads >= sm || max_keys <= kTileMinSteps * kTileKeys ? 0 : sm;
}
size_t tile_attention_part_bytes(int hd, int rep, int64_t tokens, int64_t kv_heads, int64_t max_keys, int sm) {
  return (size_t)tile_part_slots(rep, tokens, kv_heads, max_keys, sm) * tile_part_floats(hd <= 64 ? 64 : 128) *
         sizeof(float);
}

// Poll limit of the kernel's waits in later launches, for tests (0: the default).
static std::atomic<unsigned> g_tile_wait_polls{0};
int tile_set_wait_limit(unsigned polls) {
  g_tile_wait_polls = polls == 1 ? 2 : polls;  // (a limit of 1 says that a wait has run out)
  return LI4_OK;
}

// What both launches share: queries' map, work limits; the grid, or 0 and a status.
static int plan_tiles(TileArgs& a, bool paged, int dtype, CUtensorMap* q, unsigned* grid_out) {
  const SeqAttnArgs& args = a.s;
  const int rep = args.rep;
  a.tokens_per_tile = kTileRows / rep;
  // queries [token][KV head][head of the group][d]: a box is the rep rows of tokens_per_tile tokens
  const int rc = make_map(q, dtype, args.q, args.hd, rep, args.sqh, args.Hkv, args.sqh * rep, args.T, args.sqt, rep,
                          a.tokens_per_tile);
  if (rc != LI4_OK) return rc;
  a.part_slots = tile_part_slots(rep, args.T, args.Hkv, args.max_keys, current_sm_count());
  const unsigned polls = g_tile_wait_polls.load();
  a.wait_limit = polls != 0 ? polls : kTileWaitLimit + kTileWaitStep * (unsigned)((paged ? args.max_keys : args.T) / kTileKeys);
  const int64_t pairs = args.T / (2 * a.tokens_per_tile) + args.B;  // at least the sequences' pairs of tiles
  int64_t grid = pairs * args.Hkv;
  if (grid < a.part_slots) grid = a.part_slots;
  if (grid > 0x7fffffff) return set_error(LI4_ERR_UNSUPPORTED, "attention: too many items");
  *grid_out = (unsigned)grid;
  return LI4_OK;
}

int launch_tile_attention(const SeqAttnArgs& args, bool paged, int dtype, cudaStream_t stream) {
  TileArgs a;
  a.s = args;
  const int page = 1 << args.log_page;
  a.box_rows = paged ? (page < kTileKeys ? page : kTileKeys) : kTileKeys;
  CUtensorMap q, k, v;
  unsigned g = 0;
  int rc = plan_tiles(a, paged, dtype, &q, &g);
  const int64_t y = paged ? page : args.T, w = paged ? args.num_pages : 1;
  if (rc == LI4_OK)
    rc = make_map(&k, dtype, args.k, args.hd, y, args.skt, args.Hkv, args.skh, w, args.skp, a.box_rows, 1);
  if (rc == LI4_OK)
    rc = make_map(&v, dtype, args.v, args.hd, y, args.svt, args.Hkv, args.svh, w, args.svp, a.box_rows, 1);
  if (rc != LI4_OK) return rc;
  const bool half = dtype == LI4_F16;
  if (args.hd <= 64) {
    if (paged) return half ? launch_tile<__half, 64, true>(a, q, k, v, g, stream) : launch_tile<__nv_bfloat16, 64, true>(a, q, k, v, g, stream);
    return half ? launch_tile<__half, 64, false>(a, q, k, v, g, stream) : launch_tile<__nv_bfloat16, 64, false>(a, q, k, v, g, stream);
  }
  if (paged) return half ? launch_tile<__half, 128, true>(a, q, k, v, g, stream) : launch_tile<__nv_bfloat16, 128, true>(a, q, k, v, g, stream);
  return half ? launch_tile<__half, 128, false>(a, q, k, v, g, stream) : launch_tile<__nv_bfloat16, 128, false>(a, q, k, v, g, stream);
}

int launch_tile_attention_int4(const Seq4Args& args, int dtype, cudaStream_t stream) {
  Tile4Args a;
  a.s = args;
  a.box_rows = 0;
  a.k4 = args.k4;
  a.v4 = args.v4;
  CUtensorMap q;
  unsigned g = 0;
  const int rc = plan_tiles(a, true, dtype, &q, &g);
  if (rc != LI4_OK) return rc;
  const bool half = dtype == LI4_F16;  // (no maps of keys and values: the queries' stands in their places)
  if (args.hd <= 64)
    return half ? launch_tile<__half, 64, true>(a, q, q, q, g, stream) : launch_tile<__nv_bfloat16, 64, true>(a, q, q, q, g, stream);
  return half ? launch_tile<__half, 128, true>(a, q, q, q, g, stream) : launch_tile<__nv_bfloat16, 128, true>(a, q, q, q, g, stream);
}

}  // namespace li4
