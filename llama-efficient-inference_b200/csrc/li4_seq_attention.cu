// li4_seq_attention.cu -- attention of packed sequences over paged or packed keys, sm_100a.
//
// Grouped-query attention by rows: the rep query heads of a KV head, over the queries of a sequence,
// are the rows of one matrix (row = query * rep + head), so a KV head's keys and values are read once
// for the whole group.  An item is (sequence, tile of 8 NT rows, KV head); its keys come in units of
// 128 (64 dims) or 64 (128 dims).  Units of all items lie on one line; CTA g of G takes the g-th equal
// share of it, whatever the lengths are (they are read on the device: the host knows none).  A CTA that
// covers only a part of an item's keys leaves (running maximum, sum, unnormalised output) in `part`, and
// a second launch joins the parts in key order, so the result does not depend on timing.
//
// Inside a CTA each of the 4 warps streams its own quarter of every unit through its own ring of
// shared-memory stages (cp.async; no CTA barrier until the end): S^T = K Q^T and O^T += V^T P^T as
// m16n8k16 tensor-core tiles, softmax in fp32 in registers with the running maximum and sum of one
// pass.  The keys are the 16-wide side and the rows the 8-wide one, so a group of 4 or 8 heads wastes
// half of a tile or nothing (with the rows as the 16-wide side 64 requests of 300-16000 tokens took
// 85 us instead of 81).  The work is bound by the bytes of the keys and values as long as the rows
// are few: those 419 MB now take 77 us, 5.5 TB/s with the join, and with the products left out no less.
//
// A masked key's probability is zero, but zero times a NaN or an infinity is NaN.  In the steps with keys that some
// row must not see (the last tokens' own), a value that is not finite is therefore taken out of the warp's stage before
// the product and added to the rows that see it (a sum with what is not finite does not depend on its weight).
#include <cooperative_groups.h>

#include <mutex>
#include <utility>
#include <vector>

#include "li4_attention_args.cuh"
#include "li4_gemv_device.cuh"

namespace li4 {

namespace cg = cooperative_groups;

constexpr int kSeqThreads = 128;
constexpr int kSeqWarps = 4;
constexpr int kSeqStages = 3;   // stages per warp
// Keys of a warp's stage: 8 KB of keys and values, 96 KB of stages per CTA, two CTAs per SM (while one joins its warps or
// starts an item the other's copies go on: one CTA of 32-key stages at 128 dims, 32 requests of 1000-8000 tokens 81 us
// instead of 75).
__host__ __device__ constexpr int seq_keys(int D) { return 32 * 64 / D; }
__host__ __device__ constexpr int seq_unit(int D) { return kSeqWarps * seq_keys(D); }  // keys per unit
__host__ __device__ constexpr int seq_stage_bytes(int D) { return 2 * seq_keys(D) * D * 2; }
__host__ __device__ constexpr int seq_smem_bytes(int D) { return kSeqWarps * kSeqStages * seq_stage_bytes(D); }
// floats of one partial result: 8 NT rows of D outputs, then (maximum, sum) per row
__host__ __device__ constexpr int seq_part_floats(int D, int NT) { return 8 * NT * (D + 2); }

// The line of units.  An item takes kItemUnits more than its keys do: starting it and joining its warps cost about that
// much time (256 requests of 100-4000 tokens: 143 us without, 108 with 4, 107 with 2, 109 with 6; 64 of
// 300-16000 tokens 81, 77, 79, 78 us).
constexpr int kItemUnits = 4;
struct Line {
  long long total;
  int active;  // CTAs that get a share
};
__device__ __forceinline__ long long share(const Line& l, int g) { return l.total * g / l.active; }

// Key units of an item and the units that a sequence takes.
template <int D, int NT>
__device__ __forceinline__ long long seq_units(const SeqAttnArgs& a, const Seq& s, int* tiles, int* per) {
  *tiles = (int)(((long long)s.n * a.rep + 8 * NT - 1) / (8 * NT));
  *per = max(1, (s.len + seq_unit(D) - 1) / seq_unit(D));
  return (long long)*tiles * (*per + kItemUnits) * a.Hkv;
}

// Finds the sequence that holds unit share(g): each thread sums a slice of the sequences.  Every thread
// returns the line, the sequence and the units before it (b = -1: no share).
template <int D, int NT, bool PAGED>
__device__ Line find_share(const SeqAttnArgs& a, int g, int* b_out, long long* before) {
  __shared__ long long s_sum[kSeqWarps];
  __shared__ int s_b;
  __shared__ long long s_before;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.B + kSeqThreads - 1) / kSeqThreads;
  const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
  long long mine = 0;
  int tiles, units;
  for (int b = b0; b < b1; ++b) mine += seq_units<D, NT>(a, load_seq<PAGED>(a, b), &tiles, &units);
  long long incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += x;
  }
  if (lane == 31) s_sum[warp] = incl;
  if (tid == 0) s_b = -1;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kSeqWarps; ++w) {
    if (w < warp) incl += s_sum[w];
    total += s_sum[w];
  }
  Line line;
  line.total = total;
  line.active = (int)min((long long)a.grid, max(1LL, total));
  if (g < line.active && total > 0) {
    const long long at = share(line, g);
    long long excl = incl - mine;
    if (at >= excl && at < incl) {
      for (int b = b0; b < b1; ++b) {
        const long long u = seq_units<D, NT>(a, load_seq<PAGED>(a, b), &tiles, &units);
        if (at < excl + u) {
          s_b = b;
          s_before = excl;
          break;
        }
        excl += u;
      }
    }
  }
  __syncthreads();
  *b_out = s_b;
  *before = s_before;
  return line;
}

__device__ __forceinline__ void cp_async16z(uint32_t dst, const void* src, bool have) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(have ? 16 : 0) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16816(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  mma_16816(c, a[0], a[1], a[2], a[3], b0, b1);
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 8x8 values of 16 bits across the warp, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// The pages of a stage's keys from j0, 8 keys each (a page has 8 rows at least and j0 is a multiple of 16, so 8 keys share one);
// asked for a stage ahead of their copy, as the block table's answer takes a trip to L2.  -1: past the end.
template <int D>
struct KeyPages {
  int page[seq_keys(D) / 8];
};
template <int D, bool PAGED>
__device__ __forceinline__ KeyPages<D> key_pages(const SeqAttnArgs& a, int b, int j0, int end) {
  KeyPages<D> k;
#pragma unroll
  for (int q = 0; q < seq_keys(D) / 8; ++q) {
    k.page[q] = -1;
    if (j0 + 8 * q < end)
      k.page[q] = PAGED ? a.tables[(long long)b * a.table_stride + ((j0 + 8 * q) >> a.log_page)] : 0;
  }
  return k;
}

// A stage's keys: K rows then V rows, 16-byte chunk c of row r at c ^ (r & 7).  Rows past the end and
// rows of no page are zeros.
template <int D, bool PAGED>
__device__ __forceinline__ void load_stage(const SeqAttnArgs& a, const KeyPages<D>& kp, const Seq& s, int kvh, int j0, int end,
                                           uint32_t stage) {
  constexpr int CH = D / 8;           // chunks per row
  constexpr int RPI = 32 / CH;        // rows per instruction of the warp
  const int lane = threadIdx.x & 31;
  const int c = lane % CH, r0 = lane / CH;
  const bool in_head = c * 8 < a.hd;
  const uint16_t* k = a.k + (long long)kvh * a.skh + (long long)r0 * a.skt + c * 8;
  const uint16_t* v = a.v + (long long)kvh * a.svh + (long long)r0 * a.svt + c * 8;
#pragma unroll
  for (int q = 0; q < seq_keys(D) / 8; ++q) {
    const int row = PAGED ? (j0 + 8 * q) & ((1 << a.log_page) - 1) : s.start + j0 + 8 * q;
    const long long page = PAGED ? kp.page[q] : 0;
    const bool have = (PAGED ? (unsigned)kp.page[q] < (unsigned)a.num_pages : kp.page[q] == 0) && in_head;
    const uint16_t* kq = k + page * a.skp + (long long)row * a.skt;
    const uint16_t* vq = v + page * a.svp + (long long)row * a.svt;
#pragma unroll
    for (int i = 0; i < 8 / RPI; ++i) {
      const int r = q * 8 + i * RPI + r0;
      const bool ok = have && j0 + r < end;
      const uint32_t at = stage + r * (D * 2) + ((c ^ (r & 7)) << 4);
      cp_async16z(at, ok ? kq + (long long)(i * RPI) * a.skt : a.q, ok);  // (not read where !ok)
      cp_async16z(at + seq_keys(D) * D * 2, ok ? vq + (long long)(i * RPI) * a.svt : a.q, ok);
    }
  }
}

// CL: few requests of short contexts.  A cluster of CTAs takes all keys of a (request, KV head) and joins its parts through
// distributed shared memory, so there is no second launch (see seq_cluster).
template <typename T, int D, int NT, bool PAGED, bool CL>
__global__ void __launch_bounds__(kSeqThreads) seq_attention_kernel(const __grid_constant__ SeqAttnArgs a) {
  constexpr int RT = 8 * NT;
  constexpr int KS = D / 16;  // k steps of K Q^T
  constexpr int DT = D / 16;  // 16-dim tiles of the output
  constexpr int KW = seq_keys(D), KT = KW / 16, UNIT = seq_unit(D);  // a warp's keys per stage, their 16-key tiles
  constexpr int LD = D + 8;   // floats per row of the warps' outputs in shared memory
  static_assert((kSeqWarps * RT * LD + RT * (D + 2)) * 4 <= seq_smem_bytes(D), "outputs and a part fit the ring");
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ float s_ml[kSeqWarps][RT][2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ring = smem_addr(smem) + warp * kSeqStages * seq_stage_bytes(D);
  pdl_launch_dependents();
  pdl_wait_primary();

  const int g = blockIdx.x;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = CL ? (int)cluster.block_rank() : 0, ranks = CL ? (int)cluster.num_blocks() : 1;
  int b;
  long long left, rem;  // units of the share left; units into sequence b (CL: tiles left; tiles done)
  Seq s;
  int tiles, per;
  if constexpr (CL) {
    b = g / ranks / a.Hkv;
    s = load_seq<PAGED>(a, b);
    seq_units<D, NT>(a, s, &tiles, &per);
    left = tiles;
    rem = 0;
  } else {
    long long before;
    const Line line = find_share<D, NT, PAGED>(a, g, &b, &before);
    if (b < 0) return;
    const long long at0 = share(line, g);
    left = share(line, g + 1) - at0;
    rem = at0 - before;
    s = load_seq<PAGED>(a, b);
    seq_units<D, NT>(a, s, &tiles, &per);
  }

  while (left > 0) {
    int kvh, tile, u0, u1, r0 = 0, r1 = 0;  // key units; units of the item
    if constexpr (CL) {
      kvh = g / ranks % a.Hkv;
      tile = (int)rem;
      u0 = per * rank / ranks;
      u1 = per * (rank + 1) / ranks;
    } else {
      const int span = per + kItemUnits, item = (int)(rem / span);
      r0 = (int)(rem - (long long)item * span);
      r1 = (int)min((long long)span, r0 + left);
      u0 = max(0, r0 - kItemUnits);
      u1 = max(0, r1 - kItemUnits);
      kvh = item % a.Hkv;
      tile = item / a.Hkv;
    }
    const int row0 = tile * RT;
    const int rows = min(RT, s.n * a.rep - row0);
    const int first_lim = s.len - s.n + row0 / a.rep;               // last key the tile's first query sees
    const int last_lim = s.len - s.n + (row0 + rows - 1) / a.rep;   // and its last query
    const int k0 = u0 * UNIT, k1 = min(min(u1 * UNIT, s.len), last_lim + 1);

    // ---- the warp's keys: k0 + KW warp + UNIT i, their first stages under way
    const int w0 = k0 + warp * KW;
    const int steps = w0 < k1 ? (k1 - w0 + UNIT - 1) / UNIT : 0;
    KeyPages<D> pages[kSeqStages];
#pragma unroll
    for (int i = 0; i < kSeqStages; ++i) pages[i] = key_pages<D, PAGED>(a, b, w0 + i * UNIT, k1);
#pragma unroll
    for (int i = 0; i < kSeqStages - 1; ++i) {
      if (i < steps) load_stage<D, PAGED>(a, pages[i], s, kvh, w0 + i * UNIT, k1, ring + i * seq_stage_bytes(D));
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    KeyPages<D> next_pages = pages[kSeqStages - 1];

    // ---- queries as B fragments (n = row, k = dim); rows past the tile are zero rows
    uint32_t qf[NT][KS][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + lane / 4;
      const bool valid = r < rows;
      const int pr = row0 + (valid ? r : 0), tok = pr / a.rep;
      const uint16_t* q = a.q + (long long)(s.start + tok) * a.sqt + (long long)(kvh * a.rep + pr - tok * a.rep) * a.sqh;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int d = ks * 16 + c * 8 + (lane & 3) * 2;
          qf[nt][ks][c] = valid && d < a.hd ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
        }
    }
    // ---- this thread's rows of the scores and outputs: nt * 8 + (lane & 3) * 2 + {0, 1}
    int lim[NT][2];
    float o[DT][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = nt * 8 + (lane & 3) * 2 + e;
        lim[nt][e] = r < rows ? s.len - s.n + (row0 + r) / a.rep : -1;
        m[nt][e] = -INFINITY;
        l[nt][e] = 0.f;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt][nt][0] = o[dt][nt][1] = o[dt][nt][2] = o[dt][nt][3] = 0.f;
    }

    int slot = 0;
    for (int i = 0; i < steps; ++i) {
      const int ahead = i + kSeqStages - 1;
      int next = slot + kSeqStages - 1;
      if (next >= kSeqStages) next -= kSeqStages;
      __syncwarp();
      if (ahead < steps)
        load_stage<D, PAGED>(a, next_pages, s, kvh, w0 + ahead * UNIT, k1, ring + next * seq_stage_bytes(D));
      asm volatile("cp.async.commit_group;" ::: "memory");
      next_pages = key_pages<D, PAGED>(a, b, w0 + (ahead + 1) * UNIT, k1);
      asm volatile("cp.async.wait_group %0;" ::"n"(kSeqStages - 1) : "memory");
      __syncwarp();
      const uint32_t ks_at = ring + slot * seq_stage_bytes(D), vs_at = ks_at + KW * D * 2;
      const int j0 = w0 + i * UNIT;
      slot = slot + 1 == kSeqStages ? 0 : slot + 1;

      // S^T: KW keys x 8 NT rows
      float sc[KT][NT][4];
#pragma unroll
      for (int mt = 0; mt < KT; ++mt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[mt][nt][0] = sc[mt][nt][1] = sc[mt][nt][2] = sc[mt][nt][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {  // 16 keys x 16 dims: four 8x8 matrices
          uint32_t kf[4];
          const int r = mt * 16 + (lane & 15), c = ks * 2 + (lane >> 4);
          ldmatrix_x4(kf, ks_at + r * (D * 2) + ((c ^ (r & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<T>(sc[mt][nt], kf, qf[nt][ks][0], qf[nt][ks][1]);
        }
      }
      if (j0 + KW - 1 > first_lim || j0 + KW > k1) {  // some key of them is hidden from some row
#pragma unroll
        for (int mt = 0; mt < KT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = j0 + mt * 16 + (e >> 1) * 8 + lane / 4;
              sc[mt][nt][e] = j > lim[nt][e & 1] || j >= k1 ? -INFINITY : sc[mt][nt][e] * a.scale_log2;
            }
      } else {
#pragma unroll
        for (int mt = 0; mt < KT; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[mt][nt][e] *= a.scale_log2;
      }
      uint32_t pf[KT][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float base[2], keep[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(sc[0][nt][e], sc[0][nt][e + 2]);
          if constexpr (KT == 2) mx = fmaxf(mx, fmaxf(sc[KT - 1][nt][e], sc[KT - 1][nt][e + 2]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mn = fmaxf(m[nt][e], mx);
          base[e] = mn == -INFINITY ? 0.f : mn;  // nothing seen yet: every probability is exp2(-inf) = 0
          keep[e] = exp2_fast(m[nt][e] - base[e]);
          m[nt][e] = mn;
          l[nt][e] *= keep[e];
        }
        if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[dt][nt][e] *= keep[e & 1];
        }
#pragma unroll
        for (int mt = 0; mt < KT; ++mt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sc[mt][nt][e] = exp2_fast(sc[mt][nt][e] - base[e & 1]);
            l[nt][e & 1] += sc[mt][nt][e];
          }
          // [key][row] as the scores lie -> [row][key] as a B fragment wants it
          pf[mt][nt][0] = transpose8(Type16<T>::pack(sc[mt][nt][0], sc[mt][nt][1]));
          pf[mt][nt][1] = transpose8(Type16<T>::pack(sc[mt][nt][2], sc[mt][nt][3]));
        }
      }
      if (j0 + KW - 1 > first_lim) {
        uint8_t* vs = smem + (vs_at - smem_addr(smem));
        unsigned bad = 0;  // hidden keys of the stage with a value that is not finite
        constexpr int CH = D / 8;
#pragma unroll
        for (int i = 0; i < KW * CH / 32; ++i) {
          const int r = (i * 32 + lane) / CH, c = lane % CH;
          const uint4 v = *reinterpret_cast<const uint4*>(vs + r * (D * 2) + ((c ^ (r & 7)) << 4));
          const uint32_t u[4] = {v.x, v.y, v.z, v.w};
          bool odd = false;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            odd |= Type16<T>::not_finite((uint16_t)u[e]) || Type16<T>::not_finite((uint16_t)(u[e] >> 16));
          if (odd && j0 + r > first_lim) bad |= 1u << r;
        }
        bad = __reduce_or_sync(0xffffffffu, bad);
        for (unsigned rest = bad; rest != 0; rest &= rest - 1) {
          const int r = __ffs(rest) - 1;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c = dt * 2 + h;  // dim dt * 16 + 8 h + lane / 4
              uint16_t* at = reinterpret_cast<uint16_t*>(vs + r * (D * 2) + ((c ^ (r & 7)) << 4)) + lane / 4;
              const uint16_t x = *at;
              __syncwarp();
              if (Type16<T>::not_finite(x)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int e = 0; e < 2; ++e)
                    if (j0 + r <= lim[nt][e]) o[dt][nt][2 * h + e] += Type16<T>::unpack(x).x;
                *at = 0;
              }
            }
        }
        if (bad != 0) __syncwarp();
      }
      // O^T += V^T P^T: 16 dims x 16 keys by four transposed 8x8 matrices
#pragma unroll
      for (int mt = 0; mt < KT; ++mt)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          uint32_t vf[4];
          const int r = mt * 16 + (lane >> 4) * 8 + (lane & 7), c = dt * 2 + ((lane >> 3) & 1);
          ldmatrix_x4_trans(vf, vs_at + r * (D * 2) + ((c ^ (r & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<T>(o[dt][nt], vf, pf[mt][nt][0], pf[mt][nt][1]);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // every warp is done with its ring: the outputs may use it

    // ---- join the four warps
    float* so = reinterpret_cast<float*>(smem) + warp * RT * LD;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = nt * 8 + (lane & 3) * 2 + e;
        float sum = l[nt][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (lane < 4) {
          s_ml[warp][r][0] = m[nt][e];
          s_ml[warp][r][1] = sum;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          so[r * LD + dt * 16 + lane / 4] = o[dt][nt][e];
          so[r * LD + dt * 16 + 8 + lane / 4] = o[dt][nt][e + 2];
        }
      }
    __syncthreads();
    const bool whole = !CL && r0 == 0 && r1 == per + kItemUnits;
    // where a part of the item's result goes: the workspace, or this CTA's shared memory past the warps' outputs
    float* part = CL ? reinterpret_cast<float*>(smem) + kSeqWarps * RT * LD
                     : a.part + (size_t)(2 * g + (r0 == 0 ? 1 : 0)) * seq_part_floats(D, NT);
    const float* all = reinterpret_cast<const float*>(smem);
    for (int e = tid; e < RT * D / 2; e += kSeqThreads) {
      const int r = e / (D / 2), d = (e - r * (D / 2)) * 2;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kSeqWarps; ++w) M = fmaxf(M, s_ml[w][r][0]);
      const float base = M == -INFINITY ? 0.f : M;
      float L = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < kSeqWarps; ++w) {
        const float f = exp2_fast(s_ml[w][r][0] - base);
        const float2 ov = *reinterpret_cast<const float2*>(all + (w * RT + r) * LD + d);
        L += f * s_ml[w][r][1];
        x += f * ov.x;
        y += f * ov.y;
      }
      if (r >= rows) continue;
      if (whole) {
        const int pr = row0 + r, tok = pr / a.rep;
        const bool none = s.len - s.n + tok < 0;  // a row that sees no key is zero
        const float inv = none ? 0.f : 1.f / L;
        if (d < a.hd)
          *reinterpret_cast<uint32_t*>(a.out + (long long)(s.start + tok) * a.sot +
                                       (long long)(kvh * a.rep + pr - tok * a.rep) * a.soh + d) =
              none ? 0u : Type16<T>::pack(x * inv, y * inv);
      } else {
        *reinterpret_cast<float2*>(part + r * D + d) = make_float2(x, y);
        if (d == 0) *reinterpret_cast<float2*>(part + RT * D + r * 2) = make_float2(M, L);
      }
    }
    __syncthreads();
    if constexpr (CL) {
      cluster.sync();  // every CTA's part is there
      for (int e = rank * kSeqThreads + tid; e < rows * (D / 2); e += ranks * kSeqThreads) {
        const int r = e / (D / 2), d = (e - r * (D / 2)) * 2;
        float M = -INFINITY;
        for (int c = 0; c < ranks; ++c) M = fmaxf(M, cluster.map_shared_rank(part, c)[RT * D + r * 2]);
        const float base = M == -INFINITY ? 0.f : M;
        float L = 0.f, x = 0.f, y = 0.f;
#pragma unroll 4
        for (int c = 0; c < ranks; ++c) {
          const float* pc = cluster.map_shared_rank(part, c);
          const float2 ml = *reinterpret_cast<const float2*>(pc + RT * D + r * 2);
          const float2 ov = *reinterpret_cast<const float2*>(pc + r * D + d);
          const float f = exp2_fast(ml.x - base);
          L += f * ml.y;
          x += f * ov.x;
          y += f * ov.y;
        }
        const int pr = row0 + r, tok = pr / a.rep;
        const float inv = 1.f / L;
        if (d < a.hd)
          *reinterpret_cast<uint32_t*>(a.out + (long long)(s.start + tok) * a.sot +
                                       (long long)(kvh * a.rep + pr - tok * a.rep) * a.soh + d) =
              s.len - s.n + tok < 0 ? 0u : Type16<T>::pack(x * inv, y * inv);
      }
      cluster.sync();  // read by every CTA: the memory may go
      --left;
      ++rem;
      continue;
    }
    left -= r1 - r0;
    rem += r1 - r0;
    while (left > 0 && rem >= (long long)tiles * (per + kItemUnits) * a.Hkv) {
      rem -= (long long)tiles * (per + kItemUnits) * a.Hkv;
      s = load_seq<PAGED>(a, ++b);
      seq_units<D, NT>(a, s, &tiles, &per);
    }
  }
}

// Joins the parts of the item that the boundary between CTAs blockIdx.x and blockIdx.x + 1 cuts, if it is the
// first boundary inside that item; blockIdx.y takes a share of its outputs.  The parts' weights come first, all loads in
// flight together, then the outputs.
constexpr int kJoinShares = 4;
template <typename T, int D, int NT, bool PAGED>
__global__ void __launch_bounds__(kSeqThreads) seq_attention_join_kernel(const __grid_constant__ SeqAttnArgs a) {
  constexpr int RT = 8 * NT;
  extern __shared__ float s_w[];  // [parts][RT] weight of a part in a row's output
  pdl_launch_dependents();
  pdl_wait_primary();
  const int g = blockIdx.x + 1;
  int b;
  long long before;
  const Line line = find_share<D, NT, PAGED>(a, g, &b, &before);
  if (b < 0) return;
  const Seq s = load_seq<PAGED>(a, b);
  int tiles, per;
  seq_units<D, NT>(a, s, &tiles, &per);
  const long long rem = share(line, g) - before;
  const int span = per + kItemUnits, item = (int)(rem / span);
  const long long start = before + (long long)item * span, end = start + span;
  if (start == share(line, g) || share(line, g - 1) > start) return;
  // the parts are CTAs g - 1 (from the item's start) and g .. last, the last CTA with share(last) < end
  const int last = (int)min((long long)line.active - 1, (end * line.active - 1) / line.total);
  const int kvh = item % a.Hkv, row0 = item / a.Hkv * RT;
  const int rows = min(RT, s.n * a.rep - row0);
  const float* first = a.part + (size_t)(2 * (g - 1) + 1) * seq_part_floats(D, NT);
  const float* rest = a.part + (size_t)(2 * g) * seq_part_floats(D, NT);
  const size_t step = 2 * (size_t)seq_part_floats(D, NT);
  const int n = last - g + 2;
  auto part = [&](int i) { return i == 0 ? first : rest + (i - 1) * step; };
  // row r by lanes: the largest maximum, then every part's exp2(maximum - largest) / sum
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r = warp; r < rows; r += kSeqWarps) {
    float M = -INFINITY;
    for (int i = lane; i < n; i += 32) M = fmaxf(M, __ldcg(part(i) + RT * D + r * 2));
#pragma unroll
    for (int d = 16; d > 0; d /= 2) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    for (int i = lane; i < n; i += 32) {
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(part(i) + RT * D + r * 2));
      const float f = exp2_fast(ml.x - base);
      s_w[i * RT + r] = f;
      L += f * ml.y;
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) L += __shfl_xor_sync(0xffffffffu, L, d);
    for (int i = lane; i < n; i += 32) s_w[i * RT + r] *= 1.f / L;
  }
  __syncthreads();
  for (int e = blockIdx.y * kSeqThreads + threadIdx.x; e < rows * (D / 2); e += kSeqThreads * kJoinShares) {
    const int r = e / (D / 2), d = (e - r * (D / 2)) * 2;
    float x = 0.f, y = 0.f;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float2 o = __ldcg(reinterpret_cast<const float2*>(part(i) + r * D + d));
      const float f = s_w[i * RT + r];
      x += f * o.x;
      y += f * o.y;
    }
    const int pr = row0 + r, tok = pr / a.rep;
    if (d < a.hd)
      *reinterpret_cast<uint32_t*>(a.out + (long long)(s.start + tok) * a.sot +
                                   (long long)(kvh * a.rep + pr - tok * a.rep) * a.soh + d) =
          s.len - s.n + tok < 0 ? 0u : Type16<T>::pack(x, y);
  }
}

template <typename KernelT>
static int launch_attn_grid(KernelT kernel, const SeqAttnArgs& a, dim3 grid, size_t smem, int cluster,
                            cudaStream_t stream) {
  if (smem > 40 * 1024) {  // (the table is by kernel: instantiations of one signature share this function)
    static std::mutex mu;
    static std::vector<std::pair<int, const void*>> raised;
    int dev = 0;
    cudaGetDevice(&dev);
    const std::pair<int, const void*> key(dev, reinterpret_cast<const void*>(kernel));
    std::lock_guard<std::mutex> lock(mu);
    bool seen = false;
    for (auto& e : raised) seen |= (e == key);
    if (!seen) {
      const int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                                "attention: shared memory limit");
      if (rc != LI4_OK) return rc;
      raised.push_back(key);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kSeqThreads, 1, 1);
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
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, a), "attention: kernel launch");
}

// CTAs of a cluster per (request, KV head), 1: the shares of a line.  Where the pairs alone leave half of the CTAs that fit
// at once idle and no request can have more than 1024 keys per CTA, a cluster saves the second launch (a request of 576
// tokens: 4.9 us, 9.9 us by shares; 16 of them 6.9 and 13.8 us); with longer contexts equal shares are worth it (one request of 32000: 18.6 us by
// shares).
static int seq_cluster(const SeqAttnArgs& a) {
  int c = 1;
  while (c < 8 && 2LL * c * a.B * a.Hkv <= a.grid) c *= 2;
  return c > 1 && a.max_keys <= 1024LL * c ? c : 1;
}

template <typename T, int D, int NT, bool PAGED>
static int launch_seq(const SeqAttnArgs& a, cudaStream_t stream) {
  const int c = seq_cluster(a);
  if (c > 1)
    return launch_attn_grid(seq_attention_kernel<T, D, NT, PAGED, true>, a, dim3((unsigned)(a.B * a.Hkv * c)),
                            seq_smem_bytes(D), c, stream);
  int rc = launch_attn_grid(seq_attention_kernel<T, D, NT, PAGED, false>, a, dim3((unsigned)a.grid), seq_smem_bytes(D), 1,
                            stream);
  if (rc == LI4_OK)
    rc = launch_attn_grid(seq_attention_join_kernel<T, D, NT, PAGED>, a, dim3((unsigned)a.grid - 1, kJoinShares),
                          (size_t)a.grid * 8 * NT * sizeof(float), 1, stream);
  return rc;
}

template <typename T, bool PAGED>
static int launch_seq_d(const SeqAttnArgs& a, int nt, cudaStream_t stream) {
  if (a.hd <= 64)
    return nt == 1   ? launch_seq<T, 64, 1, PAGED>(a, stream)
           : nt == 2 ? launch_seq<T, 64, 2, PAGED>(a, stream)
                     : launch_seq<T, 64, 4, PAGED>(a, stream);
  return nt == 1   ? launch_seq<T, 128, 1, PAGED>(a, stream)
         : nt == 2 ? launch_seq<T, 128, 2, PAGED>(a, stream)
                   : launch_seq<T, 128, 4, PAGED>(a, stream);
}

static int seq_nt(int max_rows) { return max_rows <= 8 ? 1 : max_rows <= 16 ? 2 : 4; }
static int seq_grid(int sm) { return 2 * sm; }  // CTAs that fit at once

size_t seq_attention_part_bytes(int hd, int max_rows, int sm) {
  return (size_t)2 * seq_grid(sm) * seq_part_floats(hd <= 64 ? 64 : 128, seq_nt(max_rows)) * sizeof(float);
}

int launch_seq_attention(const SeqAttnArgs& args, bool paged, int dtype, int max_rows, cudaStream_t stream) {
  SeqAttnArgs a = args;
  a.grid = seq_grid(current_sm_count());
  const int nt = seq_nt(max_rows);
  if (dtype == LI4_F16)
    return paged ? launch_seq_d<__half, true>(a, nt, stream) : launch_seq_d<__half, false>(a, nt, stream);
  return paged ? launch_seq_d<__nv_bfloat16, true>(a, nt, stream) : launch_seq_d<__nv_bfloat16, false>(a, nt, stream);
}

// Rows (queries x heads of a KV head) up to which a sequence is streamed: where no sequence has more the streaming
// kernel runs alone, with tiles of 8, 16 or 32 rows; beside longer ones it takes those of one 8-row tile.  Beside a chunk
// of 512 tokens, 31 requests of 200-6000 tokens each, with the limit at 8 / 16 / 32 rows and tiles as high (us):
//   64 dims, 8 KV heads: 4 rows a request 63 / 64 / 71, 8 rows 64 / 65 / 72, 16 rows 96 / 67 / 77
//   128 dims, 8 KV heads: 4 rows 83 / 88 / 99, 8 rows 84 / 90 / 102, 16 rows 120 / 94 / 108
//   128 dims, 4 KV heads: 8 rows 68 / 71 / 78, 16 rows 94 / 77 / 82, 32 rows 94 / 95 / 93
//   128 dims, 1 KV head: 16 rows 50 / 47 / 59, 32 rows 50 / 50 / 61; 7 requests beside it: 16 rows 28 / 34 / 41
// So 8 is right for single tokens at groups of up to 8, and up to 1.4 times too slow for 16 rows of many requests.
constexpr int kFewRows = 32, kFewRowsBeside = 8;

constexpr int64_t kAttentionMost = 1 << 30;  // rows of a sequence, keys: what is claimed above it counts as it

static int check_attention(const li4_attention* p, bool paged, const char* what) {
  if (!p) return set_error(LI4_ERR_INVALID_ARG, "%s: null arguments", what);
  if (p->dtype != LI4_F16 && p->dtype != LI4_BF16)
    return set_error(LI4_ERR_UNSUPPORTED, "%s: dtype %d (LI4_F16 or LI4_BF16)", what, p->dtype);
  if (p->n_seqs < 0 || p->n_tokens < 0 || p->n_kv_heads < 1 || p->n_heads < p->n_kv_heads ||
      p->n_heads % p->n_kv_heads != 0 || p->max_queries < 0)
    return set_error(LI4_ERR_INVALID_ARG, "%s: n_seqs=%lld n_tokens=%lld n_heads=%lld n_kv_heads=%lld max_queries=%lld",
                     what, (long long)p->n_seqs, (long long)p->n_tokens, (long long)p->n_heads,
                     (long long)p->n_kv_heads, (long long)p->max_queries);
  if (p->head_dim < 8 || p->head_dim > 128 || p->head_dim % 8 != 0)
    return set_error(LI4_ERR_UNSUPPORTED, "%s: head_dim=%lld (a multiple of 8 up to 128)", what,
                     (long long)p->head_dim);
  if (p->n_heads / p->n_kv_heads > 128 || p->n_heads > 65535 || p->n_seqs > (1 << 24) ||
      p->n_tokens > (1LL << 30) / p->n_heads)
    return set_error(LI4_ERR_UNSUPPORTED, "%s: n_seqs=%lld n_tokens=%lld n_heads=%lld too large", what,
                     (long long)p->n_seqs, (long long)p->n_tokens, (long long)p->n_heads);
  if (!(p->scale == p->scale) || p->scale > 1e38f || p->scale < -1e38f)
    return set_error(LI4_ERR_INVALID_ARG, "%s: the scale is not finite", what);
  if (paged) {
    if (!is_pow2(p->page_size) || p->page_size < 8 || p->page_size > 1024)
      return set_error(LI4_ERR_UNSUPPORTED, "%s: page_size=%lld (a power of two from 8 to 1024)", what,
                       (long long)p->page_size);
    if (p->num_pages < 0 || p->num_pages > (1LL << 31) - 1 || p->table_width < 0 || p->table_stride < p->table_width ||
        p->table_width > kAttentionMost / p->page_size)
      return set_error(LI4_ERR_INVALID_ARG, "%s: num_pages=%lld table_width=%lld table_stride=%lld", what,
                       (long long)p->num_pages, (long long)p->table_width, (long long)p->table_stride);
  }
  if (p->n_seqs == 0 || p->n_tokens == 0) return LI4_OK;
  if (!p->q || !p->out || !p->cu_seqlens || ((!p->k || !p->v) && !(paged && p->num_pages == 0)) ||
      (paged && (!p->kv_lens || (!p->block_tables && p->table_width > 0))))
    return set_error(LI4_ERR_INVALID_ARG, "%s: null pointer", what);
  const int64_t st[] = {p->stride_qt, p->stride_qh, p->stride_ot, p->stride_oh, p->stride_kt, p->stride_kh,
                        p->stride_vt, p->stride_vh, paged ? p->stride_kp : 0, paged ? p->stride_vp : 0};
  bool aligned = aligned16(p->q) && aligned16(p->k) && aligned16(p->v) && aligned16(p->out);
  const int64_t rep = p->n_heads / p->n_kv_heads;
  const int64_t size[] = {p->n_tokens, p->n_heads, p->n_tokens, p->n_heads, paged ? p->page_size : p->n_tokens,
                          p->n_kv_heads, paged ? p->page_size : p->n_tokens, p->n_kv_heads, p->num_pages, p->num_pages};
  for (int i = 0; i < 10; ++i)  // (the stride of a dimension of one element is not used)
    aligned = aligned && st[i] % 8 == 0 && (st[i] > 0 || (st[i] == 0 && (size[i] <= 1 || (!paged && i >= 8))));
  if (!aligned || rep < 1)
    return set_error(LI4_ERR_ALIGNMENT, "%s: every row must start on a 16-byte boundary, at a positive stride", what);
  return LI4_OK;
}

static int attention_rows(const li4_attention* p) {
  const int64_t rep = p->n_heads / p->n_kv_heads;
  return (int)(p->max_queries > kAttentionMost / rep ? kAttentionMost : p->max_queries * rep);
}

// The most keys a sequence can have, as far as the host knows.
static int64_t attention_keys(const li4_attention* p) {
  if (!p->kv_lens) return p->max_queries < kAttentionMost ? p->max_queries : kAttentionMost;
  if (p->page_size < 1 || p->table_width < 1) return 0;
  return p->table_width > kAttentionMost / p->page_size ? kAttentionMost : p->table_width * p->page_size;
}

static int run_attention(const li4_attention* p, bool paged, void* workspace, size_t workspace_bytes, void* stream,
                         const char* what) {
  int rc = check_attention(p, paged, what);
  if (rc != LI4_OK) return rc;
  if (p->n_seqs == 0 || p->n_tokens == 0) {
    clear_error();
    return LI4_OK;
  }
  const size_t need = li4_attention_workspace_bytes(p);
  if (workspace_bytes < need || (need && !workspace) || !aligned16(workspace))
    return set_error(LI4_ERR_WORKSPACE, "%s: %zu bytes of 16-byte aligned workspace needed, %zu given", what, need,
                     workspace_bytes);
  SeqAttnArgs a = {};
  a.q = static_cast<const uint16_t*>(p->q);
  a.k = static_cast<const uint16_t*>(p->k);
  a.v = static_cast<const uint16_t*>(p->v);
  a.out = static_cast<uint16_t*>(p->out);
  a.sqt = p->stride_qt, a.sqh = p->stride_qh, a.sot = p->stride_ot, a.soh = p->stride_oh;
  a.skp = p->stride_kp, a.skt = p->stride_kt, a.skh = p->stride_kh;
  a.svp = p->stride_vp, a.svt = p->stride_vt, a.svh = p->stride_vh;
  a.cu = p->cu_seqlens;
  a.kv_lens = p->kv_lens;
  a.tables = p->block_tables;
  a.table_stride = p->table_stride;
  a.table_width = paged ? (int)p->table_width : 0;
  a.num_pages = paged ? (int)p->num_pages : 0;
  a.log_page = paged ? ilog2(p->page_size) : 0;
  a.B = (int)p->n_seqs;
  a.T = (int)p->n_tokens;
  a.Hkv = (int)p->n_kv_heads;
  a.rep = (int)(p->n_heads / p->n_kv_heads);
  a.hd = (int)p->head_dim;
  a.scale_log2 = p->scale * 1.44269504088896340736f;
  a.part = static_cast<float*>(workspace);
  a.max_keys = attention_keys(p);
  // Which kernel: the streaming one takes sequences of few rows, whose time is the reading of the keys, the
  // tensor-memory one (positive scales, some page) the rest.  The host knows the longest sequence as the caller
  // claims it; the device looks at each sequence's own rows, so a wrong claim only costs time.
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rows = attention_rows(p);
  const bool tiles = rows > kFewRows && a.scale_log2 > 0.f && !(paged && p->num_pages == 0);
  const bool both = tiles && paged && p->n_seqs > 1;
  rc = LI4_OK;
  if (!tiles || both) {
    a.small_rows = 0;
    a.big_rows = both ? kFewRowsBeside : 0x7fffffff;
    rc = launch_seq_attention(a, paged, p->dtype, both ? kFewRowsBeside : rows, st);
  }
  if (rc == LI4_OK && tiles) {
    a.small_rows = both ? kFewRowsBeside : 0;
    a.big_rows = 0x7fffffff;
    rc = launch_tile_attention(a, paged, p->dtype, st);
  }
  if (rc == LI4_OK) clear_error();
  return rc;
}

}  // namespace li4

extern "C" size_t li4_attention_workspace_bytes(const li4_attention* p) {
  using namespace li4;
  if (!p || p->n_seqs <= 0 || p->n_tokens <= 0 || p->n_kv_heads < 1 || p->max_queries < 0) return 0;
  const int64_t rep = p->n_heads / p->n_kv_heads;
  if (rep < 1 || rep > 128) return 0;
  const size_t seq = seq_attention_part_bytes((int)p->head_dim, attention_rows(p), current_sm_count());
  const size_t tile = attention_rows(p) > kFewRows ? tile_attention_part_bytes((int)p->head_dim, (int)rep, p->n_tokens,
                                                                               p->n_kv_heads, attention_keys(p),
                                                                               current_sm_count())
                                                   : 0;
  return seq > tile ? seq : tile;  // (the two kernels run one after the other)
}

extern "C" int li4_prompt_attention(const li4_attention* args, void* workspace, size_t workspace_bytes, void* stream) {
  return li4::run_attention(args, false, workspace, workspace_bytes, stream, "prompt_attention");
}

extern "C" int li4_paged_attention(const li4_attention* args, void* workspace, size_t workspace_bytes, void* stream) {
  return li4::run_attention(args, true, workspace, workspace_bytes, stream, "paged_attention");
}
