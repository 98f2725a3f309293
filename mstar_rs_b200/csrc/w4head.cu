// LM-head projection with 4-bit weights and group scales, on the 5th-generation
// tensor cores: the sampler's logits from a quarter of the bf16 head's bytes.
//
//   logits[b, v] = sum_G s[v, G] * sum_{k in G} hidden[b, k] * (q[v, k] - z[v, G])
//
// A code less its zero point is a whole number of at most four bits and a
// sign, exact in bf16; so is every product with a bf16 hidden value in the
// tensor core's fp32 accumulator.  The scale is applied to each group's sum,
// in fp32: rounding q * s to bf16 instead would cost 2^-9 of every weight.
//
// With few rows the weight stream bounds the product (V * d / 2 bytes), next
// to it turning the codes into bf16 (some 1.4 instructions per weight), so the
// kernel overlaps the two: one persistent CTA per SM takes an equal share of
// the (tile of 256 ids, 256 columns) units.
//   warps 0-7   expanders: a thread owns one vocabulary row: codes from shared
//               memory to bf16 pairs in registers to tensor memory (the A
//               operand; no second trip through shared memory);
//   warps 8-15  accumulators: a thread owns one vocabulary row and all of the
//               chunk's batch rows: group sums from tensor memory, times the
//               group's scale, into fp32 registers;
//   warp 16     weight producer: TMA boxes of 256 rows x 128 bytes;
//   warp 17     hidden producer: TMA boxes of 64 columns of the batch;
//   warps 18-19 MMA issuers, one per half of the tile (A from tensor memory, B
//               from shared memory).  With few batch rows an MMA is short and
//               what bounds the stream is the issuing warp's own chain of
//               waits and instructions, so the two halves have one each, the
//               warp stays converged (its operands are then uniform), and
//               with groups of 128 one barrier says that A is written and
//               the accumulator free, and one that both are done with.
// The accumulators hold up to 128 sums per thread, so the warpgroups' shares
// of the registers are set unequal (setmaxnreg).
//
// A word holds eight codes; taking codes i and i + 4 as a pair is one mask
// and one or per pair, so the pairs' order is [0 4 1 5 2 6 3 7] and a small
// kernel before puts the hidden columns into it.
//
// A tile that several CTAs share is summed by whichever of them comes last,
// in the order of the columns: nobody waits for anybody, and the sum does
// not depend on who was last.
//
// Every wait is bounded; one that runs out sets the error word, the roles
// stop issuing, drain what they issued, and the CTA exits.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"
#include "tcgen05.cuh"

namespace mstar {
namespace w4 {

constexpr int BM = 256;            // vocabulary ids per tile: two MMA tiles of 128
constexpr int KS = 256;            // columns per weight stage (128 bytes of codes: one swizzle row)
constexpr int KB = 128;            // columns per block: one A operand, one hidden stage
constexpr int W_BYTES = BM * KS / 2;
constexpr int ROWS_NT = 256;       // threads of each of the two row roles: one per row of the tile
constexpr int THREADS = 2 * ROWS_NT + 128;
// Registers per thread after the split of the 640 * 96 = 61440 that the block
// is launched with: 128 * (2 * expand + 2 * sum + issue) stays below it.
template <int N>
struct Regs {
  static constexpr int EXPAND = N > 64 ? 56 : 80, SUM = N > 64 ? 160 : 112, ISSUE = N > 64 ? 40 : 56;
  static_assert(128 * (2 * EXPAND + 2 * SUM + ISSUE) <= THREADS * 96, "registers of the launch");
};
constexpr int MAX_WS = 6, MAX_HS = 4;
constexpr int MAX_N = 128;         // batch rows per chunk
constexpr int MAX_B = 256;
constexpr int SMEM_BUDGET = 220 * 1024;
constexpr uint32_t ERR_TIMEOUT = 1u;
constexpr uint32_t A_COL = 0, D_COL = 256;  // tensor memory: [tile][buffer] of A, then the accumulators

struct Gemm {
  int B, V, d;
  int rows, nchunks, n;   // batch rows per chunk, chunks, MMA N (rows rounded up to 16)
  int nks, nblk, ntt;     // stages and blocks along d; tiles times chunks
  int wstages, hstages;
  int group, ngroups;
  const void *scales;
  int scale_dtype;
  const uint8_t *zeros;
  void *out;
  int64_t ld;
  int out_dtype;
  uint32_t *err;
  uint32_t *counters;     // [ntt] parts of a shared tile that have arrived
  float *parts;           // [grid][2][n][BM]
};

__device__ __forceinline__ uint32_t unit_start(const Gemm &g, int c) {
  return (uint32_t)((uint64_t)g.ntt * (uint64_t)g.nks * (uint64_t)c / gridDim.x);
}

// This CTA's share as segments: stages [k0, k1) of one tile.
struct Work {
  uint32_t u, u1;
  int tile, k0, k1;
  __device__ explicit Work(const Gemm &g) : u(unit_start(g, blockIdx.x)), u1(unit_start(g, blockIdx.x + 1)) {}
  __device__ bool next(const Gemm &g) {
    if (u >= u1) return false;
    tile = (int)(u / (uint32_t)g.nks);
    k0 = (int)(u % (uint32_t)g.nks);
    k1 = min(g.nks, k0 + (int)(u1 - u));
    u += (uint32_t)(k1 - k0);
    return true;
  }
  __device__ int b0() const { return 2 * k0; }
  __device__ int b1(const Gemm &g) const { return min(2 * k1, g.nblk); }
};

struct Sh {
  uint64_t wfull[MAX_WS], wempty[MAX_WS], hfull[MAX_HS], hempty[MAX_HS];
  // Per half of the tile.  Groups of 128 (one per block): ready[j] = A buffer
  // j written and the block's accumulator free, done[j] = its MMAs complete.
  // Smaller groups: ready[j] is A's alone and done[j] frees it, dfull and
  // dempty hand the accumulators over.
  uint64_t ready[2][2], done[2][2], dfull[2][2], dempty[2][2], mma_done[2];
  uint32_t tmem_base;
  int abort;
  int last;
};

__device__ __forceinline__ bool aborted(const Sh &sh) { return *reinterpret_cast<const volatile int *>(&sh.abort); }
__device__ __forceinline__ void raise(const Gemm &g, Sh &sh) {
  *reinterpret_cast<volatile int *>(&sh.abort) = 1;
  if (g.err) atomicOr(g.err, ERR_TIMEOUT);
}

// A place in a ring of `n` stages and the parity of its current use.
struct Ring {
  uint32_t i = 0, parity = 0;
  __device__ __forceinline__ void next(uint32_t n) {
    if (++i == n) i = 0, parity ^= 1u;
  }
};

// Warp-wide wait: one look, and the bounded wait behind it.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  if (__all_sync(~0u, ok)) return true;
  return __all_sync(~0u, mbar_wait(bar, parity));
}
__device__ __forceinline__ void warp_arrive(uint64_t *bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Barrier over the accumulator warps, and-reducing `v`.
__device__ __forceinline__ int sums_all(int v) {
  int r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.s32 p, %1, 0;\n bar.red.and.pred q, 1, 256, p;\n selp.s32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"(v)
      : "memory");
  return r;
}

// KN / 16 MMAs along the columns of one group: A advances by eight columns of
// tensor memory, B by 32 bytes of its rows, four steps to a box.  Issued by
// the lane with `lead` set; the warp is converged.
template <int KN>
__device__ __forceinline__ void mma_group(uint32_t lead, uint32_t d, uint32_t a, uint32_t desc_lo, uint32_t desc_hi,
                                          uint32_t box16, uint32_t idesc) {
#pragma unroll
  for (int k = 0; k < KN / 16; ++k)
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .b64 bd;\n setp.ne.b32 q, %0, 0;\n setp.ne.b32 p, %6, 0;\n"
        " mov.b64 bd, {%3, %4};\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], bd, %5, {%7, %7, %7, %7}, p;\n}\n" ::"r"(lead),
        "r"(d), "r"(a + 8u * k), "r"(desc_lo + (uint32_t)(k >> 2) * box16 + 2u * (k & 3)), "r"(desc_hi), "r"(idesc),
        "r"(k ? 1u : 0u), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t lead, uint64_t *bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %0, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n}\n" ::"r"(lead),
      "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r;
}

// 16 columns of this warp's 32 lanes, from registers.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Eight codes of a word as four bf16 pairs (i, i + 4), each code less the
// zero point: 0x4300 | q is 128 + q in bf16, and zz holds 128 + z twice.
__device__ __forceinline__ void expand(uint32_t w, __nv_bfloat162 zz, uint32_t *r) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
    const __nv_bfloat162 x = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&t), zz);
    r[i] = *reinterpret_cast<const uint32_t *>(&x);
  }
}

// The hidden rows with each eight columns in the order [0 4 1 5 2 6 3 7], and
// the arrival counters cleared.
__global__ void __launch_bounds__(256)
    w4_prepare_kernel(const __nv_bfloat16 *hidden, int64_t ld, int B, int d, int vec, uint4 *to, uint32_t *counters,
                      int ncounters) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int i = (int)(blockIdx.x * 256 + threadIdx.x);
  for (int j = i; j < ncounters; j += (int)gridDim.x * 256) counters[j] = 0u;
  const int per = d / 8;
  if (i >= B * per) return;
  const int b = i / per, k = (i - b * per) * 8;
  const __nv_bfloat16 *p = hidden + (int64_t)b * ld + k;
  uint16_t x[8];
  if (vec) {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    x[0] = (uint16_t)w.x, x[1] = (uint16_t)(w.x >> 16), x[2] = (uint16_t)w.y, x[3] = (uint16_t)(w.y >> 16);
    x[4] = (uint16_t)w.z, x[5] = (uint16_t)(w.z >> 16), x[6] = (uint16_t)w.w, x[7] = (uint16_t)(w.w >> 16);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = __bfloat16_as_ushort(p[j]);
  }
  to[i] = make_uint4(x[0] | (uint32_t)x[4] << 16, x[1] | (uint32_t)x[5] << 16, x[2] | (uint32_t)x[6] << 16,
                     x[3] | (uint32_t)x[7] << 16);
}

// Waits until each of the ring's last `n` uses (at most its stages) has landed.
__device__ void drain(const Gemm &g, Sh &sh, uint64_t *full, Ring r, uint32_t n, uint32_t stages) {
  for (uint32_t j = 0; j < n; ++j) {
    if (r.i == 0) r.i = stages, r.parity ^= 1u;
    --r.i;
    if (!mbar_wait(&full[r.i], r.parity)) raise(g, sh);
  }
}

__device__ void produce_weights(const Gemm &g, Sh &sh, uint8_t *sW, const CUtensorMap *map) {
  // one chunk: every weight is read once; several: their CTAs meet in L2
  const uint64_t pol = g.nchunks == 1 ? policy_evict_first() : policy_evict_last();
  const uint32_t stages = (uint32_t)g.wstages;
  Ring r;
  uint32_t used = 0;  // stages filled so far, up to the ring's length
  Work w(g);
  bool go = true;
  while (go && w.next(g)) {
    const int y = w.tile / g.nchunks * BM;
    for (int k = w.k0; k < w.k1; ++k) {
      if (aborted(sh) || (used == stages && !mbar_wait(&sh.wempty[r.i], r.parity ^ 1u))) {
        go = false;
        break;
      }
      mbar_expect_tx(&sh.wfull[r.i], (uint32_t)W_BYTES);
      tma_load_2d(sW + r.i * (uint32_t)W_BYTES, map, k * (KS / 2), y, &sh.wfull[r.i], pol);
      r.next(stages);
      used = min(used + 1, stages);
    }
  }
  if (!go) raise(g, sh);
  drain(g, sh, sh.wfull, r, used, stages);
}

__device__ void produce_hidden(const Gemm &g, Sh &sh, uint8_t *sH, const CUtensorMap *map) {
  const uint64_t pol = policy_evict_last();
  const uint32_t stages = (uint32_t)g.hstages, box = (uint32_t)g.n * 128u;
  Ring r;
  uint32_t used = 0;
  Work w(g);
  bool go = true;
  while (go && w.next(g)) {
    const int y = w.tile % g.nchunks * g.rows, b1 = w.b1(g);
    for (int b = w.b0(); b < b1; ++b) {
      if (aborted(sh) || (used == stages && !mbar_wait(&sh.hempty[r.i], r.parity ^ 1u))) {
        go = false;
        break;
      }
      mbar_expect_tx(&sh.hfull[r.i], 2u * box);
      uint8_t *to = sH + r.i * 2u * box;
      tma_load_2d(to, map, b * KB, y, &sh.hfull[r.i], pol);
      tma_load_2d(to + box, map, b * KB + 64, y, &sh.hfull[r.i], pol);
      r.next(stages);
      used = min(used + 1, stages);
    }
  }
  if (!go) raise(g, sh);
  drain(g, sh, sh.hfull, r, used, stages);
}

// Accumulators per half of the tile in tensor memory: one group's sums each.
template <int N>
__host__ __device__ constexpr int slots() {
  return N >= 128 ? 1 : 2;
}

template <int N, int GPB>
__device__ void issue(const Gemm &g, Sh &sh, uint8_t *sH, uint32_t tbase, uint32_t t) {
  constexpr int ND = slots<N>();
  const uint32_t lead = elect_one();
  const uint32_t idesc = idesc_bf16(128, g.n), box16 = (uint32_t)g.n * 8u;
  const uint64_t h0 = sw128_desc(smem_u32(sH));  // (stages and columns are added in its units of 16 bytes)
  const uint32_t hlo = (uint32_t)h0, hhi = (uint32_t)(h0 >> 32);
  const uint32_t hstages = (uint32_t)g.hstages, a0 = tbase + A_COL + t * 128u, d0 = tbase + D_COL + t * 128u;
  Ring h, a, dd;  // hidden stages, A buffers, accumulators
  bool first_lap = true, ok = true;
  Work w(g);
  while (ok && w.next(g)) {
    const int b1 = w.b1(g);
    for (int b = w.b0(); b < b1; ++b) {
      ok = warp_wait(&sh.hfull[h.i], h.parity) && warp_wait(&sh.ready[t][a.i], a.parity);
      if (!ok) break;
      const uint32_t lo = hlo + h.i * 2u * box16;
      if (GPB == 1) {
        tc_fence_after();
        mma_group<KB>(lead, d0 + (ND == 2 ? a.i : 0u) * (uint32_t)N, a0 + a.i * 64u, lo, hhi, box16, idesc);
      } else {
        const int groups = min(GPB, (g.d - b * KB) / (KB / GPB));
#pragma unroll
        for (int gi = 0; gi < GPB; ++gi) {
          if (gi >= groups) break;
          if (!first_lap && !(ok = warp_wait(&sh.dempty[t][dd.i], dd.parity ^ 1u))) break;
          tc_fence_after();
          constexpr int KN = KB / GPB;
          mma_group<KN>(lead, d0 + dd.i * (uint32_t)N, a0 + a.i * 64u + gi * (KN / 2),
                        lo + (uint32_t)(gi * KN / 64) * box16 + (uint32_t)(gi * KN % 64) / 8u, hhi, box16, idesc);
          commit(lead, &sh.dfull[t][dd.i]);
          dd.next(ND);
          if (dd.i == 0) first_lap = false;
        }
        if (!ok) break;
      }
      commit(lead, &sh.done[t][a.i]);
      commit(lead, &sh.hempty[h.i]);
      h.next(hstages);
      a.next(2);
    }
  }
  if (!ok) raise(g, sh);
  commit(lead, &sh.mma_done[t]);  // every MMA issued is complete before tensor memory is released
  if (!warp_wait(&sh.mma_done[t], 0)) raise(g, sh);
}

// Codes to bf16 in tensor memory, one vocabulary row per thread.
template <int GPB>
__device__ void expand_rows(const Gemm &g, Sh &sh, const uint8_t *sW, uint32_t tbase) {
  const int warp = (int)(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int t = warp >> 2, quad = warp & 3, row = t * 128 + quad * 32 + lane;
  const uint32_t at0 = tbase + ((uint32_t)(quad * 32) << 16) + A_COL + (uint32_t)t * 128u;
  const uint8_t *mine = sW + (size_t)row * (KS / 2);
  const uint32_t swz = (uint32_t)(row & 7);
  Ring st, a;
  bool first_lap = true;
  Work w(g);
  while (w.next(g)) {
    const int b0 = w.b0(), b1 = w.b1(g);
    const uint8_t *zp = nullptr;
    if (g.zeros) zp = g.zeros + (int64_t)min(w.tile / g.nchunks * BM + row, g.V - 1) * g.ngroups;
    uint32_t z[GPB], zn[GPB];
#pragma unroll
    for (int i = 0; i < GPB; ++i) z[i] = zn[i] = 8u;
    auto fetch = [&](int b) {  // (clamped: groups past the end are never used)
#pragma unroll
      for (int i = 0; i < GPB; ++i) zn[i] = __ldg(zp + min(b * GPB + i, g.ngroups - 1));
    };
    if (zp) fetch(b0);
    for (int b = b0; b < b1; ++b) {
      if (zp) {
#pragma unroll
        for (int i = 0; i < GPB; ++i) z[i] = zn[i] & 15u;
        fetch(b + 1);
      }
      if (!(b & 1) && !warp_wait(&sh.wfull[st.i], st.parity)) return raise(g, sh);
      uint4 c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)  // 32 columns: 16 bytes of codes
        c[i] = *reinterpret_cast<const uint4 *>(mine + st.i * (uint32_t)W_BYTES +
                                                (((uint32_t)((b & 1) * 4 + i) ^ swz) << 4));
      if (!first_lap && !warp_wait(&sh.done[t][a.i], a.parity ^ 1u)) return raise(g, sh);
      tc_fence_after();
      const uint32_t at = at0 + a.i * 64u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat16 zf = __ushort_as_bfloat16((unsigned short)(0x4300u | z[i * GPB / 4]));
        const __nv_bfloat162 zz = __halves2bfloat162(zf, zf);
        uint32_t r[16];
        expand(c[i].x, zz, r);
        expand(c[i].y, zz, r + 4);
        expand(c[i].z, zz, r + 8);
        expand(c[i].w, zz, r + 12);
        tmem_st16(at + (uint32_t)i * 16u, r);
      }
      if ((b & 1) || b + 1 == b1) {  // (the codes are in registers)
        warp_arrive(&sh.wempty[st.i]);
        st.next((uint32_t)g.wstages);
      }
      tmem_wait_st();
      tc_fence_before();
      warp_arrive(&sh.ready[t][a.i]);
      a.next(2);
      if (a.i == 0) first_lap = false;
    }
  }
}

template <int N>
__device__ __forceinline__ void put(const Gemm &g, int v, int chunk, const float (&acc)[N]) {
  if (v >= g.V) return;
  const uint64_t pol = policy_evict_last();
  const int b0 = chunk * g.rows, n = min(g.rows, g.B - b0);
  if (g.out_dtype == MSTAR_DTYPE_BF16) {
    __nv_bfloat16 *p = static_cast<__nv_bfloat16 *>(g.out) + (int64_t)b0 * g.ld + v;
#pragma unroll
    for (int c = 0; c < N; ++c, p += g.ld)
      if (c < n) st_last(p, __float2bfloat16_rn(acc[c]), pol);
  } else {
    float *p = static_cast<float *>(g.out) + (int64_t)b0 * g.ld + v;
#pragma unroll
    for (int c = 0; c < N; ++c, p += g.ld)
      if (c < n) st_last(p, acc[c], pol);
  }
}

// Group sums times scales, one vocabulary row per thread.
template <int N, int GPB>
__device__ void sum_rows(const Gemm &g, Sh &sh, uint32_t tbase) {
  const int warp = (int)(threadIdx.x >> 5) - 8, lane = threadIdx.x & 31;
  const int t = warp >> 2, quad = warp & 3, row = t * 128 + quad * 32 + lane;
  const uint32_t at0 = tbase + ((uint32_t)(quad * 32) << 16) + D_COL + (uint32_t)t * 128u;
  const bool f32 = g.scale_dtype == MSTAR_DTYPE_F32;
  constexpr int ND = slots<N>();
  Ring dd;  // groups of 128: the done barriers, otherwise the accumulators
  if (GPB == 1)
    for (int j = 0; j < ND; ++j) warp_arrive(&sh.ready[t][j]);  // the first blocks' accumulators are free
  Work w(g);
  while (w.next(g)) {
    const int v = w.tile / g.nchunks * BM + row, chunk = w.tile % g.nchunks;
    const int b0 = w.b0(), b1 = w.b1(g);
    const int64_t s0 = (int64_t)min(v, g.V - 1) * g.ngroups;
    float acc[N], s[GPB], sn[GPB];
#pragma unroll
    for (int c = 0; c < N; ++c) acc[c] = 0.f;
    auto fetch = [&](int b) {
#pragma unroll
      for (int i = 0; i < GPB; ++i) {
        const int64_t at = s0 + min(b * GPB + i, g.ngroups - 1);
        sn[i] = f32 ? __ldg(static_cast<const float *>(g.scales) + at)
                    : __bfloat162float(__ldg(static_cast<const __nv_bfloat16 *>(g.scales) + at));
      }
    };
    fetch(b0);
    bool ok = true;
    for (int b = b0; b < b1 && ok; ++b) {
#pragma unroll
      for (int i = 0; i < GPB; ++i) s[i] = sn[i];
      fetch(b + 1);
      const int groups = min(GPB, (g.d - b * KB) / (KB / GPB));
#pragma unroll
      for (int gi = 0; gi < GPB; ++gi) {
        if (gi >= groups) break;
        if (!warp_wait(GPB == 1 ? &sh.done[t][dd.i] : &sh.dfull[t][dd.i], dd.parity)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t at = at0 + (ND == 1 ? 0u : dd.i * (uint32_t)N);
#pragma unroll
        for (int c0 = 0; c0 < N; c0 += 16) {
          uint32_t r[16];
          tmem_ld16(at + (uint32_t)c0, r);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 16; ++c) acc[c0 + c] = fmaf(s[gi], __uint_as_float(r[c]), acc[c0 + c]);
        }
        tc_fence_before();
        // (with one accumulator it is the next block's, with two the next but one's)
        warp_arrive(GPB > 1 ? &sh.dempty[t][dd.i] : &sh.ready[t][ND == 1 ? dd.i ^ 1u : dd.i]);
        dd.next(GPB == 1 ? 2 : ND);
      }
    }
    if (!ok) raise(g, sh);
    if (!sums_all(ok)) return;
    if (w.k0 == 0 && w.k1 == g.nks) {
      put<N>(g, v, chunk, acc);
      continue;
    }
    // a shared tile: leave the part, and let the last to come add them all
    const int n = g.n;
    float *part = g.parts + ((size_t)blockIdx.x * 2 + (w.k0 == 0 ? 1 : 0)) * (size_t)n * BM + row;
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < n) __stcg(part + c * BM, acc[c]);
    __threadfence();
    sums_all(1);
    const uint32_t first = (uint32_t)w.tile * (uint32_t)g.nks, end = first + (uint32_t)g.nks;
    int c_lo = blockIdx.x, c_hi = blockIdx.x + 1;
    while (c_lo > 0 && unit_start(g, c_lo) > first) --c_lo;
    while (c_hi < (int)gridDim.x && unit_start(g, c_hi) < end) ++c_hi;
    if (threadIdx.x == ROWS_NT) sh.last = (int)atomicAdd(&g.counters[w.tile], 1u) == c_hi - c_lo - 1;
    sums_all(1);
    const bool last = *reinterpret_cast<volatile int *>(&sh.last) != 0;
    sums_all(1);  // everyone has read it
    if (!last) continue;
    __threadfence();
#pragma unroll
    for (int c = 0; c < N; ++c) acc[c] = 0.f;
    for (int q = c_lo; q < c_hi; ++q) {
      const float *p = g.parts + ((size_t)q * 2 + (unit_start(g, q) <= first ? 1 : 0)) * (size_t)n * BM + row;
#pragma unroll
      for (int c = 0; c < N; ++c)
        if (c < n) acc[c] += __ldcg(p + c * BM);
    }
    put<N>(g, v, chunk, acc);
  }
}

template <int N, int GPB>
__global__ void __launch_bounds__(THREADS, 1)
    w4_gemm_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap th, const Gemm g) {
  extern __shared__ __align__(1024) uint8_t w4_smem_raw[];
  __shared__ Sh sh;
  uint8_t *smem = w4_smem_raw + ((1024u - (smem_u32(w4_smem_raw) & 1023u)) & 1023u);
  uint8_t *sW = smem, *sH = smem + (size_t)g.wstages * W_BYTES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int s = 0; s < MAX_WS; ++s) {
      mbar_init(&sh.wfull[s], 1);
      mbar_init(&sh.wempty[s], ROWS_NT / 32);
    }
    for (int s = 0; s < MAX_HS; ++s) {
      mbar_init(&sh.hfull[s], 1);
      mbar_init(&sh.hempty[s], 2);
    }
    for (int t = 0; t < 2; ++t) {
      for (int j = 0; j < 2; ++j) {
        mbar_init(&sh.ready[t][j], GPB == 1 ? 2 * ROWS_NT / 64 : ROWS_NT / 64);
        mbar_init(&sh.done[t][j], 1);
      }
      for (int j = 0; j < 2; ++j) {
        mbar_init(&sh.dfull[t][j], 1);
        mbar_init(&sh.dempty[t][j], ROWS_NT / 64);
      }
      mbar_init(&sh.mma_done[t], 1);
    }
    sh.abort = 0;
    fence_barrier_init();
  }
  if (warp == 18) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem_base))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = sh.tmem_base;
  // the weights do not come from the kernel before; the hidden rows and the
  // counters do, and the output may still be read by what ran before that
  if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs<N>::EXPAND));
    expand_rows<GPB>(g, sh, sW, tbase);
  } else if (warp < 16) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Regs<N>::SUM));
    asm volatile("griddepcontrol.wait;" ::: "memory");
    sum_rows<N, GPB>(g, sh, tbase);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs<N>::ISSUE));
    if (warp == 16) {
      if (lane == 0) produce_weights(g, sh, sW, &tw);
    } else if (warp == 17) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      asm volatile("fence.proxy.async;" ::: "memory");
      if (lane == 0) produce_hidden(g, sh, sH, &th);
    } else {
      issue<N, GPB>(g, sh, sH, tbase, (uint32_t)warp - 18u);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 18) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tbase) : "memory");
  }
}

// ------------------------------------------------------------ host side

static Gemm plan(int B, int V, int d) {
  Gemm g{};
  g.B = B;
  g.V = V;
  g.d = d;
  g.nchunks = (B + MAX_N - 1) / MAX_N;
  g.rows = (B + g.nchunks - 1) / g.nchunks;
  g.n = (g.rows + 15) & ~15;
  g.nks = (d + KS - 1) / KS;
  g.nblk = (d + KB - 1) / KB;
  g.ntt = (V + BM - 1) / BM * g.nchunks;
  g.hstages = g.n <= 32 ? 4 : 3;
  g.wstages = std::min(MAX_WS, (SMEM_BUDGET - g.hstages * g.n * KB * 2) / W_BYTES);
  return g;
}

static int grid_of(const Gemm &g) { return (int)std::min<int64_t>(sm_count(), (int64_t)g.ntt * g.nks); }

// Workspace: arrival counters, the reordered hidden rows, the parts of shared
// tiles; each rounded to 256 bytes.
static int64_t up(int64_t b) { return (b + 255) / 256 * 256; }
static int64_t hidden_at(const Gemm &g) { return up((int64_t)g.ntt * 4); }
static int64_t parts_at(const Gemm &g) { return hidden_at(g) + up((int64_t)g.B * g.d * 2); }
static int64_t workspace_bytes(const Gemm &g) { return parts_at(g) + (int64_t)grid_of(g) * 2 * g.n * BM * 4; }

static int check_sizes(int B, int V, int d) {
  if (B < 1 || B > MAX_B) return fail(MSTAR_ERR_INVALID, "B must be in [1, 256]");
  if (V < 1 || V > (1 << 21)) return fail(MSTAR_ERR_INVALID, "V must be in [1, 2097152]");
  if (d < 32 || d % 32 || d > (1 << 18)) return fail(MSTAR_ERR_INVALID, "d must be a multiple of 32 in [32, 2^18]");
  return MSTAR_OK;
}

static int make_map(CUtensorMap *m, CUtensorMapDataType type, int size, const void *ptr, int64_t rows, int64_t cols,
                    int box_cols, int box_rows) {
  const EncodeTiled enc = tensor_map_encoder();
  if (!enc) return fail(MSTAR_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)cols * (cuuint64_t)size};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  const cuuint32_t es[2] = {1u, 1u};
  const CUresult r = enc(m, type, 2, const_cast<void *>(ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MSTAR_ERR_CUDA, "cuTensorMapEncodeTiled failed, code " + std::to_string((int)r));
  return MSTAR_OK;
}

template <int N, int GPB>
static int launch(const CUtensorMap &tw, const CUtensorMap &th, const Gemm &g, cudaStream_t st) {
  auto kern = w4_gemm_kernel<N, GPB>;
  const int smem = g.wstages * W_BYTES + g.hstages * g.n * KB * 2 + 1024;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return fail(MSTAR_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid_of(g), 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, tw, th, g);
  if (e != cudaSuccess) return fail(MSTAR_ERR_CUDA, std::string("launch: ") + cudaGetErrorString(e));
  return MSTAR_OK;
}

template <int N>
static int launch_n(const CUtensorMap &tw, const CUtensorMap &th, const Gemm &g, cudaStream_t st) {
  return g.group == 128 ? launch<N, 1>(tw, th, g, st)
         : g.group == 64 ? launch<N, 2>(tw, th, g, st)
                         : launch<N, 4>(tw, th, g, st);
}

static int logits(const void *hidden, int64_t ldh, int B, const mstar_w4_t *w, void *out, int dtype, int64_t ld,
                  void *ws, int64_t ws_bytes, uint32_t *err, cudaStream_t st) {
  int rc = check_w4(w);
  if (rc || (rc = check_sizes(B, w->V, w->d))) return rc;
  if (!hidden || !out || !ws) return fail(MSTAR_ERR_INVALID, "hidden, logits and workspace must not be NULL");
  if (reinterpret_cast<uintptr_t>(hidden) & 1u) return fail(MSTAR_ERR_INVALID, "hidden must be aligned to its type");
  if (ldh < w->d) return fail(MSTAR_ERR_INVALID, "ld_hidden must be >= d");
  if (dtype != MSTAR_DTYPE_F32 && dtype != MSTAR_DTYPE_BF16)
    return fail(MSTAR_ERR_INVALID, "dtype must be MSTAR_DTYPE_F32 or MSTAR_DTYPE_BF16");
  if (reinterpret_cast<uintptr_t>(out) & (dtype == MSTAR_DTYPE_F32 ? 3u : 1u))
    return fail(MSTAR_ERR_INVALID, "logits must be aligned to their type");
  if (ld < w->V) return fail(MSTAR_ERR_INVALID, "ld must be >= V");
  if (reinterpret_cast<uintptr_t>(ws) & 255u) return fail(MSTAR_ERR_INVALID, "workspace must be 256-byte aligned");
  Gemm g = plan(B, w->V, w->d);
  if (ws_bytes < workspace_bytes(g)) return fail(MSTAR_ERR_INVALID, "workspace too small");
  uint8_t *p = static_cast<uint8_t *>(ws);
  g.group = w->group;
  g.ngroups = w->d / w->group;
  g.scales = w->scales;
  g.scale_dtype = w->scale_dtype;
  g.zeros = static_cast<const uint8_t *>(w->zeros);
  g.out = out;
  g.ld = ld;
  g.out_dtype = dtype;
  g.err = err;
  g.counters = reinterpret_cast<uint32_t *>(p);
  g.parts = reinterpret_cast<float *>(p + parts_at(g));
  void *perm = p + hidden_at(g);
  CUtensorMap tw, th;
  if ((rc = make_map(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w->codes, w->V, w->d / 2, KS / 2, BM))) return rc;
  if ((rc = make_map(&th, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, perm, B, w->d, 64, g.n))) return rc;
  const int vec = (reinterpret_cast<uintptr_t>(hidden) % 16 == 0 && ldh % 8 == 0) ? 1 : 0;
  w4_prepare_kernel<<<(B * (w->d / 8) + 255) / 256, 256, 0, st>>>(static_cast<const __nv_bfloat16 *>(hidden), ldh, B,
                                                                w->d, vec, static_cast<uint4 *>(perm), g.counters,
                                                                g.ntt);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(MSTAR_ERR_CUDA, std::string("launch: ") + cudaGetErrorString(e));
  if (g.n <= 16) return launch_n<16>(tw, th, g, st);
  if (g.n <= 32) return launch_n<32>(tw, th, g, st);
  if (g.n <= 64) return launch_n<64>(tw, th, g, st);
  return launch_n<128>(tw, th, g, st);
}

}  // namespace w4

int check_w4(const mstar_w4_t *w) {
  if (!w) return fail(MSTAR_ERR_INVALID, "w is NULL");
  if (!w->codes || !w->scales) return fail(MSTAR_ERR_INVALID, "codes and scales must not be NULL");
  if (reinterpret_cast<uintptr_t>(w->codes) & 15u) return fail(MSTAR_ERR_INVALID, "codes must be 16-byte aligned");
  if (w->scale_dtype != MSTAR_DTYPE_F32 && w->scale_dtype != MSTAR_DTYPE_BF16)
    return fail(MSTAR_ERR_INVALID, "scale_dtype must be MSTAR_DTYPE_F32 or MSTAR_DTYPE_BF16");
  if (reinterpret_cast<uintptr_t>(w->scales) & (w->scale_dtype == MSTAR_DTYPE_F32 ? 3u : 1u))
    return fail(MSTAR_ERR_INVALID, "scales must be aligned to their type");
  if (w->group != 32 && w->group != 64 && w->group != 128)
    return fail(MSTAR_ERR_INVALID, "group must be 32, 64 or 128");
  if (w->V < 1 || w->d < w->group || w->d % w->group)
    return fail(MSTAR_ERR_INVALID, "V must be >= 1 and d a multiple of group");
  return MSTAR_OK;
}

}  // namespace mstar

using namespace mstar;

extern "C" {

int64_t mstar_lmhead_w4_workspace_bytes(int32_t B, int32_t V, int32_t d) {
  if (w4::check_sizes(B, V, d)) return -1;
  return w4::workspace_bytes(w4::plan(B, V, d));
}

int mstar_lmhead_logits_w4(const void *hidden, int64_t ld_hidden, int32_t B, const mstar_w4_t *w, void *logits,
                           int32_t dtype, int64_t ld, void *workspace, int64_t workspace_bytes, uint32_t *status,
                           void *stream) {
  return w4::logits(hidden, ld_hidden, B, w, logits, dtype, ld, workspace, workspace_bytes, status,
                    static_cast<cudaStream_t>(stream));
}

int mstar_sampler_lmhead_step_w4(const mstar_sampler_params_t *p, const void *hidden, int64_t ld_hidden,
                                 const mstar_w4_t *w, void *workspace, int64_t workspace_bytes, uint32_t *status,
                                 void *stream) {
  if (!p || !w) return fail(MSTAR_ERR_INVALID, "params and w must not be NULL");
  if (p->V != w->V) return fail(MSTAR_ERR_INVALID, "w must have the logits' V rows");
  // the step's own checks come first: nothing is launched when they fail
  int32_t cs = 0;
  int64_t smem = 0;
  int rc = mstar_sampler_plan(p, &cs, &smem);
  if (rc) return rc;
  rc = mstar_lmhead_logits_w4(hidden, ld_hidden, p->B, w, const_cast<void *>(p->logits), p->dtype, p->ld, workspace,
                              workspace_bytes, status, stream);
  return rc ? rc : mstar_sampler_step(p, stream);
}

}  // extern "C"
