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
//   warps 0-15  workers: a thread owns one vocabulary row and half of each
//               block of 128 columns: codes from shared memory to bf16 pairs
//               in registers to tensor memory (the A operand; no second trip
//               through shared memory), and for half of the batch the group
//               sums back from tensor memory into its fp32 accumulators;
//   warp 16     weight producer: TMA boxes of 256 rows x 128 bytes;
//   warp 17     hidden producer: TMA boxes of 64 columns of the batch;
//   warp 18     MMA issuer (A from tensor memory, B from shared memory).
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
constexpr int WORKERS = 512;
constexpr int THREADS = WORKERS + 96;
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
  uint64_t afull[2][2], aempty[2][2], dfull[2][4], dempty[2][4], mma_done;
  uint32_t tmem_base;
  int abort;
  int last;
};

__device__ __forceinline__ bool aborted(const Sh &sh) { return *reinterpret_cast<const volatile int *>(&sh.abort); }
__device__ __forceinline__ void raise(const Gemm &g, Sh &sh) {
  *reinterpret_cast<volatile int *>(&sh.abort) = 1;
  if (g.err) atomicOr(g.err, ERR_TIMEOUT);
}

// Barrier over the worker warps, and-reducing `v`.
__device__ __forceinline__ int workers_all(int v) {
  int r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.s32 p, %1, 0;\n bar.red.and.pred q, 1, 512, p;\n selp.s32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"(v)
      : "memory");
  return r;
}

__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
      : "memory");
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
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t *r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}

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

__device__ void produce_weights(const Gemm &g, Sh &sh, uint8_t *sW, const CUtensorMap *map) {
  const uint64_t pol = g.nchunks == 1 ? policy_evict_first() : policy_evict_last();
  uint32_t it = 0;
  Work w(g);
  bool go = true;
  while (go && w.next(g)) {
    for (int k = w.k0; k < w.k1 && go; ++k, ++it) {
      const uint32_t s = it % (uint32_t)g.wstages, use = it / (uint32_t)g.wstages;
      if (aborted(sh) || (use > 0 && !mbar_wait(&sh.wempty[s], (use - 1) & 1u))) {
        go = false;
        break;
      }
      mbar_expect_tx(&sh.wfull[s], (uint32_t)W_BYTES);
      tma_load_2d(sW + (size_t)s * W_BYTES, map, k * (KS / 2), w.tile / g.nchunks * BM, &sh.wfull[s], pol);
    }
  }
  if (!go) raise(g, sh);
  for (uint32_t j = it > (uint32_t)g.wstages ? it - (uint32_t)g.wstages : 0; j < it; ++j)  // every copy lands
    if (!mbar_wait(&sh.wfull[j % (uint32_t)g.wstages], (j / (uint32_t)g.wstages) & 1u)) raise(g, sh);
}

__device__ void produce_hidden(const Gemm &g, Sh &sh, uint8_t *sH, const CUtensorMap *map) {
  const uint64_t pol = policy_evict_last();
  const uint32_t box = (uint32_t)g.n * 128u;
  uint32_t it = 0;
  Work w(g);
  bool go = true;
  while (go && w.next(g)) {
    for (int b = w.b0(); b < w.b1(g) && go; ++b, ++it) {
      const uint32_t s = it % (uint32_t)g.hstages, use = it / (uint32_t)g.hstages;
      if (aborted(sh) || (use > 0 && !mbar_wait(&sh.hempty[s], (use - 1) & 1u))) {
        go = false;
        break;
      }
      mbar_expect_tx(&sh.hfull[s], 2u * box);
      for (int j = 0; j < 2; ++j)
        tma_load_2d(sH + (size_t)s * 2 * box + (size_t)j * box, map, b * KB + j * 64, w.tile % g.nchunks * g.rows,
                    &sh.hfull[s], pol);
    }
  }
  if (!go) raise(g, sh);
  for (uint32_t j = it > (uint32_t)g.hstages ? it - (uint32_t)g.hstages : 0; j < it; ++j)
    if (!mbar_wait(&sh.hfull[j % (uint32_t)g.hstages], (j / (uint32_t)g.hstages) & 1u)) raise(g, sh);
}

template <int NH, int GPB>
struct Ring {  // accumulators of one tile, one per group in flight
  static constexpr int N = 2 * NH;
  static constexpr int ND = N >= 128 ? 1 : N >= 64 ? 2 : 4;
};

template <int NH, int GPB>
__device__ void issue(const Gemm &g, Sh &sh, uint8_t *sH, uint32_t tbase) {
  constexpr int ND = Ring<NH, GPB>::ND;
  const uint32_t idesc = idesc_bf16(128, g.n), box = (uint32_t)g.n * 128u, h0 = smem_u32(sH);
  uint32_t ib = 0, ig = 0;
  Work w(g);
  bool go = true;
  while (go && w.next(g)) {
    for (int b = w.b0(); b < w.b1(g) && go; ++b, ++ib) {
      const uint32_t hs = ib % (uint32_t)g.hstages, buf = ib & 1u;
      const int groups = min(GPB, (g.d - b * KB) / (KB / GPB));
      if (aborted(sh) || !mbar_wait(&sh.hfull[hs], (ib / (uint32_t)g.hstages) & 1u)) {
        go = false;
        break;
      }
      for (uint32_t t = 0; t < 2 && go; ++t) {
        if (!mbar_wait(&sh.afull[t][buf], (ib >> 1) & 1u)) {
          go = false;
          break;
        }
        for (int gi = 0; gi < groups; ++gi) {
          const uint32_t q = ig + (uint32_t)gi, j = q % ND, use = q / ND;
          if (use > 0 && !mbar_wait(&sh.dempty[t][j], (use - 1) & 1u)) {
            go = false;
            break;
          }
          tc_fence_after();
          const uint32_t dcol = tbase + D_COL + t * 128u + j * (uint32_t)(2 * NH);
#pragma unroll
          for (int k = 0; k < KB / GPB / 16; ++k) {
            const uint32_t kk = (uint32_t)(gi * (KB / GPB / 16) + k);  // sixteen columns each
            mma_ts(dcol, tbase + A_COL + t * 128u + buf * 64u + kk * 8u,
                   sw128_desc(h0 + hs * 2u * box + (kk >> 2) * box + (kk & 3u) * 32u), idesc, k ? 1u : 0u);
          }
          mma_commit(&sh.dfull[t][j]);
        }
        mma_commit(&sh.aempty[t][buf]);
      }
      ig += (uint32_t)groups;
      mma_commit(&sh.hempty[hs]);
    }
  }
  if (!go) raise(g, sh);
  mma_commit(&sh.mma_done);  // every MMA issued is complete before tensor memory is released
  if (!mbar_wait(&sh.mma_done, 0)) raise(g, sh);
}

template <int NH, int GPB>
struct Worker {
  static constexpr int ND = Ring<NH, GPB>::ND;
  static constexpr int LC = NH >= 64 ? 16 : NH;  // columns per load: the accumulators leave no room for more
  const Gemm &g;
  Sh &sh;
  uint8_t *sW;
  uint32_t tbase;
  int lane, quad, t, h, row;
  bool ok = true;
  float acc[NH];
  uint32_t ib = 0, ig = 0, is = 0;  // blocks, groups and stages so far

  __device__ Worker(const Gemm &g_, Sh &sh_, uint8_t *sW_, uint32_t tb) : g(g_), sh(sh_), sW(sW_), tbase(tb) {
    const int warp = threadIdx.x >> 5;
    lane = threadIdx.x & 31;
    quad = warp & 3;  // tensor memory lanes 32 * quad .. + 31 belong to this warp
    t = (warp >> 2) & 1;
    h = warp >> 3;
    row = t * 128 + quad * 32 + lane;
  }
  __device__ __forceinline__ void wait(uint64_t *bar, uint32_t parity) {
    if (ok && !__all_sync(~0u, mbar_wait(bar, parity))) {
      ok = false;
      raise(g, sh);
    }
  }
  __device__ __forceinline__ void arrive(uint64_t *bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  }
  __device__ __forceinline__ float scale_at(int v, int G) const {
    if (v >= g.V || G >= g.ngroups) return 0.f;
    const int64_t at = (int64_t)v * g.ngroups + G;
    return g.scale_dtype == MSTAR_DTYPE_F32 ? __ldg(static_cast<const float *>(g.scales) + at)
                                            : __bfloat162float(static_cast<const __nv_bfloat16 *>(g.scales)[at]);
  }
  __device__ __forceinline__ uint32_t zero_at(int v, int G) const {
    if (!g.zeros || v >= g.V || G >= g.ngroups) return 8u;
    return __ldg(g.zeros + (int64_t)v * g.ngroups + G) & 15u;
  }
  // the group sums of one block into the accumulators
  __device__ __forceinline__ void drain(int b, const float (&s)[GPB]) {
    const int groups = min(GPB, (g.d - b * KB) / (KB / GPB));
#pragma unroll
    for (int gi = 0; gi < GPB; ++gi) {
      if (gi >= groups) break;
      const uint32_t j = ig % ND;
      wait(&sh.dfull[t][j], (ig / ND) & 1u);
      ++ig;
      if (!ok) return;
      tc_fence_after();
      const uint32_t at = tbase + ((uint32_t)(quad * 32) << 16) + D_COL + (uint32_t)t * 128u +
                          j * (uint32_t)(2 * NH) + (uint32_t)(h * NH);
#pragma unroll
      for (int c0 = 0; c0 < NH; c0 += LC) {
        uint32_t r[LC];
#pragma unroll
        for (int c = 0; c < LC; c += 8) tmem_ld8(at + (uint32_t)(c0 + c), r + c);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < LC; ++c) acc[c0 + c] = fmaf(s[gi], __uint_as_float(r[c]), acc[c0 + c]);
      }
      tc_fence_before();
      arrive(&sh.dempty[t][j]);
    }
  }
  __device__ __forceinline__ void put(int v, int chunk) {
    const uint64_t pol = policy_evict_last();
    if (v >= g.V) return;
#pragma unroll
    for (int c = 0; c < NH; ++c) {
      const int col = h * NH + c, b = chunk * g.rows + col;
      if (col < g.rows && b < g.B) {
        if (g.out_dtype == MSTAR_DTYPE_BF16)
          st_last(static_cast<__nv_bfloat16 *>(g.out) + (int64_t)b * g.ld + v, __float2bfloat16_rn(acc[c]), pol);
        else
          st_last(static_cast<float *>(g.out) + (int64_t)b * g.ld + v, acc[c], pol);
      }
    }
  }
  __device__ __forceinline__ bool segment(const Work &w) {
    const int v = w.tile / g.nchunks * BM + row, chunk = w.tile % g.nchunks;
    const int b0 = w.b0(), b1 = w.b1(g);
    float s[GPB], sn[GPB];
    uint32_t z[2], zn[2];  // this half's groups: one, or two of 32 columns
#pragma unroll
    for (int c = 0; c < NH; ++c) acc[c] = 0.f;
    auto fetch = [&](int b) {
#pragma unroll
      for (int gi = 0; gi < GPB; ++gi) sn[gi] = scale_at(v, b * GPB + gi);
      zn[0] = zero_at(v, b * GPB + h * GPB / 2);
      zn[1] = GPB == 4 ? zero_at(v, b * GPB + h * GPB / 2 + 1) : zn[0];
    };
    fetch(b0);
    for (int b = b0; b < b1; ++b, ++ib) {
      const uint32_t st = is % (uint32_t)g.wstages, buf = ib & 1u;
      float sp[GPB];  // the previous block's scales: its sums are drained after this block's codes are out
#pragma unroll
      for (int gi = 0; gi < GPB; ++gi) sp[gi] = s[gi], s[gi] = sn[gi];
      z[0] = zn[0], z[1] = zn[1];
      if (b + 1 < b1) fetch(b + 1);
      if (!(b & 1)) wait(&sh.wfull[st], (is / (uint32_t)g.wstages) & 1u);
      if (ib >= 2) wait(&sh.aempty[t][buf], ((ib >> 1) - 1) & 1u);
      if (ok) {
        tc_fence_after();
        const uint8_t *base = sW + (size_t)st * W_BYTES + (size_t)row * (KS / 2);
        const uint32_t at = tbase + ((uint32_t)(quad * 32) << 16) + A_COL + (uint32_t)t * 128u + buf * 64u +
                            (uint32_t)h * 32u;
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // 32 columns: 16 bytes of codes
          const uint32_t piece = (uint32_t)((b & 1) * 4 + h * 2 + i) ^ (uint32_t)(row & 7);
          const uint4 c = *reinterpret_cast<const uint4 *>(base + piece * 16u);
          const __nv_bfloat16 zf = __ushort_as_bfloat16((unsigned short)(0x4300u | z[i]));
          const __nv_bfloat162 zz = __halves2bfloat162(zf, zf);
          uint32_t r[16];
          expand(c.x, zz, r);
          expand(c.y, zz, r + 4);
          expand(c.z, zz, r + 8);
          expand(c.w, zz, r + 12);
          tmem_st16(at + (uint32_t)i * 16u, r);
        }
        tmem_wait_st();
        tc_fence_before();
        arrive(&sh.afull[t][buf]);
        if ((b & 1) || b + 1 == b1) arrive(&sh.wempty[st]);
      }
      if ((b & 1) || b + 1 == b1) ++is;
      if (b > b0) drain(b - 1, sp);
    }
    drain(b1 - 1, s);
    if (!workers_all(ok)) return false;
    if (w.k0 == 0 && w.k1 == g.nks) {
      put(v, chunk);
      return true;
    }
    // a shared tile: leave the part, and let the last to come add them all
    const int n = g.n;
    float *mine = g.parts + ((size_t)blockIdx.x * 2 + (w.k0 == 0 ? 1 : 0)) * (size_t)n * BM;
#pragma unroll
    for (int c = 0; c < NH; ++c)
      if (h * NH + c < n) __stcg(mine + (size_t)(h * NH + c) * BM + row, acc[c]);
    __threadfence();
    workers_all(1);
    const uint32_t first = (uint32_t)w.tile * (uint32_t)g.nks, end = first + (uint32_t)g.nks;
    int c_lo = blockIdx.x, c_hi = blockIdx.x + 1;
    while (c_lo > 0 && unit_start(g, c_lo) > first) --c_lo;
    while (c_hi < (int)gridDim.x && unit_start(g, c_hi) < end) ++c_hi;
    if (threadIdx.x == 0) sh.last = (int)atomicAdd(&g.counters[w.tile], 1u) == c_hi - c_lo - 1;
    workers_all(1);
    const bool last = *reinterpret_cast<volatile int *>(&sh.last) != 0;
    workers_all(1);  // everyone has read it
    if (!last) return true;
    __threadfence();
#pragma unroll
    for (int c = 0; c < NH; ++c) acc[c] = 0.f;
    for (int q = c_lo; q < c_hi; ++q) {
      const float *p = g.parts + ((size_t)q * 2 + (unit_start(g, q) <= first ? 1 : 0)) * (size_t)n * BM + row;
#pragma unroll
      for (int c = 0; c < NH; ++c)
        if (h * NH + c < n) acc[c] += __ldcg(p + (size_t)(h * NH + c) * BM);
    }
    put(v, chunk);
    return true;
  }
};

template <int NH, int GPB>
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
      mbar_init(&sh.wempty[s], WORKERS / 32);
    }
    for (int s = 0; s < MAX_HS; ++s) {
      mbar_init(&sh.hfull[s], 1);
      mbar_init(&sh.hempty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      for (int j = 0; j < 2; ++j) {
        mbar_init(&sh.afull[t][j], WORKERS / 64);
        mbar_init(&sh.aempty[t][j], 1);
      }
      for (int j = 0; j < 4; ++j) {
        mbar_init(&sh.dfull[t][j], 1);
        mbar_init(&sh.dempty[t][j], WORKERS / 64);
      }
    }
    mbar_init(&sh.mma_done, 1);
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
  if (warp != 16) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 16) {
    if (lane == 0) produce_weights(g, sh, sW, &tw);
  } else if (warp == 17) {
    asm volatile("fence.proxy.async;" ::: "memory");
    if (lane == 0) produce_hidden(g, sh, sH, &th);
  } else if (warp == 18) {
    if (lane == 0) issue<NH, GPB>(g, sh, sH, tbase);
  } else {
    Worker<NH, GPB> me(g, sh, sW, tbase);
    Work w(g);
    while (w.next(g))
      if (!me.segment(w)) break;
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

template <int NH, int GPB>
static int launch(const CUtensorMap &tw, const CUtensorMap &th, const Gemm &g, cudaStream_t st) {
  auto kern = w4_gemm_kernel<NH, GPB>;
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

template <int NH>
static int launch_n(const CUtensorMap &tw, const CUtensorMap &th, const Gemm &g, cudaStream_t st) {
  return g.group == 128 ? launch<NH, 1>(tw, th, g, st)
         : g.group == 64 ? launch<NH, 2>(tw, th, g, st)
                         : launch<NH, 4>(tw, th, g, st);
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
  if (g.n <= 16) return launch_n<8>(tw, th, g, st);
  if (g.n <= 32) return launch_n<16>(tw, th, g, st);
  if (g.n <= 64) return launch_n<32>(tw, th, g, st);
  return launch_n<64>(tw, th, g, st);
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
