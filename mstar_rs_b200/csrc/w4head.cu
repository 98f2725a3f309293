// LM-head projection with 4-bit weights and group scales, on the 5th-generation
// tensor cores: the sampler's logits from a quarter of the bf16 head's bytes.
//
//   logits[b, v] = sum_G s[v, G] * sum_{k in G} hidden[b, k] * (q[v, k] - z[v, G])
//
// A code less its zero point is a whole number of at most four bits and a
// sign, exact in fp16; so is every product with a hidden value in the tensor
// core's fp32 accumulator.  The scale is applied to each group's sum, in fp32:
// rounding q * s to 16 bits instead would cost 2^-9 or 2^-12 of every weight.
// The operands are fp16 and not bf16 because its ten bits take a code at two
// places of a word (below), which spares two of seven integer instructions;
// so each hidden row is first scaled by a power of two that brings its largest
// value into [2^15, 2^16).  A bf16 value keeps all its bits down to 2^-32 of the
// row's largest; below that it is off by at most half of fp16's smallest step,
// 2^-25, which is 2^-40 of the largest.
//
// With few rows the weight stream bounds the product (V * d / 2 bytes), next
// to it turning the codes into fp16 (nine instructions for eight weights) and
// storing them to tensor memory, so the kernel overlaps the three: one
// persistent CTA per SM takes an equal share of the (tile of 256 ids, 256
// columns) units.
//   expanders    a thread owns a vocabulary row: codes from shared memory to
//                fp16 pairs in registers to tensor memory (the A operand; no
//                second trip through shared memory);
//   accumulators a thread owns a vocabulary row and the chunk's batch rows:
//                group sums from tensor memory, times the group's scale, into
//                fp32 registers;
//   producers    a warp for the weights (TMA boxes of 256 rows x 128 bytes)
//                and one for the hidden rows (boxes of 64 columns);
//   MMA issuers  converged warps (their operands are then uniform);
//   counter      a warp that counts the parts of tiles shared between CTAs.
// What bounds such a pipeline are its hand-overs: a wait, a few dependent
// instructions and an arrival cost each role some hundred cycles, next to the
// 735 in which memory delivers a block of 256 x 128 codes.  So the two blocks
// of a stage have an A buffer, accumulators, expander warps and issuers of
// their own (up to 32 batch rows), each of which has twice the time.  Above 64
// rows, where each half of the tile has one accumulator, groups of 128 take one
// barrier for A written and the accumulator free and one for both done with.
//
// A word holds eight codes; codes i and i + 4 are a pair: one instruction masks
// them and sets fp16's exponent (0x6400 | q is 1024 + q; at bits 4-7 it is
// 1024 + 16 q), one subtracts.  The pairs' order is [0 4 1 5 2 6 3 7] and the
// kernel before puts the hidden columns into it.  (Codes beside fp16's exponent of
// 1024 are a known way from 4 bits to fp16: Kim et al., "Who Says Elephants Can't
// Run: Bringing Large Scale MoE Models into Cloud Scale Production", 2022.)
//
// A tile that several CTAs share is summed by the one whose part comes last, in
// the order of the columns: no CTA waits for another, and the sum does not
// depend on which it is.  A CTA takes its shared tiles first and adds at its
// end, so that neither the count nor the parts are waited for (counting and
// adding at once held the accumulators up by 8 of 51 us; B=1, V=151936,
// d=2048).
//
// Every wait is bounded; one that runs out sets the error word, the roles
// stop issuing, drain what they issued, and the CTA exits.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"
#include "ring.cuh"
#include "tcgen05.cuh"

namespace mstar {
namespace w4 {

constexpr int BM = 256;            // vocabulary ids per tile: two MMA tiles of 128
constexpr int KS = 256;            // columns per weight stage (128 bytes of codes: one swizzle row)
constexpr int KB = 128;            // columns per block: one A operand, one hidden stage
constexpr int W_BYTES = BM * KS / 2;
// Roles by the accumulator's width N.  LANES: whether the two blocks of a
// stage have expanders and issuers of their own.  The registers per thread
// that each role keeps of those that the block is launched with are set by
// setmaxnreg.
template <int N>
struct Roles {
  static constexpr int LANES = N > 32 ? 1 : 2;
  static constexpr int EXPAND = 8 * LANES;                       // expander warps: 32 rows of the tile each
  // Accumulator warps: 32 rows of the tile each, and with 64 columns half of
  // them: the accumulator is then free for the next MMAs sooner.
  static constexpr int HALVES = N == 64 ? 2 : 1;
  static constexpr int SUM = 8 * HALVES;
  static constexpr int ISSUE = 2 * LANES;                        // a warp per half of the tile
  // Producers and issuers in whole warpgroups; a warp to spare counts the parts
  // of shared tiles, otherwise the hidden rows' producer does when it is done.
  static constexpr int REST = (2 + ISSUE + 3) / 4 * 4;
  static constexpr int COUNTER = REST > 2 + ISSUE ? 2 + ISSUE : 1;
  static constexpr int THREADS = 32 * (EXPAND + SUM + REST);
  static constexpr int LAUNCH = 65536 / THREADS / 8 * 8;
  // What they hold fits but for four of the twelve variants: at 128 columns expanders
  // (56) and accumulators (160: 128 sums, 16 values read) spill 216, 152 and 32 bytes
  // with groups of 32, 64 and 128, at 64 columns with groups of 32 both spill 60.
  static constexpr int REGS_EXPAND = N > 64 ? 56 : 64;
  static constexpr int REGS_SUM = N > 64 ? 160 : 80;
  static constexpr int REGS_REST = 48;
  static_assert(32 * (EXPAND * REGS_EXPAND + SUM * REGS_SUM + REST * REGS_REST) <= THREADS * LAUNCH,
                "registers of the launch");
  // Tensor memory: A buffers [2 blocks][2 tiles][64 columns], then the
  // accumulators [slot][2 tiles][N].  A block's groups take its lane's slots in
  // turn; with one lane the blocks share the slots.
  static constexpr int D_COL = 256;
  static constexpr int SLOTS = N > 64 ? 1 : N > 32 ? 2 : 4;
  static constexpr int RING = SLOTS / LANES;  // slots per lane
  // One barrier for A written and the accumulator free, one for both done: where
  // a block has one group and the one accumulator (128 columns alone).
  template <int GPB>
  static __host__ __device__ constexpr bool merged() {
    return GPB == 1 && RING == 1;
  }
  static_assert(LANES == 1 || RING > 1, "merged barriers are written for one lane");
};
constexpr int MAX_WS = 6, MAX_HS = 8;
constexpr int MAX_N = 128;         // batch rows per chunk
constexpr int MAX_B = 256;
constexpr int SMEM_BUDGET = 220 * 1024;
constexpr uint32_t ERR_TIMEOUT = 1u;

struct Gemm {
  int B, V, d;
  int rows, nchunks, n;   // batch rows per chunk, chunks, MMA N (rows rounded up to 16)
  int nks, nblk, ntt;     // stages and blocks along d; tiles times chunks
  int wstages, hstages;
  uint32_t share, longer; // units per CTA, and how many CTAs take one more
  int group, ngroups;
  const void *scales;
  int scale_dtype;
  const uint8_t *zeros;
  int wide_scales, wide_zeros;  // whether their rows allow wide loads
  void *out;
  int64_t ld;
  int out_dtype;
  uint32_t *err;
  int withhold;           // testing: each CTA's last copy of hidden rows is never issued
  const float *row_scale; // [B] what the hidden rows were divided by
  uint32_t *counters;     // [ntt] parts of a shared tile that have arrived
  float *parts;           // [grid][2][n][BM]
};

// Shares are equal to within one unit: CTA c's begins at c * share + min(c, longer).
__device__ __forceinline__ uint32_t unit_start(const Gemm &g, int c) {
  return (uint32_t)c * g.share + min((uint32_t)c, g.longer);
}

// This CTA's share as segments, stages [k0, k1) of one tile: the tile it shares
// with the next CTA, the one it shares with the one before, then whole tiles.
struct Work {
  int tile, k0, k1;
  int t0, r0, t1, r1, at;
  __device__ explicit Work(const Gemm &g) : at(0) {
    const uint32_t u0 = unit_start(g, blockIdx.x), u1 = unit_start(g, blockIdx.x + 1);
    t0 = (int)(u0 / (uint32_t)g.nks), r0 = (int)(u0 % (uint32_t)g.nks);
    t1 = (int)(u1 / (uint32_t)g.nks), r1 = (int)(u1 % (uint32_t)g.nks);
  }
  __device__ bool next(const Gemm &g) {
    if (at == 0) {
      ++at;
      if (r1 > 0) {
        tile = t1, k0 = t0 == t1 ? r0 : 0, k1 = r1;
        return true;
      }
    }
    if (at == 1) {
      ++at;
      tile = t0 - 1;
      if (r0 > 0) {
        tile = t0, k0 = r0, k1 = g.nks;
        if (t0 < t1) return true;
      }
    }
    k0 = 0, k1 = g.nks;
    if (at == 2) ++at, tile = r0 > 0 ? t0 : t0 - 1;
    return ++tile < t1;
  }
  __device__ int b0() const { return 2 * k0; }
  __device__ int b1(const Gemm &g) const { return min(2 * k1, g.nblk); }
};

// The CTAs [c_lo, c_hi) whose shares meet `tile`.
__device__ __forceinline__ void sharers(const Gemm &g, int tile, int &c_lo, int &c_hi) {
  const uint32_t first = (uint32_t)tile * (uint32_t)g.nks, end = first + (uint32_t)g.nks;
  c_lo = blockIdx.x, c_hi = blockIdx.x + 1;
  while (c_lo > 0 && unit_start(g, c_lo) > first) --c_lo;
  while (c_hi < (int)gridDim.x && unit_start(g, c_hi) < end) ++c_hi;
}

struct Sh {
  uint64_t wfull[MAX_WS], wempty[MAX_WS], hfull[MAX_HS], hempty[MAX_HS];
  // By half of the tile t and block of the stage j: ready[t][j] = A written,
  // done[t][j] = its MMAs complete; dfull and dempty [t][slot] hand the
  // accumulators over.  Merged (128 columns, groups of 128): ready also says that
  // the accumulator is free, and done that its sums are there.
  uint64_t ready[2][2], done[2][2], dfull[2][4], dempty[2][4], mma_done[4];
  uint32_t tmem_base;
  int abort;
  int last[2];  // whether this CTA's part of the tile shared with the CTA before / after was the last
};

__device__ __forceinline__ bool aborted(const Sh &sh) { return *reinterpret_cast<const volatile int *>(&sh.abort); }
__device__ __forceinline__ void raise(const Gemm &g, Sh &sh) {
  *reinterpret_cast<volatile int *>(&sh.abort) = 1;
  if (g.err) atomicOr(g.err, ERR_TIMEOUT);
}

// The hot loops name barriers by their shared-memory address and keep what a
// hand-over costs to a few instructions: a pipeline of waits is bound by them.
//
// Waits for phase `parity`, at most LOOKS looks at the barrier, and sets `late` if
// they run out.  A look sleeps until the phase ends or some 1.5 us have passed
// (measured): 0.1 s in all, where a stage takes microseconds.  Looks are counted
// and not time, since a clock runs on while another process has the GPU.
constexpr uint32_t LOOKS = 1u << 16;
__device__ __forceinline__ void await(uint32_t bar, uint32_t parity, uint32_t &late) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .u32 n;\n mov.u32 n, %3;\n"
      "LOOK:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n @p bra SEEN;\n"
      " sub.u32 n, n, 1;\n setp.ne.u32 q, n, 0;\n @q bra LOOK;\n mov.u32 %0, 1;\nSEEN:\n}\n"
      : "+r"(late)
      : "r"(bar), "r"(parity), "n"(LOOKS)
      : "memory");
}
// One arrival of the whole warp.
__device__ __forceinline__ void arrive(uint32_t bar, bool lane0) {
  __syncwarp();
  if (lane0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Named barriers 1 and 2 tell the counting warp that a part of this CTA's two
// shared tiles is written (the accumulator warps arrive and go on); barrier 3
// tells them what it counted.
template <int N>
__device__ __forceinline__ void bar_arrive(int id) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(32 * Roles<N>::SUM + 32) : "memory");
}
template <int N>
__device__ __forceinline__ void bar_sync(int id) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(32 * Roles<N>::SUM + 32) : "memory");
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
__device__ __forceinline__ void commit(uint32_t lead, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %0, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n}\n" ::"r"(lead),
      "r"(bar)
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

// Eight codes of a word as four fp16 pairs (i, i + 4), each code less the
// zero point: nz holds -(1024 + z) twice, nz16 -(64 + z).
__device__ __forceinline__ uint32_t mask_or(uint32_t w, uint32_t mask) {
  uint32_t t;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(t) : "r"(w), "r"(mask), "r"(0x64006400u));
  return t;
}
__device__ __forceinline__ void expand(uint32_t w, uint32_t nz, uint32_t nz16, uint32_t *r) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const uint32_t x = w >> (4 * i);
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r[i]) : "r"(mask_or(x, 0x000F000Fu)), "r"(nz));
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r[i + 1]) : "r"(mask_or(x, 0x00F000F0u)), "r"(0x2C002C00u), "r"(nz16));
  }
}

// One CTA per batch row: the hidden row times a power of two, as fp16, each
// eight columns in the order [0 4 1 5 2 6 3 7]; the power's inverse; and the
// arrival counters cleared.
constexpr int PREP_NT = 256;
__global__ void __launch_bounds__(PREP_NT)
    w4_prepare_kernel(const __nv_bfloat16 *hidden, int64_t ld, int d, int vec, uint4 *to, float *row_scale,
                      uint32_t *counters, int ncounters) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ uint32_t warp_max[PREP_NT / 32];
  const int tid = threadIdx.x, per = d / 8;
  for (int j = (int)blockIdx.x * PREP_NT + tid; j < ncounters; j += (int)gridDim.x * PREP_NT) counters[j] = 0u;
  const __nv_bfloat16 *row = hidden + (int64_t)blockIdx.x * ld;
  auto load = [&](int i, uint16_t(&x)[8]) {
    const __nv_bfloat16 *p = row + i * 8;
    if (vec) {
      const uint4 w = *reinterpret_cast<const uint4 *>(p);
      x[0] = (uint16_t)w.x, x[1] = (uint16_t)(w.x >> 16), x[2] = (uint16_t)w.y, x[3] = (uint16_t)(w.y >> 16);
      x[4] = (uint16_t)w.z, x[5] = (uint16_t)(w.z >> 16), x[6] = (uint16_t)w.w, x[7] = (uint16_t)(w.w >> 16);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __bfloat16_as_ushort(p[j]);
    }
  };
  uint16_t first[8];  // (most rows are one round of the block: they are read once)
  uint32_t top = 0;
  for (int i = tid; i < per; i += PREP_NT) {
    uint16_t x[8];
    load(i, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (i == tid) first[j] = x[j];
      const uint32_t mag = x[j] & 0x7FFFu;
      if (mag < 0x7F80u) top = max(top, mag);  // the largest finite magnitude
    }
  }
  top = __reduce_max_sync(~0u, top);
  if ((tid & 31) == 0) warp_max[tid >> 5] = top;
  __syncthreads();
  top = 0;
  for (int w = 0; w < PREP_NT / 32; ++w) top = max(top, warp_max[w]);
  int e = 0;
  if (top) {
    int x;
    frexpf(__uint_as_float(top << 16), &x);  // the largest is in [2^(x-1), 2^x)
    e = 16 - x;  // at most (2 - 2^-7) 2^15 = 65280, below fp16's largest; 2^-e >= 2^-148 is a float
  }
  if (tid == 0) row_scale[blockIdx.x] = ldexpf(1.f, -e);
  for (int i = tid; i < per; i += PREP_NT) {
    uint16_t x[8];
    if (i == tid) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = first[j];
    } else {
      load(i, x);
    }
    uint32_t y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      y[j] = __half_as_ushort(__float2half_rn(ldexpf(__uint_as_float((uint32_t)x[j] << 16), e)));
    to[(int64_t)blockIdx.x * per + i] =
        make_uint4(y[0] | y[4] << 16, y[1] | y[5] << 16, y[2] | y[6] << 16, y[3] | y[7] << 16);
  }
}

// Waits until each of a ring's last `n` uses (at most its `stages`, which are
// `step` apart) has landed.
__device__ void drain(const Gemm &g, Sh &sh, uint32_t full, Ring r, uint32_t n, uint32_t stages, uint32_t step = 1) {
  uint32_t late = 0;
  for (uint32_t j = 0; j < n; ++j) {
    if (r.i == 0) r.i = stages, r.parity ^= 1u;
    --r.i;
    await(full + 8u * r.i * step, r.parity, late);
  }
  if (late) raise(g, sh);
}

__device__ void produce_weights(const Gemm &g, Sh &sh, uint8_t *sW, const CUtensorMap *map) {
  // one chunk: every weight is read once; several: their CTAs meet in L2
  const uint64_t pol = g.nchunks == 1 ? policy_evict_first() : policy_evict_last();
  const uint32_t stages = (uint32_t)g.wstages, wempty = smem_u32(sh.wempty);
  Ring r;
  uint32_t used = 0;  // stages filled so far, up to the ring's length
  uint32_t late = 0;
  Work w(g);
  bool go = true;
  while (go && w.next(g)) {
    const int y = w.tile / g.nchunks * BM;
    for (int k = w.k0; k < w.k1; ++k) {
      const bool stop = aborted(sh);
      if (used == stages) await(wempty + 8u * r.i, r.parity ^ 1u, late);
      if (late || stop) {
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
  drain(g, sh, smem_u32(sh.wfull), r, used, stages);
}

template <int N>
__device__ void produce_hidden(const Gemm &g, Sh &sh, uint8_t *sH, const CUtensorMap *map) {
  constexpr int LANES = Roles<N>::LANES;
  const uint64_t pol = policy_evict_last();
  const uint32_t stages = (uint32_t)g.hstages, per = stages / LANES, box = (uint32_t)g.n * 128u;
  LaneRings<LANES> r;
  uint32_t used[LANES] = {}, late = 0;
  const uint32_t hempty = smem_u32(sh.hempty);
  Work w(g);
  bool go = true;
  while (go && w.next(g)) {
    const int y = w.tile % g.nchunks * g.rows;
    int b1 = w.b1(g);
    if (g.withhold) {
      Work rest = w;
      b1 -= !rest.next(g);
    }
    for (int b = w.b0(); b < b1; ++b) {
      const bool second = LANES == 2 && (b & 1);  // (selects: an index would put the rings into local memory)
      const uint32_t at = second ? r.stage(LANES - 1) : r.stage(0), u = second ? used[LANES - 1] : used[0];
      const uint32_t parity = second ? r.parity(LANES - 1) : r.parity(0);
      const bool stop = aborted(sh);
      if (u == per) await(hempty + 8u * at, parity ^ 1u, late);
      if (late || stop) {
        go = false;
        break;
      }
      mbar_expect_tx(&sh.hfull[at], 2u * box);
      uint8_t *to = sH + at * 2u * box;
      tma_load_2d(to, map, b * KB, y, &sh.hfull[at], pol);
      tma_load_2d(to + box, map, b * KB + 64, y, &sh.hfull[at], pol);
      if (second) {
        r.next(LANES - 1, stages);
        used[LANES - 1] = min(u + 1, per);
      } else {
        r.next(0, stages);
        used[0] = min(u + 1, per);
      }
    }
  }
  if (!go) raise(g, sh);
#pragma unroll
  for (int lane = 0; lane < LANES; ++lane)
    drain(g, sh, smem_u32(sh.hfull + lane), r.ring[lane], used[lane], per, (uint32_t)LANES);
}

// MMAs of half t of the tile, of the blocks of `lane` (with one lane: of all).
template <int N, int GPB>
__device__ void issue(const Gemm &g, Sh &sh, uint8_t *sH, uint32_t tbase, int who) {
  using R = Roles<N>;
  constexpr int RING = R::RING;
  constexpr bool MERGED = R::template merged<GPB>();
  const int t = who & 1, lane = who >> 1;
  const uint32_t lead = elect_one();
  const uint32_t idesc = idesc_f16(128, g.n), box16 = (uint32_t)g.n * 8u;
  const uint64_t h0 = sw128_desc(smem_u32(sH));  // (stages and columns are added in its units of 16 bytes)
  const uint32_t hlo = (uint32_t)h0, hhi = (uint32_t)(h0 >> 32), hstages = (uint32_t)g.hstages;
  const uint32_t a0 = tbase + (uint32_t)t * 64u, d0 = tbase + R::D_COL + (uint32_t)(t * N);
  const uint32_t hfull = smem_u32(sh.hfull), hempty = smem_u32(sh.hempty);
  const uint32_t ready = smem_u32(sh.ready[t]), done = smem_u32(sh.done[t]);
  const uint32_t dfull = smem_u32(sh.dfull[t]), dempty = smem_u32(sh.dempty[t]);
  LaneRings<R::LANES> h;
  uint32_t rp = 0, dp = 0, fresh = 0xFu;  // parities of ready[t][j] and dempty[t][slot], a bit each; unused slots
  int slot = 0;                           // within the lane's ring
  uint32_t late = 0;
  Work w(g);
  while (!late && w.next(g)) {
    for (int k = w.k0; k < w.k1 && !late; ++k) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (j == 1 && 2 * k + 1 >= g.nblk) break;
        if (R::LANES == 2 && j != lane) continue;
        const int own = R::LANES == 2 ? j : 0;
        const uint32_t at = h.stage(own);
        await(hfull + 8u * at, h.parity(own), late);
        await(ready + 8u * j, (rp >> j) & 1u, late);
        rp ^= 1u << j;
        const uint32_t lo = hlo + at * 2u * box16, aj = a0 + (uint32_t)j * 128u;
        if (MERGED) {
          tc_fence_after();
          mma_group<KB>(lead, d0, aj, lo, hhi, box16, idesc);
        } else {
          const int groups = GPB == 1 ? 1 : min(GPB, (g.d - (2 * k + j) * KB) / (KB / GPB));
#pragma unroll
          for (int gi = 0; gi < GPB; ++gi) {
            if (gi >= groups) break;
            const uint32_t q = (R::LANES == 2 ? j * RING : 0) + slot;
            if (!((fresh >> q) & 1u)) await(dempty + 8u * q, ((dp >> q) & 1u) ^ 1u, late);
            fresh &= ~(1u << q);
            dp ^= 1u << q;
            tc_fence_after();
            constexpr int KN = KB / GPB;
            mma_group<KN>(lead, d0 + q * 2u * N, aj + gi * (KN / 2),
                          lo + (uint32_t)(gi * KN / 64) * box16 + (uint32_t)(gi * KN % 64) / 8u, hhi, box16, idesc);
            commit(lead, dfull + 8u * q);
            if (RING == 2) slot ^= 1;
          }
        }
        commit(lead, done + 8u * j);
        commit(lead, hempty + 8u * at);
        h.next(own, hstages);
      }
    }
  }
  if (late) raise(g, sh);
  late = 0;
  commit(lead, smem_u32(&sh.mma_done[who]));  // every MMA issued is complete before tensor memory is released
  await(smem_u32(&sh.mma_done[who]), 0, late);
  if (late) raise(g, sh);
}

// Codes to fp16 in tensor memory.
template <int N, int GPB>
__device__ void expand_rows(const Gemm &g, Sh &sh, const uint8_t *sW, uint32_t tbase) {
  using R = Roles<N>;
  const int warp = (int)(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const bool lane0 = lane == 0;
  const int t = (warp >> 2) & 1, quad = warp & 3, row = t * 128 + quad * 32 + lane, mine = warp >> 3;
  const uint32_t at0 = tbase + ((uint32_t)(quad * 32) << 16) + (uint32_t)t * 64u;
  const uint32_t stages = (uint32_t)g.wstages;
  const uint32_t wfull = smem_u32(sh.wfull), wempty = smem_u32(sh.wempty);
  const uint32_t ready = smem_u32(sh.ready[t]), done = smem_u32(sh.done[t]);
  // this row's 16-byte pieces of a stage lie swizzled: piece i of block j at (4 j + i) ^ (row & 7)
  uint32_t piece[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    piece[i] = smem_u32(sW) + (uint32_t)row * (KS / 2) + (((uint32_t)(4 * mine + i) ^ (uint32_t)(row & 7)) << 4);
  Ring st;
  uint32_t dp = 0, fresh = 3u;  // parities of done[t][j], a bit each; unused A buffers
  uint32_t nz[GPB], nz16[GPB], late = 0;
  // zero points: as the scales, eight bytes at a time with groups below 128 (151
  // against 144 us, 64 rows of groups of 32)
  constexpr bool WORDS = GPB > 1;
  constexpr int SPL = 4 / GPB;  // stages per load of zero points
  uint64_t zc = 0, zn = 0;      // a byte per group: from this stage on, and the next load's
#pragma unroll
  for (int i = 0; i < GPB; ++i) nz[i] = 0xE408E408u, nz16[i] = 0xD480D480u;  // zero point 8
  Work w(g);
  while (w.next(g)) {
    const uint8_t *zp = nullptr;
    if (g.zeros) zp = g.zeros + (int64_t)min(w.tile / g.nchunks * BM + row, g.V - 1) * g.ngroups;
    auto load = [&](int k) {  // of stages [k, k + SPL) (clamped: groups past the end are never used)
      uint64_t z = 0;
      if (g.wide_zeros) {
        const uint2 x = __ldg(reinterpret_cast<const uint2 *>(zp + min(k * 2 * GPB, g.ngroups - 8)));
        z = (uint64_t)x.y << 32 | x.x;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (R::LANES == 1 || ((i / GPB) & 1) == mine)
            z |= (uint64_t)__ldg(zp + min(k * 2 * GPB + i, g.ngroups - 1)) << (8 * i);
      }
      return z;
    };
    if (WORDS && zp) {
      const int k = w.k0 & ~(SPL - 1);
      zc = load(k), zn = load(k + SPL);
      zc >>= 16 * GPB * (w.k0 - k);
    }
    for (int k = w.k0; k < w.k1; ++k) {
      const bool two = 2 * k + 1 < g.nblk;  // (d's last stage may hold one block)
      const uint32_t stage = st.i * (uint32_t)W_BYTES;
      uint32_t z = 0;
      auto fetch = [&](int j) { z = __ldg(zp + min(2 * k + j, g.ngroups - 1)); };  // (with groups of 128)
      if (!WORDS && zp) fetch(R::LANES == 2 ? mine : 0);
      await(wfull + 8u * st.i, st.parity, late);
#pragma unroll
      for (int pass = 0; pass < 3 - R::LANES; ++pass) {
        const int j = R::LANES == 2 ? mine : pass;
        if (j == 1 && !two) {
          if (R::LANES == 2) arrive(wempty + 8u * st.i, lane0);
          break;
        }
        uint4 c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // 32 columns: 16 bytes of codes
          const uint32_t from = (R::LANES == 1 && j == 1 ? piece[i] ^ 64u : piece[i]) + stage;
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(c[i].x), "=r"(c[i].y), "=r"(c[i].z), "=r"(c[i].w)
                       : "r"(from));
        }
        if (zp) {
#pragma unroll
          for (int i = 0; i < GPB; ++i) {
            const uint32_t zz = ((WORDS ? (uint32_t)(zc >> (8 * (j * GPB + i))) : z) & 15u) * 0x10001u;
            nz[i] = 0xE400E400u | zz, nz16[i] = 0xD400D400u | zz << 4;
          }
        }
        if (!((fresh >> j) & 1u)) await(done + 8u * j, ((dp >> j) & 1u) ^ 1u, late);
        fresh &= ~(1u << j);
        dp ^= 1u << j;
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t r[16];
          expand(c[i].x, nz[i * GPB / 4], nz16[i * GPB / 4], r);
          expand(c[i].y, nz[i * GPB / 4], nz16[i * GPB / 4], r + 4);
          expand(c[i].z, nz[i * GPB / 4], nz16[i * GPB / 4], r + 8);
          expand(c[i].w, nz[i * GPB / 4], nz16[i * GPB / 4], r + 12);
          tmem_st16(at0 + (uint32_t)j * 128u + (uint32_t)i * 16u, r);
        }
        if (R::LANES == 2 || j == 1 || !two) arrive(wempty + 8u * st.i, lane0);  // (the codes are in registers)
        if (!WORDS && R::LANES == 1 && j == 0 && two && zp) fetch(1);
        tmem_wait_st();
        tc_fence_before();
        arrive(ready + 8u * j, lane0);
      }
      if (late) return raise(g, sh);
      st.next(stages);
      if (WORDS && zp) {
        if (SPL == 1 || ((k + 1) & (SPL - 1)) == 0)
          zc = zn, zn = load(k + 1 + SPL);
        else
          zc >>= (16 * GPB) & 63;
      }
    }
  }
}

// Sixteen of a row's sums to the logits, times what the hidden rows were divided by.
__device__ __forceinline__ void put16(const Gemm &g, int v, int chunk, int c0, const float *x) {
  if (v >= g.V) return;
  const uint64_t pol = policy_evict_last();
  const int b0 = chunk * g.rows + c0, n = min(g.rows - c0, g.B - b0);
  const float *rs = g.row_scale + b0;
  if (g.out_dtype == MSTAR_DTYPE_BF16) {
    __nv_bfloat16 *p = static_cast<__nv_bfloat16 *>(g.out) + (int64_t)b0 * g.ld + v;
#pragma unroll
    for (int c = 0; c < 16; ++c, p += g.ld)
      if (c < n) st_last(p, __float2bfloat16_rn(x[c] * rs[c]), pol);
  } else {
    float *p = static_cast<float *>(g.out) + (int64_t)b0 * g.ld + v;
#pragma unroll
    for (int c = 0; c < 16; ++c, p += g.ld)
      if (c < n) st_last(p, x[c] * rs[c], pol);
  }
}

// Two sums at a time: (a0, a1) += (x0, x1) * (s, s).
__device__ __forceinline__ void fma2(float &a0, float &a1, uint32_t x0, uint32_t x1, float s) {
  asm("{\n .reg .b64 a, x, s;\n mov.b64 a, {%0, %1};\n mov.b64 x, {%2, %3};\n mov.b64 s, {%4, %4};\n"
      " fma.rn.f32x2 a, x, s, a;\n mov.b64 {%0, %1}, a;\n}\n"
      : "+f"(a0), "+f"(a1)
      : "r"(x0), "r"(x1), "f"(s));
}

// Group sums times scales.
template <int N, int GPB, bool F32>
__device__ void sum_rows(const Gemm &g, Sh &sh, uint32_t tbase) {
  using R = Roles<N>;
  constexpr int RING = R::RING;
  constexpr bool MERGED = R::template merged<GPB>();
  constexpr int NC = N / R::HALVES;       // this warp's columns, from `from`
  // Columns loaded at a time.  With groups below 128, 32 of them would not fit the
  // registers beside the scales (32 rows, V=151936, d=2048: groups of 32 127 us with
  // 32 columns and spills, 118 with 16; groups of 64 85 and 77).
  constexpr int LC = GPB == 1 && (N == 32 || N == 64) ? 32 : 16;
  const int warp = (int)(threadIdx.x >> 5) - R::EXPAND, lane = threadIdx.x & 31;
  const int t = (warp >> 2) & 1, quad = warp & 3, row = t * 128 + quad * 32 + lane, from = (warp >> 3) * NC;
  const uint32_t at0 = tbase + ((uint32_t)(quad * 32) << 16) + R::D_COL + (uint32_t)(t * N + from);
  // A row's scales lie far from the next row's, so a warp's load touches 32
  // sectors whatever it takes of each: groups below 128 take SW words of bf16
  // (two groups each, SPL stages' worth) or a block's groups of f32 at a time
  // where the rows allow it (64 rows, V=151936, d=2048, groups of 32: 215 us with
  // single loads, 144 so; with groups of 128 the shifting costs more than the
  // two loads per stage, 46.1 against 44.4 us for one row).
  constexpr int SW = N > 64 && GPB < 4 ? 2 : 4, SPL = SW / GPB;
  constexpr bool WORDS = !F32 && GPB > 1;
  const bool lane0 = lane == 0;
  const uint32_t full = smem_u32(MERGED ? sh.done[t] : sh.dfull[t]);
  const uint32_t ready = smem_u32(sh.ready[t]), dempty = smem_u32(sh.dempty[t]);
  uint32_t fp = 0, late = 0;  // parities of done[t][j] (groups of 128) or dfull[t][slot], a bit each
  int slot = 0;
  if (MERGED) arrive(ready, lane0);  // the first block's accumulator is free
  Work w(g);
  while (w.next(g)) {
    const int v = w.tile / g.nchunks * BM + row, chunk = w.tile % g.nchunks;
    const int64_t s0 = (int64_t)min(v, g.V - 1) * g.ngroups;
    float acc[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[c] = 0.f;
    float s[2][WORDS ? 1 : GPB];
    uint32_t cur[WORDS ? SW : 1], nxt[WORDS ? SW : 1];  // from this stage on, and the next load's
    auto fetch = [&](int j, int b) {  // (clamped: groups past the end are never used)
      const float *p = static_cast<const float *>(g.scales) + s0;
      if constexpr (!F32) {
        s[j][0] = __bfloat162float(__ldg(static_cast<const __nv_bfloat16 *>(g.scales) + s0 + min(b, g.ngroups - 1)));
      } else if (GPB > 1 && g.wide_scales) {
        p += min(b * GPB, g.ngroups - GPB);
        if constexpr (GPB == 4) {
          const float4 x = __ldg(reinterpret_cast<const float4 *>(p));
          s[j][0] = x.x, s[j][1] = x.y, s[j][2] = x.z, s[j][3] = x.w;
        } else if constexpr (GPB == 2) {
          const float2 x = __ldg(reinterpret_cast<const float2 *>(p));
          s[j][0] = x.x, s[j][1] = x.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < GPB; ++i) s[j][i] = __ldg(p + min(b * GPB + i, g.ngroups - 1));
      }
    };
    auto load = [&](int k, uint32_t (&x)[WORDS ? SW : 1]) {  // of stages [k, k + SPL)
      if constexpr (WORDS) {
      const uint16_t *p = static_cast<const uint16_t *>(g.scales) + s0;
      if (g.wide_scales) {
        p += min(k * 2 * GPB, g.ngroups - 2 * SW);
        if constexpr (SW == 4) {
          const uint4 y = __ldg(reinterpret_cast<const uint4 *>(p));
          x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
        } else {
          const uint2 y = __ldg(reinterpret_cast<const uint2 *>(p));
          x[0] = y.x, x[1] = y.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < SW; ++i)
          x[i] = (uint32_t)__ldg(p + min(k * 2 * GPB + 2 * i, g.ngroups - 1)) |
                 (uint32_t)__ldg(p + min(k * 2 * GPB + 2 * i + 1, g.ngroups - 1)) << 16;
      }
      }
    };
    auto step = [&]() {  // to the next stage of a load
      if constexpr (WORDS) {
#pragma unroll
        for (int i = 0; i + GPB < SW; ++i) cur[i] = cur[i + GPB];
      }
    };
    if constexpr (!WORDS) {
      fetch(0, w.b0());
      fetch(1, w.b0() + 1);
    } else {
      const int k = w.k0 & ~(SPL - 1);
      load(k, cur);
      load(k + SPL, nxt);
      for (int i = k; i < w.k0; ++i) step();
    }
    for (int k = w.k0; k < w.k1 && !late; ++k) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int b = 2 * k + j;
        if (j == 1 && b >= g.nblk) break;
        const int groups = GPB == 1 ? 1 : min(GPB, (g.d - b * KB) / (KB / GPB));
#pragma unroll
        for (int gi = 0; gi < GPB; ++gi) {
          if (gi >= groups) break;
          const int q = MERGED ? j : (R::LANES == 2 ? j * RING : 0) + (slot >> (R::LANES == 2 ? j : 0) & 1);
          await(full + 8u * q, (fp >> q) & 1u, late);
          fp ^= 1u << q;
          if (RING == 2) slot ^= 1 << (R::LANES == 2 ? j : 0);
          tc_fence_after();
          const uint32_t at = at0 + (R::SLOTS == 1 ? 0u : (uint32_t)q * 2u * N);
#pragma unroll
          for (int c0 = 0; c0 < NC; c0 += LC) {
            uint32_t r[LC / 16][16];
#pragma unroll
            for (int c = 0; c < LC / 16; ++c) tmem_ld16(at + (uint32_t)(c0 + 16 * c), r[c]);
            tmem_wait_ld();
            if (c0 + LC == NC) {  // all is in registers: the accumulator is free
              tc_fence_before();
              // (merged: for the next block)
              arrive(!MERGED ? dempty + 8u * q : ready + 8u * (j == 0 && b + 1 < g.nblk ? 1 : 0), lane0);
            }
            float scale;
            if constexpr (!WORDS) {
              scale = s[j][gi];
            } else {
              const int i = j * GPB + gi;
              scale = __uint_as_float(i & 1 ? cur[i / 2] & 0xFFFF0000u : cur[i / 2] << 16);
            }
#pragma unroll
            for (int c = 0; c < LC; c += 2)
              fma2(acc[c0 + c], acc[c0 + c + 1], r[c / 16][c % 16], r[c / 16][c % 16 + 1], scale);
          }
        }
        if constexpr (!WORDS) fetch(j, b + 2);
      }
      if constexpr (WORDS) {
        if (((k + 1) & (SPL - 1)) == 0) {
#pragma unroll
          for (int i = 0; i < SW; ++i) cur[i] = nxt[i];
          load(k + 1 + SPL, nxt);
        } else {
          step();
        }
      }
    }
    if (late) raise(g, sh);
    if (w.k0 == 0 && w.k1 == g.nks) {
#pragma unroll
      for (int c0 = 0; c0 < NC; c0 += 16)
        if (!late) put16(g, v, chunk, from + c0, acc + c0);
      continue;
    }
    // a shared tile: leave the part (the counting warp sees an error by itself)
    const int which = w.k0 == 0 ? 1 : 0, cols = min(g.rows, g.B - chunk * g.rows);
    float *part = g.parts + ((size_t)blockIdx.x * 2 + which) * (size_t)g.n * BM + row;
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (from + c < cols) __stcg(part + (from + c) * BM, acc[c]);
    bar_arrive<N>(1 + which);
  }
  // the shared tiles for which this CTA's part was the last: add the parts in the order of the columns
  bar_sync<N>(3);
  Work again(g);
  while (again.next(g)) {
    const int which = again.k0 == 0 ? 1 : 0;
    if ((again.k0 == 0 && again.k1 == g.nks) || !sh.last[which]) continue;
    const int v = again.tile / g.nchunks * BM + row;
    const uint32_t first = (uint32_t)again.tile * (uint32_t)g.nks;
    int c_lo, c_hi;
    sharers(g, again.tile, c_lo, c_hi);
    const int chunk = again.tile % g.nchunks, cols = min(g.rows, g.B - chunk * g.rows);
    // columns at a time, and parts: with more of either the wide sizes spill and
    // the narrow ones lose registers elsewhere (128 rows, V=4099, d=1024: 30.7 us
    // with one part at a time, 29.4 with two, 34.0 with four)
    constexpr int JC = NC < 128 ? 16 : 32, JP = NC < 128 ? 1 : 2;
#pragma unroll 1
    for (int c0 = from; c0 < min(cols, from + NC); c0 += JC) {
      float sum[JC] = {};
#pragma unroll JP
      for (int q = c_lo; q < c_hi; ++q) {
        const float *p = g.parts + ((size_t)q * 2 + (unit_start(g, q) <= first ? 1 : 0)) * (size_t)g.n * BM + row;
        float x[JC];  // (columns past the last read it again: no load waits for another)
#pragma unroll
        for (int c = 0; c < JC; ++c) x[c] = __ldcg(p + min(c0 + c, cols - 1) * BM);
#pragma unroll
        for (int c = 0; c < JC; ++c) sum[c] += x[c];
      }
#pragma unroll
      for (int c = 0; c < JC; c += 16)
        if (c0 + c < cols) put16(g, v, chunk, c0 + c, sum + c);
    }
  }
}

// Counts the parts of the shared tiles as they are written.
template <int N>
__device__ void count_parts(const Gemm &g, Sh &sh, int lane) {
  Work w(g);
  while (w.next(g)) {
    if (w.k0 == 0 && w.k1 == g.nks) continue;
    const int which = w.k0 == 0 ? 1 : 0;
    bar_sync<N>(1 + which);
    if (lane == 0) {
      int c_lo, c_hi;
      sharers(g, w.tile, c_lo, c_hi);
      __threadfence();  // this CTA's part before the count
      sh.last[which] = !aborted(sh) && (int)atomicAdd(&g.counters[w.tile], 1u) == c_hi - c_lo - 1;
      __threadfence();  // the count before the others' parts
    }
    __syncwarp();
  }
  bar_arrive<N>(3);
}

template <int N, int GPB>
__global__ void __launch_bounds__(Roles<N>::THREADS, 1)
    w4_gemm_kernel(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap th, const Gemm g) {
  using R = Roles<N>;
  extern __shared__ __align__(1024) uint8_t w4_smem_raw[];
  __shared__ Sh sh;
  uint8_t *smem = w4_smem_raw + ((1024u - (smem_u32(w4_smem_raw) & 1023u)) & 1023u);
  uint8_t *sW = smem, *sH = smem + (size_t)g.wstages * W_BYTES;
  constexpr int FIRST = R::EXPAND + R::SUM;  // the weight producer's warp; the hidden rows' and the issuers' follow
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int s = 0; s < MAX_WS; ++s) {
      mbar_init(&sh.wfull[s], 1);
      mbar_init(&sh.wempty[s], R::EXPAND);
    }
    for (int s = 0; s < MAX_HS; ++s) {
      mbar_init(&sh.hfull[s], 1);
      mbar_init(&sh.hempty[s], 2);
    }
    for (int t = 0; t < 2; ++t) {
      for (int j = 0; j < 2; ++j) {
        mbar_init(&sh.ready[t][j], 4 + (R::template merged<GPB>() ? R::SUM / 2 : 0));
        mbar_init(&sh.done[t][j], 1);
      }
      for (int j = 0; j < 4; ++j) {
        mbar_init(&sh.dfull[t][j], 1);
        mbar_init(&sh.dempty[t][j], R::SUM / 2);
      }
    }
    for (int j = 0; j < 4; ++j) mbar_init(&sh.mma_done[j], 1);
    sh.abort = 0;
    fence_barrier_init();
  }
  if (warp == FIRST) {
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
  if (warp < R::EXPAND) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R::REGS_EXPAND));
    expand_rows<N, GPB>(g, sh, sW, tbase);
  } else if (warp < FIRST) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R::REGS_SUM));
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (g.scale_dtype == MSTAR_DTYPE_F32)
      sum_rows<N, GPB, true>(g, sh, tbase);
    else
      sum_rows<N, GPB, false>(g, sh, tbase);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R::REGS_REST));
    if (warp == FIRST) {
      if (lane == 0) produce_weights(g, sh, sW, &tw);
    } else if (warp == FIRST + 1) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      asm volatile("fence.proxy.async;" ::: "memory");
      if (lane == 0) produce_hidden<N>(g, sh, sH, &th);
    } else if (warp < FIRST + 2 + R::ISSUE) {
      issue<N, GPB>(g, sh, sH, tbase, warp - FIRST - 2);
    }
    if (warp == FIRST + R::COUNTER) {
      __syncwarp();
      asm volatile("griddepcontrol.wait;" ::: "memory");
      count_parts<N>(g, sh, lane);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == FIRST) {
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
  g.nks = (d + KS - 1) / KS;
  g.nblk = (d + KB - 1) / KB;
  const int tiles = (V + BM - 1) / BM;
  g.nchunks = (B + MAX_N - 1) / MAX_N;
  // Chunks of up to 128 rows read and expand each code least often, but their
  // blocks take turns in one accumulator and their shared tiles are long to add.
  // With few units per SM narrower chunks win: 64 rows while that makes at most
  // 16 units per SM (128 rows, groups of 128, d=2048: V=16384 41 -> 27 us, V=32000
  // 54 -> 42; at V=50000 they would gain too, 69 -> 57, but with groups of 32 and
  // d=4096 lose, 112 -> 123), down to 16 rows while at most 4 (128 rows, d=1024,
  // V=4099: 29 -> 16 us; at 6, V=8192, d=2048, groups of 64: 25 -> 28).
  const int64_t units = (int64_t)tiles * g.nks, sms = sm_count();
  if (units * ((B + 63) / 64) <= 16 * sms) g.nchunks = (B + 63) / 64;
  g.nchunks = (int)std::max<int64_t>(g.nchunks, std::min<int64_t>(4 * sms / units, (B + 15) / 16));
  g.rows = (B + g.nchunks - 1) / g.nchunks;
  g.nchunks = (B + g.rows - 1) / g.rows;
  g.n = (g.rows + 15) & ~15;
  g.ntt = tiles * g.nchunks;
  // (64 rows, V=151936, d=2048: 83 us with three hidden stages, 77 with four; a
  // multiple of the lanes that Roles gives each width)
  g.hstages = g.n <= 16 ? 8 : g.n <= 32 ? 6 : g.n <= 64 ? 4 : 3;
  g.wstages = std::min(MAX_WS, (SMEM_BUDGET - g.hstages * g.n * KB * 2) / W_BYTES);
  return g;
}

// A CTA per SM.  Where the units are too few for that, a tile's columns are split
// over as many CTAs as balance the units each of them takes with the parts one of
// them adds: a divisor of the stages at or above their square root (16 x 1024 x
// 4096: 20.5 us with sixteen parts, 15.3 with four).  Up to seven stages one unit
// per CTA is quicker (16 x 4099 x 1024: 12.3 us with four parts, 13.4 with two).
// Where the least such divisor is more than twice the root (a prime number of
// stages has itself alone), six parts, or the root where that is more, although
// shares then differ by a unit: 11, 13, 17, 19 and 23 stages, 16 rows, V=2048 16.4,
// 18.6, 24.0, 24.3 and 28.3 us with a part per stage, 16.4, 16.5, 18.1, 18.8 and
// 20.3 with six.  (A divisor that is near is quicker: 15 stages 16.1 us with five
// parts, 19.0 with four.)
static int grid_of(const Gemm &g) {
  int parts = g.nks;
  if (g.nks >= 8) {
    int root = 1;
    while (root * root < g.nks) ++root;
    for (int p = g.nks - 1; p >= root; --p)
      if (g.nks % p == 0) parts = p;
    if (parts * parts > 4 * g.nks) parts = std::max(6, root);
  }
  return (int)std::min<int64_t>(sm_count(), (int64_t)g.ntt * parts);
}

// Workspace: arrival counters, the hidden rows as operands, their scales, the
// parts of shared tiles; each rounded to 256 bytes.  Sized by what any batch of
// up to B rows may take (the chunks' width goes up and down with B), so that a
// workspace for the largest batch serves the smaller ones.
static int64_t up(int64_t b) { return (b + 255) / 256 * 256; }
static int64_t hidden_at(const Gemm &g) { return up((int64_t)((g.V + BM - 1) / BM) * ((g.B + 15) / 16) * 4); }
static int64_t scale_at(const Gemm &g) { return hidden_at(g) + up((int64_t)g.B * g.d * 2); }
static int64_t parts_at(const Gemm &g) { return scale_at(g) + up((int64_t)g.B * 4); }
static int64_t workspace_bytes(const Gemm &g) {
  return parts_at(g) + (int64_t)sm_count() * 2 * std::min(MAX_N, (g.B + 15) / 16 * 16) * BM * 4;
}

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
  const int rc = allow_smem<w4_gemm_kernel<N, GPB>>(smem);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid_of(g), 1, 1);
  cfg.blockDim = dim3(Roles<N>::THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tw, th, g);
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
                  void *ws, int64_t ws_bytes, uint32_t *err, bool withhold, cudaStream_t st) {
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
  const uint32_t units = (uint32_t)g.ntt * (uint32_t)g.nks, grid = (uint32_t)grid_of(g);
  g.share = units / grid;
  g.longer = units % grid;
  g.group = w->group;
  g.ngroups = w->d / w->group;
  g.scales = w->scales;
  g.scale_dtype = w->scale_dtype;
  g.zeros = static_cast<const uint8_t *>(w->zeros);
  // rows of eight groups each way: 16 bytes of scales, 8 of zero points
  g.wide_scales = g.ngroups % 8 == 0 && reinterpret_cast<uintptr_t>(w->scales) % 16 == 0;
  g.wide_zeros = g.ngroups % 8 == 0 && reinterpret_cast<uintptr_t>(w->zeros) % 8 == 0;
  g.out = out;
  g.ld = ld;
  g.out_dtype = dtype;
  g.err = err;
  g.withhold = withhold;
  g.counters = reinterpret_cast<uint32_t *>(p);
  g.parts = reinterpret_cast<float *>(p + parts_at(g));
  void *perm = p + hidden_at(g);
  CUtensorMap tw, th;
  if ((rc = make_map(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, w->codes, w->V, w->d / 2, KS / 2, BM))) return rc;
  if ((rc = make_map(&th, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, perm, B, w->d, 64, g.n))) return rc;
  const int vec = (reinterpret_cast<uintptr_t>(hidden) % 16 == 0 && ldh % 8 == 0) ? 1 : 0;
  float *row_scale = reinterpret_cast<float *>(p + scale_at(g));
  g.row_scale = row_scale;
  w4_prepare_kernel<<<B, PREP_NT, 0, st>>>(static_cast<const __nv_bfloat16 *>(hidden), ldh, w->d, vec,
                                           static_cast<uint4 *>(perm), row_scale, g.counters, g.ntt);
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
  return w4::logits(hidden, ld_hidden, B, w, logits, dtype, ld, workspace, workspace_bytes, status, false,
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
  rc = w4::logits(hidden, ld_hidden, p->B, w, const_cast<void *>(p->logits), p->dtype, p->ld, workspace,
                  workspace_bytes, status, (p->flags & MSTAR_FLAG_TEST_WITHHOLD) != 0, static_cast<cudaStream_t>(stream));
  return rc ? rc : mstar_sampler_step(p, stream);
}

}  // extern "C"
