// Embedding lookup with scaling, and its gradient by sorted tokens: the other
// end of the LM head's table.
//
//   out[n] = scale * table[ids[n]]          (a negative id: a row of zeros)
//   grad[v] = base[v] + scale * sum over n with ids[n] = v of dout[n]
//
// Lookup: a copy bound by memory; every thread moves one vector of eight
// values (from 16 or 32 bytes of a plain table, 4 of a 4-bit one) for several
// (row, column) places at once.
//
// Gradient: the tokens are sorted by id first, so each row of the table is
// summed by one owner in position order (no atomics on values: the same
// inputs give the same bits).
//   fill   the whole output: zeros, or the base.  It is most of the bytes where
//          the table is large, takes no heed of rows (an odd width would leave
//          them unaligned) and runs beside the sort; the rows that have tokens
//          are written over it.
//   sort   CTA c of C (a power of two) takes the ids v with v mod C = c, which
//          spreads frequent neighbours, and reads all ids twice: once to count
//          (per id and per warp, each warp owning a contiguous part of the
//          positions), once to place.  It counts the ids of the CTAs before it
//          as it goes, so CTAs need nothing of one another.  The order of the
//          ids is then (v mod C, v / C); all that matters is that an id's
//          tokens lie together, in position order.
//   sums   the sorted positions in chunks of equal length, whatever the ids'
//          frequencies; a chunk writes the runs that start in it, and long runs
//          that cross its borders leave 32-bit partial sums.
//   joins  the parts of each long run that crosses borders are added in order.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"

namespace mstar {
namespace emb {

constexpr int NT = 256;

// A load of memory that the kernel only reads (RO), or of any.
template <bool RO, typename A>
__device__ __forceinline__ A get(const A *p) {
  if constexpr (RO)
    return __ldg(p);
  else
    return *p;
}
// W consecutive values as one access (W = 8: 16 bytes of bf16, two of 16 of f32).
template <int W, bool RO = true>
__device__ __forceinline__ void load(const float *p, float (&x)[W]) {
  if constexpr (W == 8) {
    const float4 a = get<RO>(reinterpret_cast<const float4 *>(p)), b = get<RO>(reinterpret_cast<const float4 *>(p) + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else if constexpr (W == 2) {
    const float2 a = get<RO>(reinterpret_cast<const float2 *>(p));
    x[0] = a.x, x[1] = a.y;
  } else {
    x[0] = get<RO>(p);
  }
}
template <int W, bool RO = true>
__device__ __forceinline__ void load(const __nv_bfloat16 *p, float (&x)[W]) {
  if constexpr (W == 8) {
    const uint4 a = get<RO>(reinterpret_cast<const uint4 *>(p));
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  } else if constexpr (W == 2) {
    const uint32_t u = get<RO>(reinterpret_cast<const uint32_t *>(p));
    x[0] = __uint_as_float(u << 16);
    x[1] = __uint_as_float(u & 0xFFFF0000u);
  } else {
    x[0] = __bfloat162float(p[0]);
  }
}
// 16 bytes as four floats or eight bf16.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4 &w, float *x) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      x[i] = __uint_as_float(u[i]);
    } else {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
}
template <int W>
__device__ __forceinline__ void store(float *p, const float (&x)[W]) {
  if constexpr (W == 8) {
    __stcs(reinterpret_cast<float4 *>(p), make_float4(x[0], x[1], x[2], x[3]));
    __stcs(reinterpret_cast<float4 *>(p) + 1, make_float4(x[4], x[5], x[6], x[7]));
  } else if constexpr (W == 2) {
    *reinterpret_cast<float2 *>(p) = make_float2(x[0], x[1]);
  } else {
    *p = x[0];
  }
}
template <int W>
__device__ __forceinline__ void store(__nv_bfloat16 *p, const float (&x)[W]) {
  if constexpr (W == 8) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    __stcs(reinterpret_cast<uint4 *>(p), make_uint4(u[0], u[1], u[2], u[3]));
  } else if constexpr (W == 2) {
    *reinterpret_cast<__nv_bfloat162 *>(p) = __floats2bfloat162_rn(x[0], x[1]);
  } else {
    *p = __float2bfloat16_rn(x[0]);
  }
}

// ------------------------------------------------------------ lookup

struct Lookup {
  const void *table;
  int64_t ld;  // table row stride in values
  const int64_t *ids;
  int64_t N;
  int32_t V, d;
  float scale;
  void *out;  // [N, d]
  uint32_t *status;
  // 4-bit tables
  const uint8_t *codes;
  const void *scales;
  const uint8_t *zeros;
  int32_t scale_dtype, group_log2, ngroups;
};

__device__ __forceinline__ void bad_id(const Lookup &a, int64_t id, int col) {
  if (id >= a.V && col == 0 && a.status) atomicOr(a.status, MSTAR_STATUS_BAD_ID);
}

// i / per: a 64-bit division is some seventy instructions, and most lookups have
// fewer than 2^32 places.
__device__ __forceinline__ int64_t row_of(int64_t i, uint32_t per, bool small) {
  return small ? (int64_t)((uint32_t)i / per) : i / per;
}

// Rows that 16-byte accesses do not fit (an odd width, an unaligned view): a
// block per row, W values per access.
template <typename TI, typename TO, int W>
__global__ void __launch_bounds__(NT) embed_rows_kernel(const Lookup a) {
  constexpr int U = 4;
  const int64_t n = blockIdx.x;
  const int64_t id = a.ids[n];
  const bool ok = id >= 0 && id < a.V;
  if (threadIdx.x == 0) bad_id(a, id, 0);
  const TI *from = static_cast<const TI *>(a.table) + (ok ? id : 0) * a.ld;
  TO *to = static_cast<TO *>(a.out) + n * a.d;
  for (int col = (int)threadIdx.x * W; col < a.d; col += NT * W * U) {
    float x[U][W] = {};
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (ok && col + u * NT * W < a.d) load<W>(from + col + u * NT * W, x[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (col + u * NT * W >= a.d) break;
#pragma unroll
      for (int j = 0; j < W; ++j) x[u][j] *= a.scale;
      store<W>(to + col + u * NT * W, x[u]);
    }
  }
}

template <typename TI, typename TO, int W>
__global__ void __launch_bounds__(NT) embed_kernel(const Lookup a) {
  constexpr int U = 4;
  const uint32_t per = (uint32_t)(a.d / W);
  const int64_t total = a.N * (int64_t)per;
  const bool small = total <= 0xFFFFFFFFll;
  const int64_t i0 = (int64_t)blockIdx.x * (NT * U) + threadIdx.x;
  float x[U][W];
  int64_t at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = i0 + u * NT;
    at[u] = -1;
    if (i >= total) continue;
    const int64_t n = row_of(i, per, small);
    const int col = (int)(i - n * per) * W;
    const int64_t id = a.ids[n];
    at[u] = n * a.d + col;
    bad_id(a, id, col);
    if (id >= 0 && id < a.V) {
      load<W>(static_cast<const TI *>(a.table) + id * a.ld + col, x[u]);
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) x[u][j] = 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (at[u] < 0) continue;
#pragma unroll
    for (int j = 0; j < W; ++j) x[u][j] *= a.scale;
    store<W>(static_cast<TO *>(a.out) + at[u], x[u]);
  }
}

// Eight values (one word of codes, all of one group) per place.
template <typename TO>
__global__ void __launch_bounds__(NT) embed_w4_kernel(const Lookup a) {
  constexpr int U = 4;
  const uint32_t per = (uint32_t)a.d / 8;
  const int64_t total = a.N * (int64_t)per;
  const bool small = total <= 0xFFFFFFFFll;
  const int64_t i0 = (int64_t)blockIdx.x * (NT * U) + threadIdx.x;
  uint32_t w[U];
  float s[U], z[U];
  int64_t at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = i0 + u * NT;
    at[u] = -1;
    if (i >= total) continue;
    const int64_t n = row_of(i, per, small);
    const int col = (int)(i - n * per) * 8;
    const int64_t id = a.ids[n];
    at[u] = n * a.d + col;
    w[u] = 0u;
    s[u] = z[u] = 0.f;
    bad_id(a, id, col);
    if (id < 0 || id >= a.V) continue;
    w[u] = __ldg(reinterpret_cast<const uint32_t *>(a.codes + id * (a.d / 2) + col / 2));
    const int64_t g = id * a.ngroups + (col >> a.group_log2);
    s[u] = a.scale_dtype == MSTAR_DTYPE_F32 ? __ldg(static_cast<const float *>(a.scales) + g)
                                            : __bfloat162float(static_cast<const __nv_bfloat16 *>(a.scales)[g]);
    z[u] = a.zeros ? (float)(__ldg(a.zeros + g) & 15) : 8.f;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (at[u] < 0) continue;
    float x[8];
    // (q - z) s as stored weights are used elsewhere, then the lookup's scale
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = ((float)((w[u] >> (4 * j)) & 15u) - z[u]) * s[u] * a.scale;
    store<8>(static_cast<TO *>(a.out) + at[u], x);
  }
}

// ------------------------------------------------------------ gradient

constexpr int SORT_NT = 1024;
constexpr int SORT_NW = SORT_NT / 32;
constexpr int SORT_U = 8;        // ids per lane and step
constexpr int MAX_BINS = SORT_NT;  // ids per CTA of the sort
constexpr int SUM_NT = 128;
constexpr int JOIN_G = 8;
constexpr int MAX_CHUNK = 128;
constexpr int STAGE_BYTES = 28 * 1024;  // (seven CTAs of the sums per SM: 1036, one wave of the usual thousand)
constexpr int LONG_RUN = 32;  // a run of at most this many tokens belongs to the chunk in which it starts

struct Grad {
  const void *dout;
  int64_t ldo;  // dout row stride in values
  const int64_t *ids;
  int32_t N, V, d;
  float scale;
  const void *base;  // [V, d] of the output's type, or NULL
  void *out;         // [V, d]
  uint32_t *status;
  int32_t bins, c_log2;  // ids per CTA of the sort, and how many CTAs
  int32_t chunk, nchunks, col_tiles;
  int32_t *start;    // [C * bins + 1] first sorted place of each id, in the sort's order of ids
  int32_t *pos;      // [N] positions, sorted by id, then by position
  int32_t *key;      // [N] their ids
  float *part;       // [nchunks][2][d]: a run from the chunk before / into the chunk after
};

// out = base, or zeros, as 16-byte vectors between single bytes.
constexpr int FILL_NT = 256, FILL_U = 4;
__global__ void __launch_bounds__(FILL_NT) fill_kernel(uint8_t *out, const uint8_t *base, int64_t bytes) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t stride = (int64_t)gridDim.x * FILL_NT, me = (int64_t)blockIdx.x * FILL_NT + threadIdx.x;
  const int64_t head = min(bytes, (int64_t)(-reinterpret_cast<intptr_t>(out) & 15));
  const bool vec = !base || ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(base)) & 15u) == 0;
  const int64_t nv = vec ? (bytes - head) / 16 : 0;
  uint4 *o = reinterpret_cast<uint4 *>(out + head);
  const uint4 *b = base ? reinterpret_cast<const uint4 *>(base + head) : nullptr;
  int64_t i = me;
  for (; i + (FILL_U - 1) * stride < nv; i += FILL_U * stride) {
    uint4 w[FILL_U];
#pragma unroll
    for (int u = 0; u < FILL_U; ++u) w[u] = b ? __ldcs(b + i + u * stride) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int u = 0; u < FILL_U; ++u) __stcs(o + i + u * stride, w[u]);
  }
  for (; i < nv; i += stride) __stcs(o + i, b ? __ldcs(b + i) : make_uint4(0u, 0u, 0u, 0u));
  // what the vectors leave: pairs of bytes (both types are of two or four)
  const int64_t rest = bytes - nv * 16;
  for (i = me * 2; i < rest; i += stride * 2) {
    const int64_t at = i < head ? i : i + nv * 16;
    *reinterpret_cast<uint16_t *>(out + at) = base ? *reinterpret_cast<const uint16_t *>(base + at) : (uint16_t)0;
  }
}

// An id's place in the sort's order.
__device__ __forceinline__ int rank_of(const Grad &a, int v) {
  return (v & ((1 << a.c_log2) - 1)) * a.bins + (v >> a.c_log2);
}

// (40 registers: the fill's blocks keep their place on the SM beside a block of this)
__global__ void __maxnreg__(40) sort_tokens_kernel(const Grad a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(16) int32_t cnt[];  // [SORT_NW][bins]
  __shared__ int32_t below_w[SORT_NW], scan_w[SORT_NW];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int me = (int)blockIdx.x, mask = (1 << a.c_log2) - 1;
  for (int i = tid; i < SORT_NW * a.bins / 4; i += SORT_NT) reinterpret_cast<int4 *>(cnt)[i] = make_int4(0, 0, 0, 0);
  __syncthreads();
  const int n0 = (int)((int64_t)a.N * warp / SORT_NW), n1 = (int)((int64_t)a.N * (warp + 1) / SORT_NW);
  int32_t *mine = cnt + warp * a.bins;
  int id[SORT_U];  // -1: none, or not in the table
  bool bad = false;
  auto load_ids = [&](int n) {
    int64_t x[SORT_U];
#pragma unroll
    for (int u = 0; u < SORT_U; ++u) x[u] = n + 32 * u < n1 ? __ldg(a.ids + n + 32 * u) : -1;
#pragma unroll
    for (int u = 0; u < SORT_U; ++u) {
      bad |= x[u] >= a.V;
      id[u] = x[u] >= 0 && x[u] < a.V ? (int)x[u] : -1;
    }
  };
  int below = 0;
  for (int nb = n0; nb < n1; nb += 32 * SORT_U) {  // (the same steps for every lane: each gets its ids, or -1)
    load_ids(nb + lane);
#pragma unroll
    for (int u = 0; u < SORT_U; ++u) {
      const int c = id[u] & mask;
      below += id[u] >= 0 && c < me;
      if (id[u] >= 0 && c == me) atomicAdd(&mine[id[u] >> a.c_log2], 1);
    }
  }
  if (bad && me == 0 && a.status) atomicOr(a.status, MSTAR_STATUS_BAD_ID);
  below = __reduce_add_sync(~0u, below);
  if (lane == 0) below_w[warp] = below;
  __syncthreads();
  // exclusive prefix over the ids (a thread each), then over the warps of each id
  int tot = 0;
  if (tid < a.bins)
    for (int w = 0; w < SORT_NW; ++w) tot += cnt[w * a.bins + tid];
  int inc = tot;
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(~0u, inc, o);
    if (lane >= o) inc += t;
  }
  if (lane == 31) scan_w[warp] = inc;
  __syncthreads();
  const int first = __reduce_add_sync(~0u, below_w[lane]);
  const int before = __reduce_add_sync(~0u, lane < warp ? scan_w[lane] : 0);
  const int all = __reduce_add_sync(~0u, scan_w[lane]);
  int at = first + before + inc - tot;
  if (tid < a.bins) {
    a.start[me * a.bins + tid] = at;
    for (int w0 = 0; w0 < SORT_NW; w0 += 8) {
      int t[8];
#pragma unroll
      for (int w = 0; w < 8; ++w) t[w] = cnt[(w0 + w) * a.bins + tid];
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        cnt[(w0 + w) * a.bins + tid] = at;
        at += t[w];
      }
    }
  }
  if (tid == 0 && me == mask) a.start[(mask + 1) * a.bins] = first + all;
  __syncthreads();
  const bool kept = n1 - n0 <= 32 * SORT_U;  // the counting step's ids are still here
  for (int nb = n0; nb < n1; nb += 32 * SORT_U) {
    if (!kept) load_ids(nb + lane);
#pragma unroll
    for (int u = 0; u < SORT_U; ++u) {
      const bool in = id[u] >= 0 && (id[u] & mask) == me;
      if (!__any_sync(~0u, in)) continue;
      const int b = in ? id[u] >> a.c_log2 : -1;
      const unsigned same = __match_any_sync(~0u, b);
      const int rank = __popc(same & ((1u << lane) - 1u));
      int to = 0;
      if (in) to = mine[b] + rank;
      __syncwarp();
      if (in && rank == 0) mine[b] = to + __popc(same);
      __syncwarp();
      if (in) {
        a.pos[to] = nb + 32 * u + lane;
        a.key[to] = id[u];
      }
    }
  }
  // the fill runs beside this; what comes after both waits for this kernel alone
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// (base may be the output, whose rows this kernel writes: no read-only load)
template <typename TO, int W>
__device__ __forceinline__ void load_base(const Grad &a, int v, int col, float (&b)[W]) {
  if (a.base) load<W, false>(static_cast<const TO *>(a.base) + (int64_t)v * a.d + col, b);
}
template <typename TO, int W>
__device__ __forceinline__ void finish(const Grad &a, int v, int col, float (&acc)[W], const float (&b)[W]) {
#pragma unroll
  for (int j = 0; j < W; ++j) acc[j] *= a.scale;
  if (a.base) {
#pragma unroll
    for (int j = 0; j < W; ++j) acc[j] += b[j];
  }
  store<W>(static_cast<TO *>(a.out) + (int64_t)v * a.d + col, acc);
}

template <typename TI, typename TO, int W>
__global__ void __launch_bounds__(SUM_NT) sum_tokens_kernel(const Grad a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ int32_t skey[MAX_CHUNK + LONG_RUN + 2], spos[MAX_CHUNK + LONG_RUN];
  const int c = (int)blockIdx.x / a.col_tiles;
  const int col = (((int)blockIdx.x % a.col_tiles) * SUM_NT + (int)threadIdx.x) * W;
  const int s0 = c * a.chunk, most = min(a.N, s0 + a.chunk + LONG_RUN) - s0;  // tokens that may be this chunk's
  const int total = a.start[a.bins << a.c_log2];  // (places past it hold nothing; they are masked below)
  // the chunk's ids and positions first, so that the rows' loads wait for nothing
  for (int i = (int)threadIdx.x; i < most + 2; i += SUM_NT) {
    const int s = s0 - 1 + i;
    const int key = s >= 0 && s < a.N ? a.key[s] : -1, pos = i < most ? a.pos[s0 + i] : 0;
    skey[i] = s < total ? key : -1;
    if (i < most) spos[i] = pos;
  }
  const int s1 = min(total, s0 + a.chunk);
  if (s0 >= s1) return;
  __syncthreads();
  bool from_before = skey[0] == skey[1];
  int begin = 0, end = s1 - s0;
  if (from_before) {  // a short run that started before is not this chunk's
    const int r = rank_of(a, skey[1]), stop = a.start[r + 1];
    if (stop - a.start[r] <= LONG_RUN) begin = stop - s0, from_before = false;
  }
  if (begin >= end) return;
  if (skey[end] == skey[end + 1]) {  // a short run that goes on behind is
    const int r = rank_of(a, skey[end]), stop = a.start[r + 1];
    if (stop - a.start[r] <= LONG_RUN) end = stop - s0;
  }
  if (col >= a.d) return;
  // A batch of rows is in flight at once, through registers; with 16-byte
  // accesses through asynchronous copies into shared memory, the next batch
  // while one is added (each thread reads back only what it copied itself).  30011
  // tokens of 1024 bf16 over 4099 ids: 59.3 us with one batch of 32 KB, 57.1 so.
  constexpr int BATCH = W == 8 ? STAGE_BYTES / 2 / (SUM_NT * W * (int)sizeof(TI)) : 8;
  constexpr int PARTS = W * (int)sizeof(TI) / 16;  // 16-byte copies per thread and row
  __shared__ __align__(16) uint8_t stage[W == 8 ? STAGE_BYTES : 16];
  float acc[W] = {}, b[W];
  load_base<TO, W>(a, skey[begin + 1], col, b);  // (read as a run begins: it is there when the run ends)
  uint8_t *half = stage;  // the batch at hand; the next one lands in the other half
  auto copy = [&](int s, uint8_t *to) {
    const int n = min(BATCH, end - s);
    for (int u = 0; u < n; ++u) {
      const TI *from = static_cast<const TI *>(a.dout) + (int64_t)spos[s + u] * a.ldo + col;
#pragma unroll
      for (int i = 0; i < PARTS; ++i)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         smem_u32(to + ((u * PARTS + i) * SUM_NT + (int)threadIdx.x) * 16)),
                     "l"(reinterpret_cast<const uint4 *>(from) + i)
                     : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if constexpr (W == 8) copy(begin, half);
  for (int s = begin; s < end; s += BATCH) {
    const int n = min(BATCH, end - s);
    float x[W == 8 ? 1 : BATCH][W];
    if constexpr (W == 8) {
      copy(s + BATCH, half == stage ? stage + STAGE_BYTES / 2 : stage);  // (past the end: an empty group)
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
#pragma unroll
      for (int u = 0; u < BATCH; ++u)
        if (u < n) load<W>(static_cast<const TI *>(a.dout) + (int64_t)spos[s + u] * a.ldo + col, x[u]);
    }
    auto take = [&](int u, const float *y) {
#pragma unroll
      for (int j = 0; j < W; ++j) acc[j] += y[j];
      const int key = skey[s + u + 1];
      const bool goes_on = skey[s + u + 2] == key;
      if (goes_on && s + u + 1 < end) return;
      if (from_before || goes_on) {  // the run crosses a border of the chunk
        store<W>(a.part + ((int64_t)c * 2 + (from_before ? 0 : 1)) * a.d + col, acc);
      } else {
        finish<TO, W>(a, key, col, acc, b);
      }
      from_before = false;
#pragma unroll
      for (int j = 0; j < W; ++j) acc[j] = 0.f;
      if (s + u + 1 < end) load_base<TO, W>(a, skey[s + u + 2], col, b);
    };
    if constexpr (W == 8) {
      for (int u = 0; u < n; ++u) {
        float y[8];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          const uint4 w = *reinterpret_cast<const uint4 *>(half + ((u * PARTS + i) * SUM_NT + (int)threadIdx.x) * 16);
          unpack16<TI>(w, y + i * (8 / PARTS));
        }
        take(u, y);
      }
      half = half == stage ? stage + STAGE_BYTES / 2 : stage;
    } else {
#pragma unroll
      for (int u = 0; u < BATCH; ++u)
        if (u < n) take(u, x[u]);
    }
  }
}

// CTA i looks at the borders i, i + grid, ... for runs that start before and go
// on behind; JOIN_G groups of threads take such a run's parts in turn (a
// frequent id's run has a hundred), and the first adds the groups' sums in
// their order.
template <typename TO, int W>
__global__ void __launch_bounds__(SUM_NT *JOIN_G) join_tokens_kernel(const Grad a) {
  __shared__ float sums[JOIN_G][SUM_NT * W];
  __shared__ int found[SUM_NT * JOIN_G], nfound;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = (int)threadIdx.x % SUM_NT, group = (int)threadIdx.x / SUM_NT;
  const int col = ((int)blockIdx.y * SUM_NT + lane) * W;
  const int total = a.start[a.bins << a.c_log2];
  const int full = (total - 1) / a.chunk;  // chunks with tokens behind their border
  for (int c0 = (int)blockIdx.x; c0 < full; c0 += (int)gridDim.x * SUM_NT * JOIN_G) {
    __syncthreads();
    if (threadIdx.x == 0) nfound = 0;
    __syncthreads();
    const int mine = c0 + (int)threadIdx.x * (int)gridDim.x;
    if (mine < full) {
      const int s1 = (mine + 1) * a.chunk, id = a.key[s1 - 1], r = rank_of(a, id), first = a.start[r];
      if (a.key[s1] == id && first >= mine * a.chunk && a.start[r + 1] - first > LONG_RUN)
        found[atomicAdd(&nfound, 1)] = mine;
    }
    __syncthreads();
    for (int f = 0; f < nfound; ++f) {  // (their order does not matter: each is an id of its own)
      const int c = found[f], id = a.key[(c + 1) * a.chunk - 1];
      const int last = (a.start[rank_of(a, id) + 1] - 1) / a.chunk;  // the chunk in which it ends
      float acc[W] = {}, b[W];
      if (col < a.d) {
        if (group == 0) load_base<TO, W>(a, id, col, b);
        // part 0 is this chunk's end of the run, part k > 0 chunk c + k's beginning
#pragma unroll 4
        for (int k = group; k <= last - c; k += JOIN_G) {
          float x[W];
          load<W>(a.part + ((int64_t)(c + k) * 2 + (k == 0 ? 1 : 0)) * a.d + col, x);
#pragma unroll
          for (int j = 0; j < W; ++j) acc[j] += x[j];
        }
      }
      __syncthreads();  // the run before has been added
#pragma unroll
      for (int j = 0; j < W; ++j) sums[group][lane + j * SUM_NT] = acc[j];
      __syncthreads();
      if (group == 0 && col < a.d) {
#pragma unroll
        for (int j = 0; j < W; ++j)
          for (int k = 1; k < JOIN_G; ++k) acc[j] += sums[k][lane + j * SUM_NT];
        finish<TO, W>(a, id, col, acc, b);
      }
    }
  }
}

// ------------------------------------------------------------ host side

static int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MSTAR_OK : fail(MSTAR_ERR_CUDA, std::string("launch: ") + cudaGetErrorString(e));
}

static int check_dtype(int dtype, const char *what) {
  if (dtype == MSTAR_DTYPE_F32 || dtype == MSTAR_DTYPE_BF16) return MSTAR_OK;
  return fail(MSTAR_ERR_INVALID, std::string(what) + " must be MSTAR_DTYPE_F32 or MSTAR_DTYPE_BF16");
}

static int es(int dtype) { return dtype == MSTAR_DTYPE_F32 ? 4 : 2; }

// Widest access that every row of a matrix allows: 8 values (16-byte
// accesses), 2 (one access of a pair) or 1.
static int width(const void *p, int64_t ld, int dtype) {
  const uint64_t a = reinterpret_cast<uintptr_t>(p) | (uint64_t)ld * (uint64_t)es(dtype);
  return a % 16 == 0 ? 8 : a % (2 * (uint64_t)es(dtype)) == 0 ? 2 : 1;
}
static int width_of(int d, int w) { return d % 8 == 0 && w == 8 ? 8 : d % 2 == 0 && w >= 2 ? 2 : 1; }

static int check_lookup(const int64_t *ids, int64_t N, int V, int d, const void *out, int out_dtype) {
  if (!ids || !out) return fail(MSTAR_ERR_INVALID, "ids and out must not be NULL");
  if (N < 1 || N > (1 << 28)) return fail(MSTAR_ERR_INVALID, "N must be in [1, 2^28]");
  if (V < 1 || V > (1 << 21)) return fail(MSTAR_ERR_INVALID, "V must be in [1, 2097152]");
  if (d < 1 || d > (1 << 20)) return fail(MSTAR_ERR_INVALID, "d must be in [1, 2^20]");
  int rc = check_dtype(out_dtype, "out_dtype");
  if (rc) return rc;
  if (reinterpret_cast<uintptr_t>(out) & (es(out_dtype) - 1))
    return fail(MSTAR_ERR_INVALID, "out must be aligned to its type");
  if ((N * d + NT * 4 - 1) / (NT * 4) > 0x7FFFFFFF) return fail(MSTAR_ERR_INVALID, "N * d is too large");
  return MSTAR_OK;
}

template <typename TI, typename TO>
static int launch_lookup(const Lookup &a, int w, cudaStream_t st) {
  if (w == 8)
    embed_kernel<TI, TO, 8><<<(unsigned)((a.N * (a.d / 8) + NT * 4 - 1) / (NT * 4)), NT, 0, st>>>(a);
  else if (w == 2)
    embed_rows_kernel<TI, TO, 2><<<(unsigned)a.N, NT, 0, st>>>(a);
  else
    embed_rows_kernel<TI, TO, 1><<<(unsigned)a.N, NT, 0, st>>>(a);
  return launched();
}

// CTAs of the sort: a power of two that leaves each at most MAX_BINS ids, and
// enough of them to fill the GPU.
static int sort_log2(int V) {
  int l = 7;
  while (((V + (1 << l) - 1) >> l) > MAX_BINS) ++l;
  return l;
}
static int sort_bins(int V) { return (((V + (1 << sort_log2(V)) - 1) >> sort_log2(V)) + 3) / 4 * 4; }

// Workspace: start [C * bins + 1], pos [N], key [N], part [nchunks][2][d], each
// rounded to 256 bytes.
// The chunks' length is an order of additions and a size of scratch, so it goes by
// a B200's 148 SMs and not by those that the current device shows.
constexpr int SMS = 148;
struct Layout {
  int chunk, nchunks;
  int64_t start, pos, key, part, bytes;
};
static Layout layout(int N, int V, int d) {
  Layout l{};
  // chunks long enough to amortise a border, short enough for some waves of CTAs
  const int64_t tiles = (d + SUM_NT * 8 - 1) / (SUM_NT * 8);
  l.chunk = (int)std::min<int64_t>(MAX_CHUNK, std::max<int64_t>(32, (int64_t)N * tiles / (SMS * 16)));
  l.nchunks = (N + l.chunk - 1) / l.chunk;
  const auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
  l.start = 0;
  l.pos = up((((int64_t)sort_bins(V) << sort_log2(V)) + 1) * 4);
  l.key = l.pos + up((int64_t)N * 4);
  l.part = l.key + up((int64_t)N * 4);
  // parts: as many as any batch of up to N tokens has (the chunks' length grows
  // with N between 32 and 128, where their number stays near 16 SMS / tiles, at
  // most a 32nd above it), so that a workspace for the largest batch serves the
  // smaller ones
  const int64_t most =
      std::min<int64_t>((N + 31) / 32, std::max<int64_t>(SMS * 16 * 33 / 32 / tiles + 3, (N + 127) / 128));
  l.bytes = l.part + up(std::max<int64_t>(most, l.nchunks) * 2 * d * 4);
  return l;
}

template <typename TI, typename TO, int W>
static int launch_grad(Grad &a, cudaStream_t st) {
  a.col_tiles = (a.d + SUM_NT * W - 1) / (SUM_NT * W);
  const int smem = SORT_NW * a.bins * 4;
  int rc = allow_smem<sort_tokens_kernel>(smem);
  if (rc) return rc;
  const bool fill = a.base != a.out;
  if (fill) {  // (two blocks per SM leave the sort its place beside them)
    const int64_t bytes = (int64_t)a.V * a.d * (int)sizeof(TO);
    const int64_t blocks = (bytes / 16 + FILL_NT * FILL_U - 1) / (FILL_NT * FILL_U);
    fill_kernel<<<(unsigned)std::max<int64_t>(1, std::min<int64_t>(blocks, 2 * sm_count())), FILL_NT, 0, st>>>(
        static_cast<uint8_t *>(a.out), static_cast<const uint8_t *>(a.base), bytes);
    if ((rc = launched())) return rc;
  }
  // the next kernels may be placed while the one before runs; they wait for it before they read
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1u << a.c_log2, 1, 1);
  cfg.blockDim = dim3(SORT_NT, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = fill ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&cfg, sort_tokens_kernel, a);
  const int64_t work = (int64_t)a.nchunks * a.col_tiles;
  cfg.numAttrs = 1;
  cfg.dynamicSmemBytes = 0;
  if (e == cudaSuccess) {
    cfg.gridDim = dim3((unsigned)work, 1, 1);
    cfg.blockDim = dim3(SUM_NT, 1, 1);
    e = cudaLaunchKernelEx(&cfg, sum_tokens_kernel<TI, TO, W>, a);
  }
  if (e == cudaSuccess && a.nchunks > 1) {
    cfg.gridDim = dim3((unsigned)std::min(a.nchunks - 1, sm_count()), (unsigned)a.col_tiles, 1);
    cfg.blockDim = dim3(SUM_NT * JOIN_G, 1, 1);
    e = cudaLaunchKernelEx(&cfg, join_tokens_kernel<TO, W>, a);
  }
  return e == cudaSuccess ? MSTAR_OK : fail(MSTAR_ERR_CUDA, std::string("launch: ") + cudaGetErrorString(e));
}

template <typename TI, typename TO>
static int launch_grad_w(Grad &a, int w, cudaStream_t st) {
  return w == 8   ? launch_grad<TI, TO, 8>(a, st)
         : w == 2 ? launch_grad<TI, TO, 2>(a, st)
                  : launch_grad<TI, TO, 1>(a, st);
}

}  // namespace emb
}  // namespace mstar

using namespace mstar;

extern "C" {

int mstar_embed_tokens(const int64_t *ids, int64_t N, const void *table, int32_t dtype, int32_t V, int32_t d,
                       int64_t ld, float scale, void *out, int32_t out_dtype, uint32_t *status, void *stream) {
  int rc = emb::check_lookup(ids, N, V, d, out, out_dtype);
  if (rc) return rc;
  if (!table) return fail(MSTAR_ERR_INVALID, "table must not be NULL");
  if ((rc = emb::check_dtype(dtype, "dtype"))) return rc;
  if (ld < d) return fail(MSTAR_ERR_INVALID, "ld must be >= d");
  if (reinterpret_cast<uintptr_t>(table) & (emb::es(dtype) - 1))
    return fail(MSTAR_ERR_INVALID, "table must be aligned to its type");
  emb::Lookup a{};
  a.table = table;
  a.ld = ld;
  a.ids = ids;
  a.N = N;
  a.V = V;
  a.d = d;
  a.scale = scale;
  a.out = out;
  a.status = status;
  const int w = emb::width_of(d, std::min(emb::width(table, ld, dtype), emb::width(out, d, out_dtype)));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool fi = dtype == MSTAR_DTYPE_F32, fo = out_dtype == MSTAR_DTYPE_F32;
  if (fi) return fo ? emb::launch_lookup<float, float>(a, w, st) : emb::launch_lookup<float, __nv_bfloat16>(a, w, st);
  return fo ? emb::launch_lookup<__nv_bfloat16, float>(a, w, st)
            : emb::launch_lookup<__nv_bfloat16, __nv_bfloat16>(a, w, st);
}

int mstar_embed_tokens_w4(const int64_t *ids, int64_t N, const mstar_w4_t *w, float scale, void *out,
                          int32_t out_dtype, uint32_t *status, void *stream) {
  int rc = check_w4(w);
  if (rc) return rc;
  if ((rc = emb::check_lookup(ids, N, w->V, w->d, out, out_dtype))) return rc;
  if (reinterpret_cast<uintptr_t>(out) & 15u) return fail(MSTAR_ERR_INVALID, "out must be 16-byte aligned");
  emb::Lookup a{};
  a.ids = ids;
  a.N = N;
  a.V = w->V;
  a.d = w->d;
  a.scale = scale;
  a.out = out;
  a.status = status;
  a.codes = static_cast<const uint8_t *>(w->codes);
  a.scales = w->scales;
  a.zeros = static_cast<const uint8_t *>(w->zeros);
  a.scale_dtype = w->scale_dtype;
  a.group_log2 = w->group == 32 ? 5 : w->group == 64 ? 6 : 7;
  a.ngroups = w->d / w->group;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)((N * (w->d / 8) + emb::NT * 4 - 1) / (emb::NT * 4));
  if (out_dtype == MSTAR_DTYPE_F32)
    emb::embed_w4_kernel<float><<<grid, emb::NT, 0, st>>>(a);
  else
    emb::embed_w4_kernel<__nv_bfloat16><<<grid, emb::NT, 0, st>>>(a);
  return emb::launched();
}

int64_t mstar_embed_grad_workspace_bytes(int32_t N, int32_t V, int32_t d) {
  if (N < 1 || N > (1 << 24) || V < 1 || V > (1 << 21) || d < 1 || d > (1 << 16)) return -1;
  return emb::layout(N, V, d).bytes;
}

int mstar_embed_tokens_grad(const int64_t *ids, int32_t N, const void *dout, int32_t dtype, int64_t ld, int32_t V,
                            int32_t d, float scale, const void *base, void *out, int32_t out_dtype, void *workspace,
                            int64_t workspace_bytes, uint32_t *status, void *stream) {
  if (!ids || !dout || !out || !workspace)
    return fail(MSTAR_ERR_INVALID, "ids, dout, out and workspace must not be NULL");
  if (N < 1 || N > (1 << 24)) return fail(MSTAR_ERR_INVALID, "N must be in [1, 2^24]");
  if (V < 1 || V > (1 << 21)) return fail(MSTAR_ERR_INVALID, "V must be in [1, 2097152]");
  if (d < 1 || d > (1 << 16)) return fail(MSTAR_ERR_INVALID, "d must be in [1, 65536]");
  int rc = emb::check_dtype(dtype, "dtype");
  if (rc || (rc = emb::check_dtype(out_dtype, "out_dtype"))) return rc;
  if (ld < d) return fail(MSTAR_ERR_INVALID, "ld must be >= d");
  if (reinterpret_cast<uintptr_t>(dout) & (emb::es(dtype) - 1))
    return fail(MSTAR_ERR_INVALID, "dout must be aligned to its type");
  if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(base)) & (emb::es(out_dtype) - 1))
    return fail(MSTAR_ERR_INVALID, "base and out must be aligned to their type");
  if (reinterpret_cast<uintptr_t>(workspace) & 255u)
    return fail(MSTAR_ERR_INVALID, "workspace must be 256-byte aligned");
  const emb::Layout l = emb::layout(N, V, d);
  if (workspace_bytes < l.bytes) return fail(MSTAR_ERR_INVALID, "workspace too small");
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  emb::Grad a{};
  a.dout = dout;
  a.ldo = ld;
  a.ids = ids;
  a.N = N;
  a.V = V;
  a.d = d;
  a.scale = scale;
  a.base = base;
  a.out = out;
  a.status = status;
  a.bins = emb::sort_bins(V);
  a.c_log2 = emb::sort_log2(V);
  a.chunk = l.chunk;
  a.nchunks = l.nchunks;
  a.start = reinterpret_cast<int32_t *>(ws + l.start);
  a.pos = reinterpret_cast<int32_t *>(ws + l.pos);
  a.key = reinterpret_cast<int32_t *>(ws + l.key);
  a.part = reinterpret_cast<float *>(ws + l.part);
  int w = std::min(emb::width(dout, ld, dtype), emb::width(out, d, out_dtype));
  if (base) w = std::min(w, emb::width(base, d, out_dtype));
  w = emb::width_of(d, w);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool fi = dtype == MSTAR_DTYPE_F32, fo = out_dtype == MSTAR_DTYPE_F32;
  if (fi)
    return fo ? emb::launch_grad_w<float, float>(a, w, st) : emb::launch_grad_w<float, __nv_bfloat16>(a, w, st);
  return fo ? emb::launch_grad_w<__nv_bfloat16, float>(a, w, st)
            : emb::launch_grad_w<__nv_bfloat16, __nv_bfloat16>(a, w, st);
}

}  // extern "C"
