// Log-probabilities of given token ids and the clipped policy loss, over rows
// of logits as the LM head leaves them; each with its gradient to the logits.
//
//   x = logits / T,  lse = log sum_v exp(x_v),  logp = x_id - lse
//   d logp / d logits_v = (onehot_v - exp(x_v - lse)) / T
//
// One thread-block cluster of S CTAs takes a row; each CTA reads its slice
// once, in 16-byte vectors, keeping per thread a running maximum and a sum
// of exponentials (one pass, no separate search for the maximum), which the
// threads, the warps and (over distributed shared memory) the CTAs join.  The
// policy loss writes the gradient in the same pass: the slice stays in shared
// memory, each thread re-reading only the vectors that it stored itself, so
// the logits are read from memory once and the gradient written once.
//
// Arithmetic: exponents are kept in units of log 2, t = x * c - M with c =
// log2(e) / T rounded to 32 bits and M the (scaled, rounded) running maximum.
// M's rounding cancels, because the same M enters the final logarithm, and
// c's is relative to x - max, so the terms that carry the sum are exact to
// the last bits.  Sums are 32 bits per thread (a few hundred terms), joined
// in a tree; each row's scalars (lse, logp, the ratio and the KL term, which
// are differences of nearby numbers) are computed in 64 bits by one thread.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace mstar {
namespace rows {

constexpr int NT = 256;
constexpr int NW = NT / 32;
constexpr int MAX_S = 8;                  // portable cluster width
constexpr int SLICE_BYTES = 48 * 1024;    // four slices share an SM's shared memory
constexpr int MAX_RESIDENT = 200 * 1024;  // larger slices are read from memory twice
// Values at or below FLOOR count as masked while the running maximum is
// tracked (a mask of the type's lowest value would overflow when scaled by
// c); a row whose largest value is not inside (FLOOR, -FLOOR) takes the
// exact path, which subtracts before it scales.
constexpr float FLOOR = -1e30f;

enum : int { LOGPROBS = 0, POLICY = 1, POLICY_GRAD = 2 };

struct Args {
  const void *logits;
  int64_t ld;
  int32_t N, V, S;
  int32_t slice_vecs;  // vectors of shared memory per CTA (POLICY_GRAD, resident)
  const int64_t *ids;
  float c;             // log2(e) / T
  double inv_t;
  float *logp, *lse, *loss;
  void *dlogits;
  int64_t ldd;
  const float *old_logp, *ref_logp, *adv, *weights;
  double clip_min, clip_max, beta;
  uint32_t *status;
};

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ void unpack(const uint4 &w, float (&x)[4]) {
    x[0] = __uint_as_float(w.x);
    x[1] = __uint_as_float(w.y);
    x[2] = __uint_as_float(w.z);
    x[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int E = 8;
  static __device__ __forceinline__ void unpack(const uint4 &w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);  // the output's own type: one rounding
      u[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row as aligned vectors [0, nv) behind `head` and before `tail` single values.
template <typename T>
struct Row {
  const T *p;
  int head, nv, tail;
  __device__ Row(const T *row, int V) : p(row) {
    const int mis = (int)(reinterpret_cast<uintptr_t>(row) & 15u) / (int)sizeof(T);
    head = mis ? min(V, Vec<T>::E - mis) : 0;
    nv = (V - head) / Vec<T>::E;
    tail = V - head - nv * Vec<T>::E;
  }
  __device__ __forceinline__ const uint4 *vecs() const { return reinterpret_cast<const uint4 *>(p + head); }
};

// Running (maximum, sum) in scaled units: s = sum 2^(x c - M).
struct Stat {
  float m, M, s;  // raw maximum, scaled maximum, sum
  __device__ explicit Stat(float c) : m(FLOOR), M(FLOOR * c), s(0.f) {}
  template <int E>
  __device__ __forceinline__ void add(const float (&x)[E], float c) {
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < E; ++i) mx = fmaxf(mx, x[i]);
    if (mx > m) {
      const float M2 = mx * c;
      s *= ex2(M - M2);
      m = mx;
      M = M2;
    }
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) part += ex2(fmaf(x[i], c, -M));
    s += part;
  }
};

__device__ __forceinline__ void join(float &M, float &s, float M2, float s2) {
  const float Mx = fmaxf(M, M2);
  s = s * ex2(M - Mx) + s2 * ex2(M2 - Mx);
  M = Mx;
}

struct Scalars {
  float M, k, g;  // gradient: 2^(x c - M) * k, plus g at the id (in the exact path M is the raw maximum)
  int exact;
};

struct Sh {
  float2 warp[NW];
  float2 cta[MAX_S];
  Scalars row;
};

// Joins (a, b) over the cluster's threads; every thread of the block gets the
// result.  `phase` picks how: 0 joins (maximum, sum) pairs, 1 takes the
// maximum of a, 2 adds b in a fixed order.
template <int PHASE>
__device__ float2 cluster_join(Sh &sh, int S, int rank, float a, float b) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const float a2 = __shfl_xor_sync(~0u, a, o), b2 = __shfl_xor_sync(~0u, b, o);
    if (PHASE == 0) join(a, b, a2, b2);
    if (PHASE == 1) a = fmaxf(a, a2);
    if (PHASE == 2) b += b2;
  }
  if (PHASE != 0) {  // an earlier join's readers are done
    if (S == 1)
      __syncthreads();
    else
      cg::this_cluster().sync();
  }
  if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  if (threadIdx.x < (unsigned)S) {  // thread j tells CTA j
    float2 t = sh.warp[0];
    for (int w = 1; w < NW; ++w) {
      const float2 u = sh.warp[w];
      if (PHASE == 0) join(t.x, t.y, u.x, u.y);
      if (PHASE == 1) t.x = fmaxf(t.x, u.x);
      if (PHASE == 2) t.y += u.y;
    }
    if (S == 1)
      sh.cta[0] = t;
    else
      *cg::this_cluster().map_shared_rank(&sh.cta[rank], threadIdx.x) = t;
  }
  if (S == 1)
    __syncthreads();
  else
    cg::this_cluster().sync();
  float2 t = sh.cta[0];
  for (int j = 1; j < S; ++j) {
    const float2 u = sh.cta[j];
    if (PHASE == 0) join(t.x, t.y, u.x, u.y);
    if (PHASE == 1) t.x = fmaxf(t.x, u.x);
    if (PHASE == 2) t.y += u.y;
  }
  return t;
}

// The row's scalars in 64 bits, by one thread: xr is the maximum that the
// sum is relative to.  Every CTA of the row computes them; rank 0 writes them.
template <int MODE>
__device__ Scalars scalars(const Args &a, int row, int64_t id, bool ok, double xr, float s, bool empty, float x_id,
                           bool writer) {
  Scalars r{0.f, 0.f, 0.f, 0};
  const double ls = log((double)s);
  const double lse = empty ? -INFINITY : xr * a.inv_t + ls;
  const double lp = !ok ? 0.0 : empty ? -INFINITY : ((double)x_id - xr) * a.inv_t - ls;
  if (writer) {
    a.logp[row] = (float)lp;
    if (a.lse) a.lse[row] = (float)lse;
    const uint32_t bits = (empty ? MSTAR_STATUS_EMPTY : 0u) | (id >= a.V ? MSTAR_STATUS_BAD_ID : 0u);
    if (a.status && bits) atomicOr(a.status, bits);
  }
  if (MODE == LOGPROBS) return r;
  double loss = 0.0, d = 0.0;
  if (ok && !empty) {
    const double A = a.adv[row];
    const double ratio = a.old_logp ? exp(lp - (double)a.old_logp[row]) : isnan(lp) ? lp : 1.0;
    const double plain = ratio * A, cut = fmin(fmax(ratio, a.clip_min), a.clip_max) * A;
    loss = -fmin(plain, cut);
    if (isnan(plain)) loss = plain;
    d = plain <= cut ? -plain : isnan(plain) ? plain : 0.0;
    if (a.ref_logp && a.beta != 0.0) {
      const double q = (double)a.ref_logp[row] - lp, e = expm1(q);
      loss += a.beta * (q == INFINITY ? q : e - q);
      d -= a.beta * e;
    }
    if (lp == -INFINITY) d = 0.0;  // an id of probability zero stays there: no gradient
  }
  if (writer) a.loss[row] = (float)loss;
  const double g = d * (a.weights ? (double)a.weights[row] : 1.0) * a.inv_t;
  r.g = (float)g;
  r.k = empty ? 0.f : (float)(-g / (double)s);
  return r;
}

template <typename T, int MODE, bool RESIDENT>
__global__ void __launch_bounds__(NT) token_rows_kernel(const Args a) {
  constexpr int E = Vec<T>::E;
  constexpr int U = 4;  // vectors in flight per thread
  extern __shared__ __align__(16) uint4 stored[];
  __shared__ Sh sh;
  const int S = a.S, rank = (int)(blockIdx.x % (unsigned)S), row = (int)(blockIdx.x / (unsigned)S);
  const int tid = threadIdx.x;
  const Row<T> in(static_cast<const T *>(a.logits) + (int64_t)row * a.ld, a.V);
  const int v0 = (int)((int64_t)in.nv * rank / S), v1 = (int)((int64_t)in.nv * (rank + 1) / S);
  // the values before and after the aligned vectors: one each to the first threads of the first and last CTA
  const int fringe = rank == 0 && tid < in.head ? tid
                     : rank == S - 1 && tid >= 32 && tid < 32 + in.tail ? in.head + in.nv * E + tid - 32
                                                                       : -1;
  const int64_t id = a.ids[row];
  const bool ok = id >= 0 && id < a.V;
  T *out = MODE == POLICY_GRAD ? static_cast<T *>(a.dlogits) + (int64_t)row * a.ldd : nullptr;
  const bool vec_out = MODE == POLICY_GRAD && (reinterpret_cast<uintptr_t>(out + in.head) & 15u) == 0;
  if (MODE != LOGPROBS && !ok) {  // a padding row: nothing of it is read
    if (rank == 0 && tid == 0) {
      a.loss[row] = 0.f;
      a.logp[row] = 0.f;
      if (a.lse) a.lse[row] = 0.f;
      if (id >= 0 && a.status) atomicOr(a.status, MSTAR_STATUS_BAD_ID);
    }
    if (MODE == POLICY_GRAD) {
      if (fringe >= 0) put(out + fringe, 0.f);
      for (int v = v0 + tid; v < v1; v += NT) {
        T *o = out + in.head + (int64_t)v * E;
        if (vec_out)
          __stcs(reinterpret_cast<uint4 *>(o), make_uint4(0u, 0u, 0u, 0u));
        else
          for (int i = 0; i < E; ++i) put(o + i, 0.f);
      }
    }
    return;
  }
  if (S > 1) cg::this_cluster().sync();  // a CTA writes into a peer's shared memory only once the peer runs
  const float x_id = ok ? to_f(in.p[id]) : 0.f;
  const float x_fringe = fringe >= 0 ? to_f(in.p[fringe]) : 0.f;
  const float c = a.c;
  Stat st(c);
  for (int v = v0 + tid; v < v1; v += NT * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * NT < v1) w[u] = __ldcs(in.vecs() + v + u * NT);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * NT < v1) {
        if (MODE == POLICY_GRAD && RESIDENT) stored[v + u * NT - v0] = w[u];
        float x[E];
        Vec<T>::unpack(w[u], x);
        st.add(x, c);
      }
  }
  if (fringe >= 0) {
    const float x[1] = {x_fringe};
    st.add(x, c);
  }
  float2 t = cluster_join<0>(sh, S, rank, st.M, st.s);
  const bool exact = !(t.x > FLOOR * c && t.x < -FLOOR * c);
  bool empty = false;
  auto load = [&](int v) {
    return MODE == POLICY_GRAD && RESIDENT ? stored[v - v0] : in.vecs()[v];
  };
  if (exact) {  // the row's largest value is at the edge of the type (or nothing is left of it)
    float m = fringe >= 0 ? x_fringe : -INFINITY;
    for (int v = v0 + tid; v < v1; v += NT) {
      float x[E];
      Vec<T>::unpack(load(v), x);
#pragma unroll
      for (int i = 0; i < E; ++i) m = fmaxf(m, x[i]);
    }
    m = cluster_join<1>(sh, S, rank, m, 0.f).x;
    float s = fringe >= 0 ? ex2((x_fringe - m) * c) : 0.f;
    for (int v = v0 + tid; v < v1; v += NT) {
      float x[E];
      Vec<T>::unpack(load(v), x);
#pragma unroll
      for (int i = 0; i < E; ++i) s += ex2((x[i] - m) * c);
    }
    t = make_float2(m, cluster_join<2>(sh, S, rank, 0.f, s).y);
    empty = m == -INFINITY;
  }
  if (tid == 0) {
    const double xr = exact ? (double)t.x : (double)t.x / (double)c;
    Scalars r = scalars<MODE>(a, row, id, ok, xr, t.y, empty, x_id, rank == 0);
    r.M = t.x;
    r.exact = exact;
    sh.row = r;
  }
  if (MODE != POLICY_GRAD) return;
  __syncthreads();
  const Scalars r = sh.row;
  auto grad = [&](float x, int at) {
    // (an empty row, or a row whose loss does not move with it: zeros, whatever its logits hold)
    float y = r.k == 0.f ? 0.f : ex2(r.exact ? (x - r.M) * c : fmaf(x, c, -r.M)) * r.k;
    return at == (int)id ? y + r.g : y;
  };
  if (fringe >= 0) put(out + fringe, grad(x_fringe, fringe));
  for (int v = v0 + tid; v < v1; v += NT) {
    float x[E], y[E];
    Vec<T>::unpack(load(v), x);
    const int at = in.head + v * E;
#pragma unroll
    for (int i = 0; i < E; ++i) y[i] = grad(x[i], at + i);
    if (vec_out)
      __stcs(reinterpret_cast<uint4 *>(out + at), Vec<T>::pack(y));
    else
#pragma unroll
      for (int i = 0; i < E; ++i) put(out + at + i, y[i]);
  }
}

struct GradArgs {
  const void *logits;
  int64_t ld;
  int32_t N, V, S;
  const int64_t *ids;
  float c;
  double inv_t;
  const float *lse, *dlogp;
  void *dlogits;
  int64_t ldd;
};

// dlogits = dlogp / T * (onehot - 2^(x c - lse T c)): lse enters through its
// own reference point lse * T, so c's rounding is relative to x - lse * T, and
// the part of lse T c that 32 bits lose goes into the row's factor.
template <typename T>
__global__ void __launch_bounds__(NT) token_logprobs_grad_kernel(const GradArgs a) {
  constexpr int E = Vec<T>::E;
  constexpr int U = 4;
  __shared__ float sM, sk, sg;
  const int S = a.S, rank = (int)(blockIdx.x % (unsigned)S), row = (int)(blockIdx.x / (unsigned)S);
  const int tid = threadIdx.x;
  const Row<T> in(static_cast<const T *>(a.logits) + (int64_t)row * a.ld, a.V);
  T *out = static_cast<T *>(a.dlogits) + (int64_t)row * a.ldd;
  const bool vec_out = (reinterpret_cast<uintptr_t>(out + in.head) & 15u) == 0;
  const int v0 = (int)((int64_t)in.nv * rank / S), v1 = (int)((int64_t)in.nv * (rank + 1) / S);
  const int fringe = rank == 0 && tid < in.head ? tid
                     : rank == S - 1 && tid >= 32 && tid < 32 + in.tail ? in.head + in.nv * E + tid - 32
                                                                       : -1;
  const int64_t id = a.ids[row];
  if (tid == 0) {
    const bool ok = id >= 0 && id < a.V && a.lse[row] != -INFINITY;
    const double g = ok ? (double)a.dlogp[row] * a.inv_t : 0.0;
    const double M = (double)a.lse[row] / a.inv_t * (double)a.c;
    sM = (float)M;
    sg = (float)g;
    sk = (float)(-g * exp2((double)(float)M - M));
    if (!ok) sM = 0.f, sk = 0.f;
  }
  __syncthreads();
  const float M = sM, k = sk, g = sg, c = a.c;
  auto grad = [&](float x, int at) {
    const float y = k == 0.f ? 0.f : ex2(fmaf(x, c, -M)) * k;
    return at == (int)id ? y + g : y;
  };
  if (fringe >= 0) put(out + fringe, grad(to_f(in.p[fringe]), fringe));
  for (int v = v0 + tid; v < v1; v += NT * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * NT < v1) w[u] = __ldcs(in.vecs() + v + u * NT);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * NT < v1) {
        float x[E], y[E];
        Vec<T>::unpack(w[u], x);
        const int at = in.head + (v + u * NT) * E;
#pragma unroll
        for (int i = 0; i < E; ++i) y[i] = grad(x[i], at + i);
        if (vec_out)
          __stcs(reinterpret_cast<uint4 *>(out + at), Vec<T>::pack(y));
        else
#pragma unroll
          for (int i = 0; i < E; ++i) put(out + at + i, y[i]);
      }
  }
}

// ------------------------------------------------------------ host side

// CTAs per row: slices of at most SLICE_BYTES, and narrower ones (down to
// 8 KB) while the rows alone leave SMs idle.
static int slices(int N, int64_t row_bytes) {
  int S = 1;
  while (S < MAX_S && row_bytes > (int64_t)S * SLICE_BYTES) S *= 2;
  while (S < MAX_S && (int64_t)N * S < 2 * sm_count() && row_bytes > (int64_t)S * 8192) S *= 2;
  return S;
}

static int check_rows(const void *logits, int dtype, int N, int V, int64_t ld, const int64_t *ids, double temperature) {
  if (!logits || !ids) return fail(MSTAR_ERR_INVALID, "logits and ids must not be NULL");
  if (dtype != MSTAR_DTYPE_F32 && dtype != MSTAR_DTYPE_BF16)
    return fail(MSTAR_ERR_INVALID, "dtype must be MSTAR_DTYPE_F32 or MSTAR_DTYPE_BF16");
  if (N < 1 || N > (1 << 24)) return fail(MSTAR_ERR_INVALID, "N must be in [1, 2^24]");
  if (V < 1 || V > (1 << 21)) return fail(MSTAR_ERR_INVALID, "V must be in [1, 2097152]");
  if (ld < V) return fail(MSTAR_ERR_INVALID, "ld must be >= V");
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == MSTAR_DTYPE_F32 ? 3u : 1u))
    return fail(MSTAR_ERR_INVALID, "logits must be aligned to their type");
  if (!(temperature >= 1e-5 && temperature <= 1e5))
    return fail(MSTAR_ERR_INVALID, "temperature must be in [1e-5, 1e5]");
  return MSTAR_OK;
}

static int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? MSTAR_OK : fail(MSTAR_ERR_CUDA, std::string("launch: ") + cudaGetErrorString(e));
}

template <typename T, int MODE, bool RESIDENT>
static int launch(const Args &a, int smem, cudaStream_t st) {
  auto kern = token_rows_kernel<T, MODE, RESIDENT>;
  if (smem > 48 * 1024 - (int)sizeof(Sh)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(MSTAR_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.N * (unsigned)a.S, 1, 1);
  cfg.blockDim = dim3(NT, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) return fail(MSTAR_ERR_CUDA, std::string("launch: ") + cudaGetErrorString(e));
  return MSTAR_OK;
}

template <typename T>
static int run(Args &a, int mode, cudaStream_t st) {
  a.S = slices(a.N, (int64_t)a.V * (int)sizeof(T));
  if (mode == LOGPROBS) return launch<T, LOGPROBS, false>(a, 0, st);
  if (mode == POLICY) return launch<T, POLICY, false>(a, 0, st);
  const int64_t vecs = ((int64_t)a.V / Vec<T>::E + a.S - 1) / a.S;
  if (vecs * 16 <= MAX_RESIDENT) return launch<T, POLICY_GRAD, true>(a, (int)vecs * 16, st);
  return launch<T, POLICY_GRAD, false>(a, 0, st);
}

static void set_temperature(double temperature, float &c, double &inv_t) {
  inv_t = 1.0 / temperature;
  c = (float)(1.4426950408889634074 * inv_t);
}

}  // namespace rows
}  // namespace mstar

using namespace mstar;

extern "C" {

int mstar_token_logprobs(const void *logits, int32_t dtype, int32_t N, int32_t V, int64_t ld, const int64_t *ids,
                         double temperature, float *logp, float *lse, uint32_t *status, void *stream) {
  int rc = rows::check_rows(logits, dtype, N, V, ld, ids, temperature);
  if (rc) return rc;
  if (!logp) return fail(MSTAR_ERR_INVALID, "logp must not be NULL");
  rows::Args a{};
  a.logits = logits;
  a.ld = ld;
  a.N = N;
  a.V = V;
  a.ids = ids;
  rows::set_temperature(temperature, a.c, a.inv_t);
  a.logp = logp;
  a.lse = lse;
  a.status = status;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == MSTAR_DTYPE_F32 ? rows::run<float>(a, rows::LOGPROBS, st)
                                  : rows::run<__nv_bfloat16>(a, rows::LOGPROBS, st);
}

int mstar_token_logprobs_grad(const void *logits, int32_t dtype, int32_t N, int32_t V, int64_t ld, const int64_t *ids,
                              double temperature, const float *lse, const float *dlogp, void *dlogits,
                              int64_t ld_dlogits, void *stream) {
  int rc = rows::check_rows(logits, dtype, N, V, ld, ids, temperature);
  if (rc) return rc;
  if (!lse || !dlogp || !dlogits) return fail(MSTAR_ERR_INVALID, "lse, dlogp and dlogits must not be NULL");
  if (ld_dlogits < V) return fail(MSTAR_ERR_INVALID, "ld_dlogits must be >= V");
  if (reinterpret_cast<uintptr_t>(dlogits) & (dtype == MSTAR_DTYPE_F32 ? 3u : 1u))
    return fail(MSTAR_ERR_INVALID, "dlogits must be aligned to their type");
  rows::GradArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.N = N;
  a.V = V;
  a.ids = ids;
  rows::set_temperature(temperature, a.c, a.inv_t);
  a.lse = lse;
  a.dlogp = dlogp;
  a.dlogits = dlogits;
  a.ldd = ld_dlogits;
  const int es = dtype == MSTAR_DTYPE_F32 ? 4 : 2;
  const int64_t per = (int64_t)rows::NT * 4 * 16;  // one unrolled step of a block
  a.S = (int)std::max<int64_t>(1, ((int64_t)V * es + per - 1) / per);
  while (a.S > 1 && (int64_t)N * a.S > 0x7FFFFFFF) a.S = (a.S + 1) / 2;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == MSTAR_DTYPE_F32)
    rows::token_logprobs_grad_kernel<float><<<(unsigned)N * (unsigned)a.S, rows::NT, 0, st>>>(a);
  else
    rows::token_logprobs_grad_kernel<__nv_bfloat16><<<(unsigned)N * (unsigned)a.S, rows::NT, 0, st>>>(a);
  return rows::launched();
}

int mstar_policy_loss(const mstar_policy_params_t *p, void *stream) {
  if (!p) return fail(MSTAR_ERR_INVALID, "params is NULL");
  int rc = rows::check_rows(p->logits, p->dtype, p->N, p->V, p->ld, p->ids, p->temperature);
  if (rc) return rc;
  if (!p->advantages || !p->loss || !p->logp)
    return fail(MSTAR_ERR_INVALID, "advantages, loss and logp must not be NULL");
  if (!(p->clip_low >= 0.0 && p->clip_low <= 1.0) || !(p->clip_high >= 0.0))
    return fail(MSTAR_ERR_INVALID, "clip_low must be in [0, 1] and clip_high >= 0");
  if (!(p->kl_coef >= 0.0 && p->kl_coef <= 1e300)) return fail(MSTAR_ERR_INVALID, "kl_coef must be >= 0");
  if (p->kl_coef > 0.0 && !p->ref_logp) return fail(MSTAR_ERR_INVALID, "kl_coef needs ref_logp");
  if (p->dlogits && p->ld_dlogits < p->V) return fail(MSTAR_ERR_INVALID, "ld_dlogits must be >= V");
  if (reinterpret_cast<uintptr_t>(p->dlogits) & (p->dtype == MSTAR_DTYPE_F32 ? 3u : 1u))
    return fail(MSTAR_ERR_INVALID, "dlogits must be aligned to their type");
  rows::Args a{};
  a.logits = p->logits;
  a.ld = p->ld;
  a.N = p->N;
  a.V = p->V;
  a.ids = p->ids;
  rows::set_temperature(p->temperature, a.c, a.inv_t);
  a.logp = p->logp;
  a.lse = p->lse;
  a.loss = p->loss;
  a.dlogits = p->dlogits;
  a.ldd = p->ld_dlogits;
  a.old_logp = p->old_logp;
  a.ref_logp = p->ref_logp;
  a.adv = p->advantages;
  a.weights = p->weights;
  a.clip_min = 1.0 - p->clip_low;
  a.clip_max = 1.0 + p->clip_high;
  a.beta = p->kl_coef;
  a.status = p->status;
  const int mode = p->dlogits ? rows::POLICY_GRAD : rows::POLICY;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return p->dtype == MSTAR_DTYPE_F32 ? rows::run<float>(a, mode, st) : rows::run<__nv_bfloat16>(a, mode, st);
}

}  // extern "C"
