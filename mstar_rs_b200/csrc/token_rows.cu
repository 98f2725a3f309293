// Log-probabilities of given token ids and the clipped policy loss, over rows
// of logits as the LM head leaves them; each with its gradient to the logits.
//
//   x = logits / T,  lse = log sum_v exp(x_v),  logp = x_id - lse
//   d logp / d logits_v = (onehot_v - exp(x_v - lse)) / T
//
// One thread-block cluster of S CTAs takes a row; each CTA passes once over its
// slice, in 16-byte vectors, keeping per thread a running maximum and a sum
// of exponentials (no separate search for the maximum), which the threads,
// the warps and (over distributed shared memory) the CTAs join.  The policy
// loss writes the gradient in the same launch and reads the slice again for
// it, from L2: the rows in flight (148 SMs x 6 CTAs x 76 KB of 151936 bf16)
// fit there, so memory sees each logit once.  Keeping the slice in shared
// memory instead left room for too few CTAs to cover the joins (577 against
// 470 us for 4096 such rows).
//
// What bounds it: memory (4 bytes per bf16 logit, read and written: 380 us for
// 4096 x 151936 at 6553 GB/s), and close behind it the special-function unit
// (two exponentials per logit at 16 a cycle and SM: 328 us).
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
#include <cfloat>
#include <cmath>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace mstar {
namespace rows {

constexpr int NT = 256;
constexpr int NW = NT / 32;
constexpr int MAX_S = 8;                  // portable cluster width
constexpr int SLICE_BYTES = 80 * 1024;  // of a row per CTA, where there are rows enough
// Terms carry the rounding of the scaled maximum M, at most 2^5 below EDGE = 2^30,
// but from 2^32 on it leaves the exponent's range.  So a row whose M is not inside
// (-EDGE, EDGE) takes the exact path, which subtracts before it scales (a row whose
// every id is masked by -1e10), and a running maximum starts at -EDGE and not below
// it: a thread may meet masked ids alone before the first other one, and a sum that
// has left the range does not come back when the maximum rises.  Beside -EDGE,
// which is exact, a masked id's term is 1 at most.
constexpr float EDGE = 0x1p30f;

enum : int { LOGPROBS = 0, POLICY = 1, POLICY_GRAD = 2 };

struct Args {
  const void *logits;
  int64_t ld;
  int32_t N, V, S;
  const int64_t *ids;
  float c;             // log2(e) / T
  float floor;         // -EDGE / c
  double inv_t;
  float *logp, *lse, *loss;
  void *dlogits;
  int64_t ldd;
  const float *old_logp, *ref_logp, *adv, *weights;
  double clip_min, clip_max, beta;
  uint32_t *status;
};

// A 16-byte vector as floats, its largest value, and back.
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
  static __device__ __forceinline__ float largest(const uint4 &w) {
    return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
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
  static __device__ __forceinline__ float largest(const uint4 &w) {
    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&w);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
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

// Calls f(i) for i = first, first + NT, ... below `end`, with the vectors of
// U of them loaded before any is used: f gets the index and the vector.
template <int U, typename Load, typename F>
__device__ __forceinline__ void each_vector(int first, int end, Load load, F f) {
  int v = first;
  for (; v + (U - 1) * NT < end; v += U * NT) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = load(v + u * NT);
#pragma unroll
    for (int u = 0; u < U; ++u) f(v + u * NT, w[u]);
  }
  if (v < end) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (v + u * NT < end) w[u] = load(v + u * NT);
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (v + u * NT < end) f(v + u * NT, w[u]);
  }
}

// Running (maximum, sum) in scaled units: s = sum 2^(x c - M), in two halves.
struct Stat {
  float m, M, s0, s1;  // raw maximum, scaled maximum, sums
  __device__ explicit Stat(float floor) : m(floor), M(-EDGE), s0(0.f), s1(0.f) {}
  __device__ __forceinline__ void raise(float mx, float c) {
    if (mx > m) {
      const float M2 = mx * c, f = ex2(M - M2);
      s0 *= f;
      s1 *= f;
      m = mx;
      M = M2;
    }
  }
  template <typename T>
  __device__ __forceinline__ void add(const uint4 &w, float c) {
    raise(Vec<T>::largest(w), c);
    float x[Vec<T>::E];
    Vec<T>::unpack(w, x);
#pragma unroll
    for (int i = 0; i < Vec<T>::E; i += 2) {
      s0 += ex2(fmaf(x[i], c, -M));
      s1 += ex2(fmaf(x[i + 1], c, -M));
    }
  }
  __device__ __forceinline__ void add_one(float x, float c) {
    raise(x, c);
    s0 += ex2(fmaf(x, c, -M));
  }
};

struct Scalars {
  float M, k, g;  // gradient: 2^(x c - M) * k, plus g at the id (in the exact path M is the raw maximum)
  int exact;
};

struct Sh {
  float2 warp[NW];
  float2 cta[MAX_S];
  Scalars row;
};

// The largest of a warp's values, none of them NaN.
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
  return x;
}
// (M, s) pairs of a warp as one: the largest M, and the sums relative to it.
__device__ __forceinline__ void warp_join(float &M, float &s) {
  const float top = warp_max(M);
  s = warp_sum(s * ex2(M - top));
  M = top;
}

// Joins (a, b) over the cluster: KIND 0 joins (maximum, sum) pairs, 1 takes
// the maximum of a, 2 adds b.  Only warp 0 of each CTA gets the result
// (every lane of it).  `first`: no join of this cluster came before.
template <int KIND>
__device__ __forceinline__ float2 cluster_join(Sh &sh, int S, int rank, float a, float b, bool first) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (KIND == 0) warp_join(a, b);
  if (KIND == 1) a = warp_max(a);
  if (KIND == 2) b = warp_sum(b);
  if (!first) {  // an earlier join's readers are done
    if (S == 1)
      __syncthreads();
    else
      cg::this_cluster().sync();
  }
  if (lane == 0) sh.warp[warp] = make_float2(a, b);
  __syncthreads();
  if (warp == 0) {
    const float2 t = sh.warp[lane & (NW - 1)];  // (each warp's pair on four lanes)
    a = t.x, b = lane < NW ? t.y : 0.f;
    if (KIND == 0) warp_join(a, b);
    if (KIND == 1) a = warp_max(a);
    if (KIND == 2) b = warp_sum(b);
    if (S > 1) {
      if (first) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
      if (lane < S) *cg::this_cluster().map_shared_rank(&sh.cta[rank], lane) = make_float2(a, b);
    }
  } else if (S > 1 && first) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  }
  if (S > 1) {
    cg::this_cluster().sync();
    if (warp == 0) {
      const float2 t = sh.cta[lane & (S - 1)];
      a = t.x, b = lane < S ? t.y : 0.f;
      if (KIND == 0) warp_join(a, b);
      if (KIND == 1) a = warp_max(a);
      if (KIND == 2) b = warp_sum(b);
    }
  }
  return make_float2(a, b);
}

// What a row's loss takes besides its logits, read before the pass over them.
struct Token {
  float x, old_logp, ref_logp, adv, weight;
  template <int MODE>
  static __device__ __forceinline__ Token read(const Args &a, int row, float x_id) {
    Token t{x_id, 0.f, 0.f, 0.f, 1.f};
    if (MODE != LOGPROBS) {
      t.adv = a.adv[row];
      if (a.old_logp) t.old_logp = a.old_logp[row];
      if (a.ref_logp) t.ref_logp = a.ref_logp[row];
      if (a.weights) t.weight = a.weights[row];
    }
    return t;
  }
};

// lse as a float: -infinity stands for an empty row, so what 32 bits cannot
// hold (the lowest value over a T below 1) becomes their largest or lowest.
__device__ __forceinline__ float finite(double lse) {
  return fabs(lse) > (double)FLT_MAX ? (float)copysign((double)FLT_MAX, lse) : (float)lse;
}

// The row's scalars in 64 bits, by a whole warp (its lanes hold the same
// values; the ratio and the KL term take a lane each): xr is the maximum
// that the sum s is relative to.  Every CTA of the row computes them; one
// writes them.
template <int MODE>
__device__ __forceinline__ Scalars scalars(const Args &a, int row, int64_t id, bool ok, double xr, float s, bool empty,
                                           const Token &tok, bool writer) {
  Scalars r{0.f, 0.f, 0.f, 0};
  const int lane = threadIdx.x & 31;
  const double ls = log((double)s);
  const double lse = empty ? -INFINITY : xr * a.inv_t + ls;
  const double lp = !ok ? 0.0 : empty ? -INFINITY : ((double)tok.x - xr) * a.inv_t - ls;
  writer = writer && lane == 0;
  if (writer) {
    a.logp[row] = (float)lp;
    if (a.lse) a.lse[row] = empty ? -INFINITY : finite(lse);
    const uint32_t bits = (empty ? MSTAR_STATUS_EMPTY : 0u) | (id >= a.V ? MSTAR_STATUS_BAD_ID : 0u);
    if (a.status && bits) atomicOr(a.status, bits);
  }
  if (MODE == LOGPROBS) return r;
  // lane 0: exp(logp - old) - 1, lane 1: exp(ref - logp) - 1
  const double q = lane == 1       ? (double)tok.ref_logp - lp
                   : a.old_logp ? lp - (double)tok.old_logp
                   : isnan(lp)  ? lp
                                : 0.0;
  const double e = expm1(q);
  const double ratio = 1.0 + __shfl_sync(~0u, e, 0), eq = __shfl_sync(~0u, e, 1), qq = __shfl_sync(~0u, q, 1);
  double loss = 0.0, d = 0.0;
  if (ok && !empty) {
    const double A = tok.adv;
    const double plain = ratio * A, cut = fmin(fmax(ratio, a.clip_min), a.clip_max) * A;
    loss = -fmin(plain, cut);
    if (isnan(plain)) loss = plain;
    d = plain <= cut ? -plain : isnan(plain) ? plain : 0.0;
    if (a.ref_logp && a.beta != 0.0) {
      loss += a.beta * (qq == INFINITY ? qq : eq - qq);
      d -= a.beta * eq;
    }
    if (lp == -INFINITY) d = 0.0;  // an id of probability zero stays there: no gradient
  }
  if (writer) a.loss[row] = (float)loss;
  const double g = d * (double)tok.weight * a.inv_t;
  r.g = (float)g;
  r.k = empty ? 0.f : -r.g / s;
  return r;
}

// A vector of the gradient, at its place; without 16-byte alignment value by value.
template <typename T>
__device__ __forceinline__ void store(T *o, bool vec_out, const float (&x)[Vec<T>::E]) {
  if (vec_out) {
    __stcs(reinterpret_cast<uint4 *>(o), Vec<T>::pack(x));
  } else {
#pragma unroll
    for (int i = 0; i < Vec<T>::E; ++i) put(o + i, x[i]);
  }
}

// 2^(x c - M) * k over a slice; with `exact`, 2^((x - M) c) * k.  k = 0 (an
// empty row, or one whose loss does not move with it): zeros, whatever it holds.
template <typename T, typename Load>
__device__ __forceinline__ void write_grad(const Row<T> &in, T *out, bool vec_out, int v0, int v1, int fringe,
                                           float x_fringe, float c, float M, float k, bool exact, Load load) {
  constexpr int E = Vec<T>::E;
  constexpr int UW = 4;  // vectors in flight per thread
  T *o = out + in.head;
  const int first = v0 + (int)threadIdx.x;
  if (k == 0.f) {
    if (fringe >= 0) put(out + fringe, 0.f);
    const float zero[E] = {};
    for (int v = first; v < v1; v += NT) store<T>(o + v * E, vec_out, zero);
  } else if (!exact) {
    if (fringe >= 0) put(out + fringe, ex2(fmaf(x_fringe, c, -M)) * k);
    each_vector<UW>(first, v1, load, [&](int v, const uint4 &w) {
      float x[E];
      Vec<T>::unpack(w, x);
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = ex2(fmaf(x[i], c, -M)) * k;
      store<T>(o + v * E, vec_out, x);
    });
  } else {
    if (fringe >= 0) put(out + fringe, ex2((x_fringe - M) * c) * k);
    for (int v = first; v < v1; v += NT) {
      float x[E];
      Vec<T>::unpack(load(v), x);
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = ex2((x[i] - M) * c) * k;
      store<T>(o + v * E, vec_out, x);
    }
  }
}

// (six blocks per SM: 40 registers; without the bound 60, four blocks and 506 in
// place of 470 us for 4096 rows of 151936 bf16)
template <typename T, int MODE>
__global__ void __launch_bounds__(NT, 6) token_rows_kernel(const Args a) {
  constexpr int E = Vec<T>::E;
  constexpr int U = 6;  // vectors in flight per thread
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
  // a CTA writes into a peer's shared memory only once the peer runs: every
  // CTA arrives here, and waits before it writes
  if (S > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const float x_id = ok ? to_f(in.p[id]) : 0.f;
  Token tok{};
  if (tid < 32) tok = Token::read<MODE>(a, row, x_id);
  const float x_fringe = fringe >= 0 ? to_f(in.p[fringe]) : 0.f;
  const float c = a.c;
  Stat st(a.floor);
  // (a gradient reads the slice again, from L2: the rows in flight are some
  // tens of megabytes; otherwise it is read once)
  each_vector<U>(
      v0 + tid, v1, [&](int v) { return MODE == POLICY_GRAD ? in.vecs()[v] : __ldcs(in.vecs() + v); },
      [&](int, const uint4 &w) { st.add<T>(w, c); });
  if (fringe >= 0) st.add_one(x_fringe, c);
  float2 t = cluster_join<0>(sh, S, rank, st.M, st.s0 + st.s1, true);
  if (tid < 32) {
    Scalars r{};
    const bool exact = !(t.x > -EDGE && t.x < EDGE);
    if (!exact) r = scalars<MODE>(a, row, id, ok, (double)t.x / (double)c, t.y, false, tok, rank == 0);
    r.M = t.x;
    r.exact = exact;
    if (tid == 0) sh.row = r;
  }
  __syncthreads();
  auto load = [&](int v) { return __ldcs(in.vecs() + v); };
  if (sh.row.exact) {  // the row's largest value is at the edge of the type (or nothing is left of it)
    // A maximum passes over NaN: a row of -inf alone and one of NaN and -inf both
    // have -inf.  The sum tells them apart (0 and NaN; warp 0 holds it).
    const bool nan = isnan(t.y);
    float m = fringe >= 0 ? x_fringe : -INFINITY;
    for (int v = v0 + tid; v < v1; v += NT) m = fmaxf(m, Vec<T>::largest(load(v)));
    m = cluster_join<1>(sh, S, rank, m, 0.f, false).x;
    if (tid == 0) sh.row.M = m;
    __syncthreads();
    m = sh.row.M;
    float s = fringe >= 0 ? ex2((x_fringe - m) * c) : 0.f;
    for (int v = v0 + tid; v < v1; v += NT) {
      float x[E];
      Vec<T>::unpack(load(v), x);
#pragma unroll
      for (int i = 0; i < E; ++i) s += ex2((x[i] - m) * c);
    }
    t = cluster_join<2>(sh, S, rank, 0.f, s, false);
    if (tid < 32) {
      Scalars r = scalars<MODE>(a, row, id, ok, (double)m, t.y, m == -INFINITY && !nan, tok, rank == 0);
      r.M = m;
      r.exact = 1;
      if (tid == 0) sh.row = r;
    }
    __syncthreads();
  }
  if (MODE != POLICY_GRAD) return;
  const Scalars r = sh.row;
  write_grad<T>(in, out, vec_out, v0, v1, fringe, x_fringe, c, r.M, r.k, r.exact, load);
  // the id's own element: its probability's share, plus g
  const int own = (int)id - in.head;
  const bool mine = own < 0 ? rank == 0 : own >= in.nv * E ? rank == S - 1 : own >= v0 * E && own < v1 * E;
  if (!mine) return;
  __syncthreads();  // the element is written once more, after whoever wrote it
  if (tid == 0) {
    const float p = r.k == 0.f ? 0.f : ex2(r.exact ? (x_id - r.M) * c : fmaf(x_id, c, -r.M)) * r.k;
    put(out + id, p + r.g);
  }
}

struct GradArgs {
  const void *logits;
  int64_t ld;
  int32_t N, V, S;
  const int64_t *ids;
  float c;
  double inv_t, tc;  // 1 / T; T times the rounded c
  const float *lse, *dlogp;
  void *dlogits;
  int64_t ldd;
};

// A row whose |lse| is at least FAR (every id under a finite mask, or a small T):
// 32 bits hold an lse to 2^-24 of itself, an error that every probability of the
// row takes over (from 2^24 on not even log V is left).  So one block sums such a
// row anew.  The sum's own lse counts where the given one is a rounding of it;
// another (of a row that is part of a longer one) is taken as given.  The first
// pass ends before the second writes: dlogits may be logits.  Below FAR the error
// is at most 2^-16 in f32, as the sums' own, and 2^-9 in bf16, half of its
// rounding.  1000 rows of 32001 f32 take 67 us where all are summed anew and 43
// where none is (bf16: 36 and 26).
template <typename T>
constexpr float FAR = sizeof(T) == 4 ? 256.f : 32768.f;

template <typename T>
__device__ __noinline__ void far_row_grad(const T *row, T *out, int V, int id, float c, double inv_t, float lse,
                                          float g) {
  constexpr int E = Vec<T>::E;
  constexpr int U = 4;  // vectors in flight per thread
  __shared__ float2 part[NW];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Row<T> in(row, V);
  const bool vec_out = (reinterpret_cast<uintptr_t>(out + in.head) & 15u) == 0;
  const int fringe = tid < in.head ? tid : tid >= 32 && tid < 32 + in.tail ? in.head + in.nv * E + tid - 32 : -1;
  const auto load = [&](int v) { return in.vecs()[v]; };
  // the running maximum starts at the lowest value: masked ids give 0 beside it
  float m = -FLT_MAX, s = 0.f;
  const float x_fringe = fringe >= 0 ? to_f(row[fringe]) : -INFINITY;
  each_vector<U>(tid, in.nv, load, [&](int, const uint4 &w) {
    const float top = Vec<T>::largest(w);
    if (top > m) {
      s *= ex2((m - top) * c);
      m = top;
    }
    float x[E];
    Vec<T>::unpack(w, x);
#pragma unroll
    for (int i = 0; i < E; ++i) s += ex2((x[i] - m) * c);
  });
  const float own_m = m;
  m = warp_max(fmaxf(m, x_fringe));
  s = warp_sum(s * ex2((own_m - m) * c) + ex2((x_fringe - m) * c));
  if (lane == 0) part[warp] = make_float2(m, s);
  __syncthreads();
  const float2 t = part[lane & (NW - 1)];  // (each warp's pair on four lanes)
  m = warp_max(t.x);
  s = warp_sum(lane < NW ? t.y * ex2((t.x - m) * c) : 0.f);
  const double own = (double)m * inv_t + log((double)s), given = lse;
  // -g exp(x / T - lse) = k 2^((x - m) c)
  const bool same = fabs((double)finite(own) - given) <= fabs(given) * 0x1p-23;
  const float k = same ? -g / s : (float)(-(double)g * exp((double)m * inv_t - given));
  const auto share = [&](float x) {
    const float p = ex2((x - m) * c);
    return p == 0.f ? 0.f : p * k;
  };
  if (fringe >= 0) put(out + fringe, share(x_fringe) + (fringe == id ? g : 0.f));
  T *o = out + in.head;
  each_vector<U>(tid, in.nv, load, [&](int v, const uint4 &w) {
    float x[E];
    Vec<T>::unpack(w, x);
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = share(x[i]) + (in.head + v * E + i == id ? g : 0.f);
    store<T>(o + v * E, vec_out, x);
  });
}

// dlogits = dlogp / T * (onehot - 2^(x c - lse T c)): lse enters through its
// own reference point lse * T, so c's rounding is relative to x - lse * T, and
// the part of lse T c that 32 bits lose goes into the row's factor.
template <typename T>
__global__ void __launch_bounds__(NT) token_logprobs_grad_kernel(const GradArgs a) {
  constexpr int E = Vec<T>::E;
  constexpr int U = 4;  // vectors in flight per thread
  __shared__ float sM, sk, sg;
  __shared__ bool far;
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
    const float lse = a.lse[row];
    const bool ok = id >= 0 && id < a.V && lse != -INFINITY;
    const float g = ok ? (float)((double)a.dlogp[row] * a.inv_t) : 0.f;
    const double M = (double)lse * a.tc;
    sM = ok ? (float)M : 0.f;
    sg = g;
    sk = ok ? -g * ex2((float)((double)(float)M - M)) : 0.f;
    far = ok && fabsf(lse) >= FAR<T> && fabsf(lse) < INFINITY;
  }
  __syncthreads();
  if (far) {
    if (rank == 0) far_row_grad<T>(in.p, out, a.V, (int)id, a.c, a.inv_t, a.lse[row], sg);
    return;
  }
  const float M = sM, k = sk, g = sg, c = a.c;
  if (fringe >= 0) {
    const float x = to_f(in.p[fringe]);
    put(out + fringe, (k == 0.f ? 0.f : ex2(fmaf(x, c, -M)) * k) + (fringe == id ? g : 0.f));
  }
  const int64_t own = id - in.head;  // where the id lies among the vectors' values
  const int own_vec = own >= 0 && own < (int64_t)in.nv * E ? (int)(own / E) : -1;
  T *o = out + in.head;
  each_vector<U>(
      v0 + tid, v1, [&](int v) { return __ldcs(in.vecs() + v); },
      [&](int v, const uint4 &w) {
        float x[E];
        Vec<T>::unpack(w, x);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = ex2(fmaf(x[i], c, -M)) * k;
        if (k == 0.f) {
#pragma unroll
          for (int i = 0; i < E; ++i) x[i] = 0.f;
        }
        if (v == own_vec) {
#pragma unroll
          for (int i = 0; i < E; ++i) x[i] += own == (int64_t)v * E + i ? g : 0.f;
        }
        store<T>(o + v * E, vec_out, x);
      });
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

template <typename T, int MODE>
static int launch(const Args &a, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.N * (unsigned)a.S, 1, 1);
  cfg.blockDim = dim3(NT, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.S;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, token_rows_kernel<T, MODE>, a);
  if (e != cudaSuccess) return fail(MSTAR_ERR_CUDA, std::string("launch: ") + cudaGetErrorString(e));
  return MSTAR_OK;
}

template <typename T>
static int run(Args &a, int mode, cudaStream_t st) {
  a.S = slices(a.N, (int64_t)a.V * (int)sizeof(T));
  if (mode == LOGPROBS) return launch<T, LOGPROBS>(a, st);
  return mode == POLICY ? launch<T, POLICY>(a, st) : launch<T, POLICY_GRAD>(a, st);
}

static void set_temperature(double temperature, float &c, double &inv_t) {
  inv_t = 1.0 / temperature;
  c = (float)(1.4426950408889634074 * inv_t);
}
static void set_temperature(double temperature, Args &a) {
  set_temperature(temperature, a.c, a.inv_t);
  a.floor = -EDGE / a.c;
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
  rows::set_temperature(temperature, a);
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
  a.tc = temperature * (double)a.c;
  a.lse = lse;
  a.dlogp = dlogp;
  a.dlogits = dlogits;
  a.ldd = ld_dlogits;
  const int es = dtype == MSTAR_DTYPE_F32 ? 4 : 2;
  const int64_t per = (int64_t)rows::NT * 4 * 16 * 4;  // four unrolled steps of a block
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
  rows::set_temperature(p->temperature, a);
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
