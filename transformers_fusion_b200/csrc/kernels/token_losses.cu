// Losses of post-training on rows of logits, with the gradient of the logits: log-probabilities of given tokens, the clipped policy loss with
// a KL term, the paired preference loss, distillation from a teacher's top logits.
//
// Of a row z (V values) every one of them needs m = max z, S = sum exp((z - m) / tau), lse = m / tau + log S, and what it computes from them is
// one scalar c and few targets y_j with weights q_j:   dz = c p - sum_j q_j onehot(y_j),   p = exp((z - m) / tau) / S.
// The arithmetic is 32-bit; exponents are taken of z - m (exact for 16-bit logits that lie within a factor of two of m, and small where p is
// not), so that the soft-max of a long row is good to a few 1e-7.  Log-probabilities of a row, the sums over rows and the margins of pairs are 64-bit: a
// margin is the difference of two sums over a thousand tokens.  The gradient is rounded once, to the type of the logits.
//
// Reference counterparts: token log-probs, ratio clipping and KL of the RL trainers (src/trainer/trainer_rl.cpp:557-1350).
#include "tfb_host.h"
#include "tfb_ptx.cuh"

TFB_BOUNDS_DEFINE(token_losses)

namespace tfb {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int TL_MAX_TOP = 1024;      // entries of a teacher's row

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Rows of logits and of their gradient: row t is position t % S of sequence t / S.  Strides in elements; the last dimension is dense.
struct RowsArg {
  const void* z;
  void* dz;                            // null: no gradient
  long long zb, zs, db, ds;
  int T, S, V, f32;
};

enum : int { MODE_STATS = 0, MODE_GRAD = 1, MODE_POLICY = 2, MODE_DISTILL = 3 };
enum : int { KL_K3 = 0, KL_K1 = 1 };
enum : int { MEAN_TOKENS = 0, MEAN_SEQUENCES = 1, MEAN_SUM = 2 };

struct LossArg {
  const void* targets;                 // [T] int64 or int32
  int idx64;
  long long ignore;
  // statistics
  float* logp;                         // [T]
  float* stats;                        // [2, T]: m and log S apart, since their sum in 32 bits loses log S where |m| is large; MODE_GRAD reads them
  float* lse;                          // [T] or null: the sum
  double* logp64;                      // [T], preference
  // MODE_GRAD: coefficient of a row
  const float* dlogp;                  // [T], or [T / S] with per_seq
  int per_seq;
  // MODE_POLICY
  const float *adv, *old_lp, *ref_lp;
  int adv_seq, ratio, kl_kind;
  float lo, hi, kl_coef;               // clip to [lo, hi]
  // MODE_DISTILL
  const void *top_ids, *top_z;         // [T, K]
  int K, top_f32;
  float inv_tau, tau;
  // means: weight of a row = 1 / (scale * denom[per-sequence or 0])
  const float* denom;
  int mean;
  float scale;
  float* terms;                        // [3, T]: weighted loss, kl, share of clipped tokens
};

__device__ __forceinline__ long long ld_idx(const void* p, long long i, int is64) {
  return is64 ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

__device__ __forceinline__ float ld_z(const void* row, long long i, int f32) {
  return f32 ? static_cast<const float*>(row)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]);
}

// (m, s) of a part of a row: s = sum exp2((z - m) k).  A part without a finite or infinite value has m = -inf, s = 0.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2, float k) {
  const float M = fmaxf(m, m2);
  const float r = M == -INFINITY ? 0.f : M;
  s = s * ex2((m - r) * k) + s2 * ex2((m2 - r) * k);
  m = M;
}

__device__ __forceinline__ void block_join(float& m, float& s, float k, float2* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) join(m, s, __shfl_xor_sync(~0u, m, o), __shfl_xor_sync(~0u, s, o), k);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  if (lane == 0) sh[warp] = make_float2(m, s);
  __syncthreads();
  const float2 v = lane < nw ? sh[lane] : make_float2(-INFINITY, 0.f);
  m = v.x;
  s = v.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) join(m, s, __shfl_xor_sync(~0u, m, o), __shfl_xor_sync(~0u, s, o), k);
  // a join rounds its two sides differently, so the lanes' sums differ in their last bits: all go on with one
  m = __shfl_sync(~0u, m, 0);
  s = __shfl_sync(~0u, s, 0);
}

__device__ __forceinline__ float weight_of(const LossArg& a, long long t, int S) {
  if (a.mean == MEAN_SUM) return 1.f / a.scale;
  return 1.f / (a.scale * a.denom[a.mean == MEAN_SEQUENCES ? t / S : 0]);
}

// The policy's term of one token: l, its KL estimate, whether the clip took its gradient, and g = dl / dlp.
//   s = r A, r = exp(lp - old); with a clip the smaller of that and clamp(r) A, whose gradient is 0 where it is the smaller one.
//   Without a ratio s = A lp.  kl: k3 = exp(x) - 1 - x, k1 = x, x = ref - lp.
__device__ __forceinline__ void policy_terms(const LossArg& a, float lp, float lp_old, float ref_lp, float A, float& l, float& kl, float& clipped, float& g) {
  float s, ds;
  clipped = 0.f;
  if (a.ratio) {
    const float r = expf(lp_old);
    s = ds = r * A;
    const float c = fminf(fmaxf(r, a.lo), a.hi) * A;
    if (c < s) { s = c; ds = 0.f; clipped = 1.f; }
  } else {
    s = A * lp;
    ds = A;
  }
  kl = 0.f;
  float dkl = 0.f;
  if (a.ref_lp) {
    const float e = expm1f(ref_lp);
    kl = a.kl_kind == KL_K3 ? e - ref_lp : ref_lp;
    dkl = a.kl_kind == KL_K3 ? -e : -1.f;
  }
  l = fmaf(a.kl_coef, kl, -s);
  g = lp != lp ? lp : fmaf(a.kl_coef, dkl, -ds);       // also where the objective's gradient does not depend on lp
}

// ---------------------------------------------------------------------------------------------------------------------
// The general form: one block per row, the row read twice.  Takes any alignment and any vocabulary: values up to the first 16-byte boundary and
// behind the last one by themselves, vectors between.
// ---------------------------------------------------------------------------------------------------------------------
template <class T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16(v); }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};

// values in front of the first 16-byte boundary of a row
template <class T>
__device__ __forceinline__ int head_of(const T* p, int V) {
  return min(V, int(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
}

template <class T>
__device__ __forceinline__ void row_stats(const T* row, int V, float k, float& m, float& s) {
  constexpr int N = Vec<T>::N;
  m = -INFINITY;
  s = 0.f;
  const int head = head_of(row, V), nv = (V - head) / N;
  const uint4* v = reinterpret_cast<const uint4*>(row + head);
  for (int i = threadIdx.x; i < nv; i += blockDim.x) {
    float f[N], mx = m;
    Vec<T>::unpack(v[i], f);
#pragma unroll
    for (int j = 0; j < N; ++j) mx = fmaxf(mx, f[j]);
    const float r = mx == -INFINITY ? 0.f : mx;
    s *= ex2((m - r) * k);
#pragma unroll
    for (int j = 0; j < N; ++j) s += ex2((f[j] - r) * k);
    m = mx;
  }
  const int tail = head + nv * N;
  if (int(threadIdx.x) < head) join(m, s, Vec<T>::get(row[threadIdx.x]), 1.f, k);
  if (tail + int(threadIdx.x) < V) join(m, s, Vec<T>::get(row[tail + threadIdx.x]), 1.f, k);
}

template <class T>
__device__ __forceinline__ void row_zero(T* row, int V) {
  constexpr int N = Vec<T>::N;
  const int head = head_of(row, V), nv = (V - head) / N, tail = head + nv * N;
  for (int i = threadIdx.x; i < nv; i += blockDim.x) reinterpret_cast<uint4*>(row + head)[i] = make_uint4(0, 0, 0, 0);
  if (int(threadIdx.x) < head) row[threadIdx.x] = Vec<T>::put(0.f);
  if (tail + int(threadIdx.x) < V) row[tail + threadIdx.x] = Vec<T>::put(0.f);
}

// dz = c exp2((z - m) k), minus hot at index y
template <class T>
__device__ __forceinline__ void row_grad(const T* row, T* out, int V, float k, float m, float c, long long y, float hot) {
  constexpr int N = Vec<T>::N;
  const int head = head_of(row, V), nv = (V - head) / N, tail = head + nv * N;
  const bool same = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const uint4* v = reinterpret_cast<const uint4*>(row + head);
  auto one = [&](int i) {
    float g = c * ex2((Vec<T>::get(row[i]) - m) * k);
    if (i == y) g -= hot;
    out[i] = Vec<T>::put(g);
  };
  for (int i = threadIdx.x; i < nv; i += blockDim.x) {
    float f[N];
    Vec<T>::unpack(v[i], f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      f[j] = c * ex2((f[j] - m) * k);
      if (head + i * N + j == y) f[j] -= hot;
    }
    if (same) {
      reinterpret_cast<uint4*>(out + head)[i] = Vec<T>::pack(f);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) out[head + i * N + j] = Vec<T>::put(f[j]);
    }
  }
  if (int(threadIdx.x) < head) one(threadIdx.x);
  if (tail + int(threadIdx.x) < V) one(tail + threadIdx.x);
}

constexpr int ROW_THREADS = 512;

template <class T, int MODE>
__global__ void __launch_bounds__(ROW_THREADS) row_loss_kernel(const RowsArg r, const LossArg a) {
  tfb::pdl_sync();
  __shared__ float2 sh[32];
  extern __shared__ char dyn[];                        // MODE_DISTILL: K teacher weights, K ids
  const long long t = blockIdx.x, b = t / r.S, pos = t - b * r.S;
  const T* row = static_cast<const T*>(r.z) + b * r.zb + pos * r.zs;
  T* out = r.dz ? static_cast<T*>(r.dz) + b * r.db + pos * r.ds : nullptr;
  const float k = MODE == MODE_DISTILL ? LOG2E * a.inv_tau : LOG2E;

  if constexpr (MODE == MODE_DISTILL) {
    const bool off = ld_idx(a.top_ids, t * a.K, a.idx64) < 0;
    if (off) {
      if (threadIdx.x == 0) { a.logp[t] = 0.f; a.terms[t] = 0.f; }
      if (out) row_zero(out, r.V);
      return;
    }
    float* q = reinterpret_cast<float*>(dyn);
    int* id = reinterpret_cast<int*>(q + a.K);
    float m, s;
    row_stats(row, r.V, k, m, s);
    block_join(m, s, k, sh);
    __syncthreads();
    // the teacher's weights: soft-max over the row's entries
    float tm = -INFINITY, ts = 0.f;
    for (int j = threadIdx.x; j < a.K; j += blockDim.x) {
      const long long y = ld_idx(a.top_ids, t * a.K + j, a.idx64);
      TFB_BOUNDS(y < r.V, 3, y, r.V);
      const bool have = y >= 0 && y < r.V;
      const float z = have ? ld_z(a.top_z, t * a.K + j, a.top_f32) : -INFINITY;
      q[j] = z;
      id[j] = y >= r.V ? -2 : (have ? int(y) : -1);
      join(tm, ts, z, 1.f, k);
    }
    block_join(tm, ts, k, sh);
    const float tr = tm == -INFINITY ? 0.f : tm;
    float kl = 0.f;
    bool bad = false;
    const float mr = m == -INFINITY ? 0.f : m, ls = logf(s), lts = logf(ts);
    for (int j = threadIdx.x; j < a.K; j += blockDim.x) {
      if (id[j] == -2) bad = true;
      const float lq = (q[j] - tr) * a.inv_tau - lts, w = ex2((q[j] - tr) * k) / ts;
      q[j] = id[j] >= 0 ? w : 0.f;
      if (id[j] >= 0 && q[j] != 0.f) kl += q[j] * (lq - ((Vec<T>::get(row[id[j]]) - mr) * a.inv_tau - ls));
    }
    const int any_bad = __syncthreads_or(bad);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) kl += __shfl_xor_sync(~0u, kl, o);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5].x = kl;
    __syncthreads();
    const float w = any_bad ? NAN : weight_of(a, t, r.S);
    if (threadIdx.x == 0) {
      kl = 0.f;
      for (int i = 0; i < int(blockDim.x >> 5); ++i) kl += sh[i].x;
      if (any_bad) kl = NAN;
      a.logp[t] = kl;
      a.terms[t] = kl * a.tau * a.tau * w;
    }
    if (!out) return;
    // the entries' own gradients, each from its value of z, before the row is written (it may be written in place)
    const float c = a.tau * w;
    constexpr int PER = TL_MAX_TOP / ROW_THREADS;
    float g[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int j = threadIdx.x + u * ROW_THREADS;
      g[u] = 0.f;
      if (j < a.K && id[j] >= 0) {
        float sum = 0.f;
        for (int i = 0; i < a.K; ++i) sum += id[i] == id[j] ? q[i] : 0.f;       // an id may come twice
        g[u] = c * (ex2((Vec<T>::get(row[id[j]]) - mr) * k) / s - sum);
      }
    }
    __syncthreads();
    row_grad(row, out, r.V, k, mr, c / s, -1, 0.f);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int j = threadIdx.x + u * ROW_THREADS;
      if (j < a.K && id[j] >= 0) out[id[j]] = Vec<T>::put(g[u]);
    }
    return;
  } else {
    const long long y = ld_idx(a.targets, t, a.idx64);
    if (y == a.ignore) {
      if (threadIdx.x == 0) {
        if (MODE == MODE_STATS && a.logp64) a.logp64[t] = 0.0;
        if (MODE == MODE_STATS && a.lse) a.lse[t] = 0.f;
        if (MODE == MODE_STATS && a.stats) a.stats[t] = a.stats[r.T + t] = 0.f;
        if (MODE != MODE_GRAD && a.logp) a.logp[t] = 0.f;
        if (MODE == MODE_POLICY) a.terms[t] = a.terms[r.T + t] = a.terms[2ll * r.T + t] = 0.f;
      }
      if (MODE != MODE_STATS && out) row_zero(out, r.V);
      return;
    }
    if (threadIdx.x == 0) TFB_BOUNDS(y >= 0 && y < r.V, 3, y, r.V);
    const float zy = y >= 0 && y < r.V ? Vec<T>::get(row[y]) : NAN;       // a target outside the vocabulary makes its row NaN
    if constexpr (MODE == MODE_GRAD) {
      const float m = a.stats[t], mr = m == -INFINITY ? 0.f : m, p = ex2(-a.stats[r.T + t] * k);       // 1 / S
      const float c = zy != zy ? NAN : (a.per_seq ? a.dlogp[b] : a.dlogp[t]);
      __syncthreads();
      row_grad(row, out, r.V, k, mr, -c * p, y, -c);
    } else {
      float m, s;
      row_stats(row, r.V, k, m, s);
      block_join(m, s, k, sh);
      const float lp = (zy - m) - logf(s);
      float g = 0.f, w = 0.f;
      if constexpr (MODE == MODE_POLICY) w = weight_of(a, t, r.S);
      if (threadIdx.x == 0 || MODE == MODE_POLICY) {
        if constexpr (MODE == MODE_POLICY) {
          float l, kl, clipped;
          policy_terms(a, lp, a.old_lp ? lp - a.old_lp[t] : 0.f, a.ref_lp ? a.ref_lp[t] - lp : 0.f, a.adv[a.adv_seq ? b : t], l, kl, clipped, g);
        }
      }
      if (threadIdx.x == 0) {
        const double ls = log(double(s)), lp64 = double(zy) - double(m) - ls;
        if (MODE == MODE_STATS && a.logp64) a.logp64[t] = lp64;
        if (MODE == MODE_STATS && a.lse) a.lse[t] = float(double(m) + ls);
        if (MODE == MODE_STATS && a.stats) { a.stats[t] = m; a.stats[r.T + t] = float(ls); }
        if (a.logp) a.logp[t] = float(lp64);
        if constexpr (MODE == MODE_POLICY) {
          float l, kl, clipped, gg;
          policy_terms(a, float(lp64), a.old_lp ? float(lp64 - double(a.old_lp[t])) : 0.f, a.ref_lp ? float(double(a.ref_lp[t]) - lp64) : 0.f,
                       a.adv[a.adv_seq ? b : t], l, kl, clipped, gg);
          a.terms[t] = w * l;
          a.terms[r.T + t] = w * kl;
          a.terms[2ll * r.T + t] = w * clipped;
        }
      }
      if (MODE == MODE_POLICY && out) {
        const float c = w * g;
        row_grad(row, out, r.V, k, m == -INFINITY ? 0.f : m, -c / s, y, -c);
      }
    }
  }
}

// denom[0] = number of rows that count (at least 1), or denom[i] = that of sequence i.  `stride`: distance between the indices that say so (targets: 1,
// a teacher's ids: K); a row counts where its index is not `ignore` (targets) or not negative (first id).
__global__ void __launch_bounds__(1024) row_count_kernel(const void* idx, int idx64, long long stride, long long ignore, int negative, int N, int S, int per_seq,
                                                         float* denom) {
  tfb::pdl_sync();
  __shared__ int sh[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto counts = [&](long long t) {
    const long long y = ld_idx(idx, t * stride, idx64);
    return negative ? y >= 0 : y != ignore;
  };
  if (per_seq) {
    for (int n = blockIdx.x * 32 + warp; n < N; n += gridDim.x * 32) {
      int c = 0;
      for (int i = lane; i < S; i += 32) c += counts((long long)n * S + i);
      c = __reduce_add_sync(~0u, c);
      if (lane == 0) denom[n] = float(max(c, 1));
    }
    return;
  }
  int c = 0;
  for (long long t = threadIdx.x; t < (long long)N * S; t += 1024) c += counts(t);
  c = __reduce_add_sync(~0u, c);
  if (lane == 0) sh[warp] = c;
  __syncthreads();
  if (warp == 0) {
    c = __reduce_add_sync(~0u, sh[lane]);
    if (lane == 0) denom[0] = float(max(c, 1));
  }
}

__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  __syncthreads();
  if (lane == 0) sh[warp] = v;
  __syncthreads();
  v = lane < nw ? sh[lane] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// out[i] = sum of terms[i * T ...], i < n, in 64 bits and always in the same order
__global__ void __launch_bounds__(1024) term_sum_kernel(const float* terms, int T, int n, float* out) {
  tfb::pdl_sync();
  __shared__ double sh[32];
  for (int i = 0; i < n; ++i) {
    double v = 0.0;
    for (int t = threadIdx.x; t < T; t += 1024) v += double(terms[(long long)i * T + t]);
    v = block_sum(v, sh);
    if (threadIdx.x == 0) out[i] = float(v);
  }
}

// One block per pair: sums of both answers' log-probabilities, margin, loss, and the coefficient of each answer's rows.
struct PairArg {
  const double* lp;                    // [2N, S]
  const void* targets;
  int idx64;
  long long ignore;
  const float* ref;                    // [2N] or null
  int N, S, kind, average;             // kind: 0 sigmoid, 1 hinge, 2 squared
  float beta, smooth;
  float *logp, *margins, *coef, *terms;   // [2N], [N], [2N], [N]
};
__global__ void __launch_bounds__(256) pair_kernel(const PairArg a) {
  tfb::pdl_sync();
  __shared__ double sh[32];
  const int n = blockIdx.x;
  double L[2], cnt[2];
  for (int h = 0; h < 2; ++h) {
    const long long t0 = (long long)(n + h * a.N) * a.S;
    double v = 0.0, c = 0.0;
    for (int i = threadIdx.x; i < a.S; i += 256) {
      v += a.lp[t0 + i];
      c += ld_idx(a.targets, t0 + i, a.idx64) != a.ignore ? 1.0 : 0.0;
    }
    L[h] = block_sum(v, sh);
    cnt[h] = a.average ? fmax(1.0, block_sum(c, sh)) : 1.0;
    L[h] /= cnt[h];
  }
  if (threadIdx.x) return;
  const double h = (L[0] - (a.ref ? double(a.ref[n]) : 0.0)) - (L[1] - (a.ref ? double(a.ref[a.N + n]) : 0.0));
  const double x = double(a.beta) * h;
  double l, dl;                        // of h
  if (a.kind == 0) {
    const double e = exp(-fabs(x)), sneg = x >= 0 ? e / (1.0 + e) : 1.0 / (1.0 + e);      // sigmoid(-x)
    l = log1p(e) + fmax(-x, 0.0) + double(a.smooth) * x;          // -(1 - s) log sig(x) - s log sig(-x)
    dl = double(a.beta) * (double(a.smooth) - sneg);
  } else if (a.kind == 1) {
    l = fmax(0.0, 1.0 - x);
    dl = x < 1.0 ? -double(a.beta) : 0.0;
    if (x != x) { l = x; dl = x; }
  } else {
    const double d = h - 0.5 / double(a.beta);
    l = d * d;
    dl = 2.0 * d;
  }
  a.terms[n] = float(l / a.N);
  a.margins[n] = float(x);
  for (int i = 0; i < 2; ++i) {
    a.logp[n + i * a.N] = float(L[i]);
    a.coef[n + i * a.N] = float((i ? -dl : dl) / a.N / cnt[i]);
  }
}

template <int MODE>
static int launch_rows(const RowsArg& r, const LossArg& a, cudaStream_t st) {
  const size_t smem = MODE == MODE_DISTILL ? size_t(a.K) * 8 : 0;
  if (r.f32) tfb::launch_k_rows(r.T, row_loss_kernel<float, MODE>, r.T, ROW_THREADS, smem, st, r, a);
  else tfb::launch_k_rows(r.T, row_loss_kernel<__nv_bfloat16, MODE>, r.T, ROW_THREADS, smem, st, r, a);
  return int(cudaGetLastError());
}

static bool bad_rows(const RowsArg& r) { return !r.z || r.T <= 0 || r.S <= 0 || r.V <= 0 || r.T % r.S; }

}  // namespace tfb

using namespace tfb;

// logp, lse [T], stats [2, T] (each may be null); 0 where the target is `ignore`.
TFB_API int tfb_token_logprobs(const RowsArg* r, const void* targets, int idx64, long long ignore, float* logp, float* lse, float* stats, void* stream) {
  if (!r || bad_rows(*r) || !targets) return TFB_ERR_ARG;
  LossArg a = {};
  a.targets = targets; a.idx64 = idx64; a.ignore = ignore;
  a.logp = logp; a.lse = lse; a.stats = stats;
  return launch_rows<MODE_STATS>(*r, a, static_cast<cudaStream_t>(stream));
}

// dz = dlogp (onehot(target) - softmax z)
TFB_API int tfb_token_logprobs_bwd(const RowsArg* r, const void* targets, int idx64, long long ignore, const float* stats, const float* dlogp,
                                   void* stream) {
  if (!r || bad_rows(*r) || !targets || !stats || !dlogp || !r->dz) return TFB_ERR_ARG;
  LossArg a = {};
  a.targets = targets; a.idx64 = idx64; a.ignore = ignore;
  a.stats = const_cast<float*>(stats); a.dlogp = dlogp;
  return launch_rows<MODE_GRAD>(*r, a, static_cast<cudaStream_t>(stream));
}

struct PolicyArg {
  const void* targets;
  int idx64;
  long long ignore;
  const float *adv, *old_lp, *ref_lp;
  int adv_seq, ratio, kl_kind, mean;
  float lo, hi, kl_coef;
  const float* n_valid;                // 1 value: overrides the count of the mean over tokens
  float *logp, *out;                   // [T], [3]: loss, kl, share of clipped tokens
  float *denom, *terms;                // workspace: [max(1, T / S)], [3 T]
};
TFB_API int tfb_policy_loss(const RowsArg* r, const PolicyArg* p, void* stream) {
  if (!r || !p || bad_rows(*r) || !p->targets || !p->adv || !p->logp || !p->out || !p->denom || !p->terms) return TFB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int N = r->T / r->S;
  LossArg a = {};
  a.targets = p->targets; a.idx64 = p->idx64; a.ignore = p->ignore;
  a.logp = p->logp; a.adv = p->adv; a.old_lp = p->old_lp; a.ref_lp = p->ref_lp;
  a.adv_seq = p->adv_seq; a.ratio = p->ratio; a.kl_kind = p->kl_kind;
  a.lo = p->lo; a.hi = p->hi; a.kl_coef = p->kl_coef;
  a.mean = p->mean; a.scale = p->mean == MEAN_SEQUENCES ? float(N) : 1.f;
  a.denom = p->n_valid && p->mean == MEAN_TOKENS ? p->n_valid : p->denom;
  a.terms = p->terms;
  if (a.denom == p->denom && p->mean != MEAN_SUM) {
    const int seq = p->mean == MEAN_SEQUENCES;
    tfb::launch_k_rows(r->T, row_count_kernel, seq ? (N + 31) / 32 : 1, 1024, 0, st, p->targets, p->idx64, 1ll, p->ignore, 0, N, r->S, seq, p->denom);
  }
  if (int rc = launch_rows<MODE_POLICY>(*r, a, st)) return rc;
  tfb::launch_k_rows(r->T, term_sum_kernel, 1, 1024, 0, st, p->terms, r->T, 3, p->out);
  return int(cudaGetLastError());
}

struct PreferenceArg {
  const void* targets;
  int idx64;
  long long ignore;
  const float* ref;
  int kind, average;
  float beta, smooth;
  float *loss, *margins, *logp;        // [1], [N], [2N]
  double* lp64;                        // workspace: [T], [2, T], [2N], [N]
  float *stats, *coef, *terms;
};
TFB_API int tfb_preference_loss(const RowsArg* r, const PreferenceArg* p, void* stream) {
  if (!r || !p || bad_rows(*r) || (r->T / r->S) % 2 || !p->targets || !p->loss || !p->margins || !p->logp || !p->lp64 || !p->stats || !p->coef || !p->terms)
    return TFB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LossArg a = {};
  a.targets = p->targets; a.idx64 = p->idx64; a.ignore = p->ignore;
  a.stats = p->stats; a.logp64 = p->lp64;
  if (int rc = launch_rows<MODE_STATS>(*r, a, st)) return rc;
  PairArg q = {p->lp64, p->targets, p->idx64, p->ignore, p->ref, r->T / r->S / 2, r->S, p->kind, p->average, p->beta, p->smooth, p->logp, p->margins, p->coef, p->terms};
  tfb::launch_k_rows(r->T, pair_kernel, q.N, 256, 0, st, q);
  tfb::launch_k_rows(r->T, term_sum_kernel, 1, 1024, 0, st, p->terms, q.N, 1, p->loss);
  if (!r->dz) return int(cudaGetLastError());
  a.dlogp = p->coef; a.per_seq = 1; a.logp64 = nullptr;
  return launch_rows<MODE_GRAD>(*r, a, st);
}

struct DistillArg {
  const void *top_ids, *top_z;
  int idx64, top_f32, K;
  float tau;
  const float* n_valid;
  float *kl, *loss;                    // [T], [1]
  float *denom, *terms;                // workspace: [1], [T]
};
TFB_API int tfb_distill_loss(const RowsArg* r, const DistillArg* p, void* stream) {
  if (!r || !p || bad_rows(*r) || !p->top_ids || !p->top_z || p->K <= 0 || !(p->tau > 0.f) || !p->kl || !p->loss || !p->denom || !p->terms) return TFB_ERR_ARG;
  if (p->K > TL_MAX_TOP) return TFB_ERR_LIMIT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LossArg a = {};
  a.idx64 = p->idx64; a.logp = p->kl; a.top_ids = p->top_ids; a.top_z = p->top_z; a.K = p->K; a.top_f32 = p->top_f32;
  a.tau = p->tau; a.inv_tau = 1.f / p->tau;
  a.mean = MEAN_TOKENS; a.scale = 1.f; a.denom = p->n_valid ? p->n_valid : p->denom; a.terms = p->terms;
  if (!p->n_valid)
    tfb::launch_k_rows(r->T, row_count_kernel, 1, 1024, 0, st, p->top_ids, p->idx64, (long long)p->K, 0ll, 1, 1, r->T, 0, p->denom);
  if (int rc = launch_rows<MODE_DISTILL>(*r, a, st)) return rc;
  tfb::launch_k_rows(r->T, term_sum_kernel, 1, 1024, 0, st, p->terms, r->T, 1, p->loss);
  return int(cudaGetLastError());
}
