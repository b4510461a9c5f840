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
#include "row_losses.cuh"
#include "tfb_host.h"

TFB_BOUNDS_DEFINE(token_losses)

namespace tfb {

constexpr int TL_MAX_TOP = 1024;      // entries of a teacher's row

// Rows of logits and of their gradient: row t is position t % S of sequence t / S.  Strides in elements; the last dimension is dense.
struct RowsArg {
  const void* z;
  void* dz;                            // null: no gradient
  long long zb, zs, db, ds;
  int T, S, V, f32;
  int* status;                         // device status word of the bounded waits
};

enum : int { MODE_STATS = 0, MODE_GRAD = 1, MODE_POLICY = 2, MODE_DISTILL = 3, MODE_SCORE = 4 };
enum : int { KL_K3 = 0, KL_K1 = 1, KL_LOG_RATIO = 2 };
enum : int { MEAN_TOKENS = 0, MEAN_SEQUENCES = 1, MEAN_SUM = 2 };

struct LossArg {
  const void* targets;                 // [T] int64 or int32
  int idx64;
  long long ignore;
  // statistics
  float* logp;                         // [T]
  float* stats;                        // [2, T]: m and log S apart, since their sum in 32 bits loses log S where |m| is large; MODE_GRAD reads them
  double* logp64;                      // [T], preference
  // MODE_SCORE: rows without their targets' columns, which are -inf in z
  const float* zy;                     // [T] the targets' logits
  float* lse;                          // [T]
  // MODE_GRAD: coefficient of a row
  const float* dlogp;                  // [T], or [T / S] with per_seq
  int per_seq, split;                  // blocks of a row
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
  float* terms;                        // general form, [3, T]: weighted loss, kl, share of clipped tokens
  int* zero;                           // a word that the first block clears for the kernel that follows, or null
};

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

__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
// (m, s) of all lanes together, the same bits in every lane
__device__ __forceinline__ void warp_join(float& m, float& s, float k) {
  const float M = warp_max(m), r = M == -INFINITY ? 0.f : M;
  s = warp_sum(s * ex2((m - r) * k));
  m = M;
}
// log s to a few 1e-8 (absolute), where logf(s) alone has the rounding of its result: the exponent's part in 64 bits, the rest in [0, log 2)
__device__ __forceinline__ double log64(float s) {
  if (!(s >= 1.f && s < INFINITY)) return double(logf(s));
  const int e = (__float_as_int(s) >> 23) - 127;
  return double(e) * 0.6931471805599453 + double(logf(__int_as_float((__float_as_int(s) & 0x7fffff) | 0x3f800000)));
}

__device__ __forceinline__ float weight_of(const LossArg& a, long long t, int S) {
  if (a.mean == MEAN_SUM) return 1.f / a.scale;
  return 1.f / (a.scale * a.denom[a.mean == MEAN_SEQUENCES ? t / S : 0]);
}

// The policy's term of one token: l, its KL estimate, whether the clip took its gradient, and g = dl / dlp.
//   s = r A, r = exp(lp - old); with a clip the smaller of that and clamp(r) A, whose gradient is 0 where it is the smaller one.
//   Without older log-probabilities old is lp itself, so that a row without a log-probability (NaN, -inf) has no ratio either: its loss is NaN as its gradient is.
//   Without a ratio s = A lp.  kl: k3 = exp(x) - 1 - x, k1 = x, log_ratio = -x, x = ref - lp.
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
    kl = a.kl_kind == KL_K3 && ref_lp != INFINITY ? e - ref_lp : a.kl_kind == KL_LOG_RATIO ? -ref_lp : ref_lp;
    dkl = a.kl_kind == KL_K3 ? -e : a.kl_kind == KL_LOG_RATIO ? 1.f : -1.f;
  }
  // a KL term that is only reported has no part in the loss, not even an infinite one; a NaN has, also where the gradient does not depend on lp
  l = a.kl_coef != 0.f ? fmaf(a.kl_coef, kl, -s) : -s;
  g = lp != lp ? lp : a.kl_coef != 0.f ? fmaf(a.kl_coef, dkl, -ds) : -ds;
}

__device__ __forceinline__ void policy_row(const LossArg& a, double lp, long long t, long long b, float& l, float& kl, float& clipped, float& g) {
  policy_terms(a, float(lp), float(lp - (a.old_lp ? double(a.old_lp[t]) : lp)), a.ref_lp ? float(double(a.ref_lp[t]) - lp) : 0.f, a.adv[a.adv_seq ? b : t], l, kl,
               clipped, g);
}

// what a row leaves behind: m, log S and the log-probability of its target (MODE_SCORE: that and the row's logsumexp; see put_score for rows that count)
template <int MODE>
__device__ __forceinline__ void put_stats(const LossArg& a, int T, long long t, float m, double ls, double lp) {
  if (MODE != MODE_GRAD && a.logp) a.logp[t] = float(lp);
  if (MODE == MODE_SCORE) a.lse[t] = float(lp);
  if (MODE != MODE_STATS) return;
  if (a.logp64) a.logp64[t] = lp;
  if (a.stats) {
    a.stats[t] = m;
    a.stats[T + t] = float(ls);
  }
}

__device__ __forceinline__ void put_score(const LossArg& a, long long t, bool in, float m, float s) {
  score_of(m, double(s), a.zy[t], in, a.logp[t], a.lse[t]);
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

// maximum and sum of a batch of values, joined to (m, s): one rescaling for all of them, short chains
template <int U, int N>
__device__ __forceinline__ void batch_stats(const float (&f)[U][N], float k, float& m, float& s) {
  float mx = m;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float a = fmax3(f[u][0], f[u][1], f[u][2]);
    if constexpr (N == 8) a = fmax3(fmax3(a, f[u][3], f[u][4]), f[u][5], fmaxf(f[u][6], f[u][7]));
    else a = fmaxf(a, f[u][3]);
    mx = fmaxf(mx, a);
  }
  const float ref = mx == -INFINITY ? 0.f : mx;
  const float2 neg = make_float2(-ref, -ref), k2 = make_float2(k, k);
  float2 t[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    t[u] = make_float2(0.f, 0.f);
#pragma unroll
    for (int x = 0; x < N; x += 2) {
      const float2 d = mul2(add2(make_float2(f[u][x], f[u][x + 1]), neg), k2);
      t[u] = add2(t[u], make_float2(ex2(d.x), ex2(d.y)));
    }
  }
#pragma unroll
  for (int u = 1; u < U; ++u) t[0] = add2(t[0], t[u]);
  s = fmaf(s, ex2((m - ref) * k), t[0].x + t[0].y);
  m = mx;
}

// tid, nt: thread of those that share the row, and how many they are
template <class T, int U>
__device__ __forceinline__ void row_stats(const T* row, int V, float k, float& m, float& s, int tid, int nt) {
  constexpr int N = Vec<T>::N;
  m = -INFINITY;
  s = 0.f;
  const int head = head_of(row, V), nv = (V - head) / N;
  const uint4* v = reinterpret_cast<const uint4*>(row + head);
  int i = tid;
  for (; i + (U - 1) * nt < nv; i += U * nt) {
    uint4 w[U];
    float f[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = v[i + u * nt];
#pragma unroll
    for (int u = 0; u < U; ++u) Vec<T>::unpack(w[u], f[u]);
    batch_stats<U, N>(f, k, m, s);
  }
  for (; i < nv; i += nt) {
    float f[1][N];
    Vec<T>::unpack(v[i], f[0]);
    batch_stats<1, N>(f, k, m, s);
  }
  const int tail = head + nv * N;
  if (tid < head) join(m, s, Vec<T>::get(row[tid]), 1.f, k);
  if (tail + tid < V) join(m, s, Vec<T>::get(row[tail + tid]), 1.f, k);
}

template <class T>
__device__ __forceinline__ void row_zero(T* row, int V, int tid, int nt) {
  constexpr int N = Vec<T>::N;
  const int head = head_of(row, V), nv = (V - head) / N, tail = head + nv * N;
  for (int i = tid; i < nv; i += nt) reinterpret_cast<uint4*>(row + head)[i] = make_uint4(0, 0, 0, 0);
  if (tid < head) row[tid] = Vec<T>::put(0.f);
  if (tail + tid < V) row[tail + tid] = Vec<T>::put(0.f);
}

// dz = c exp2((z - m) k), minus hot at index y
template <class T>
__device__ __forceinline__ void row_grad(const T* row, T* out, int V, float k, float m, float c, long long y, float hot, int tid, int nt) {
  constexpr int N = Vec<T>::N;
  const int head = head_of(row, V), nv = (V - head) / N, tail = head + nv * N;
  const bool same = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const uint4* v = reinterpret_cast<const uint4*>(row + head);
  auto one = [&](int i) {
    float g = c * ex2((Vec<T>::get(row[i]) - m) * k);
    if (i == y) g -= hot;
    out[i] = Vec<T>::put(g);
  };
  for (int i = tid; i < nv; i += nt) {
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
  if (tid < head) one(tid);
  if (tail + tid < V) one(tail + tid);
}

// An id may come twice among a teacher's entries, and the gradient at either has the weights of both.  A table of the ids (twice as many places as entries, -1 where
// empty) tells whether one does, since looking through all of a row's entries for each of them takes K^2 steps.
__host__ __device__ constexpr int top_table(int K) {
  int n = 64;
  while (n < 2 * K) n *= 2;
  return n;
}
__device__ __forceinline__ bool seen_before(int* table, int places, int id) {
  for (unsigned at = unsigned(id) * 2654435769u >> 16;; ++at) {      // (Knuth's multiplicative hash)
    const int o = atomicCAS(table + (at & unsigned(places - 1)), -1, id);
    if (o == -1 || o == id) return o == id;
  }
}

// In the general form a warp looks through up to 64 entries as fast: us, so / with the table, 8192 x 2000 20 entries 38 / 46, 64 45 / 53, 128 67 / 67; 20000 x 260 20 entries
// 44 / 47, 64 58 / 55, 128 113 / 61.
__host__ __device__ constexpr int row_table(bool warp, int K) { return warp && K <= 64 ? 0 : top_table(K); }

constexpr int ROW_THREADS = 512, WARP_ROWS = 8, WARP_TOP = 128;      // rows of a block, and most entries of a teacher's, with a warp to a row

// WARP: a warp to a row, WARP_ROWS rows to a block; else a block to a row.
template <class T, int MODE, bool WARP>
__global__ void __launch_bounds__(WARP ? WARP_ROWS * 32 : ROW_THREADS, WARP ? 5 : MODE == MODE_GRAD ? 4 : 3) row_loss_kernel(const RowsArg r, const LossArg a) {
  tfb::pdl_sync();
  __shared__ float2 sh[32];
  const int warp = threadIdx.x >> 5, split = !WARP && MODE == MODE_GRAD ? a.split : 1;
  const int nt = WARP ? 32 : ROW_THREADS * split, tid = WARP ? threadIdx.x & 31 : threadIdx.x + (split > 1 ? blockIdx.x % split * ROW_THREADS : 0);
  auto sync = [&] { if constexpr (WARP) __syncwarp(); else __syncthreads(); };
  auto join_all = [&](float& m, float& s, float k) { if constexpr (WARP) warp_join(m, s, k); else block_join(m, s, k, sh); };
  extern __shared__ __align__(128) char dyn[];         // MODE_DISTILL: K teacher weights, K ids, the ids' table
  if (a.zero && blockIdx.x == 0 && threadIdx.x == 0) *a.zero = 0;
  // the gradient of given statistics goes from the last row to the first: the pass that took them has left the last ones in L2
  const long long place = MODE == MODE_GRAD ? (gridDim.x - 1 - blockIdx.x) / split : blockIdx.x, t = WARP ? place * WARP_ROWS + warp : place;
  if (WARP && t >= r.T) return;
  const long long b = t / r.S, pos = t - b * r.S;
  const T* row = static_cast<const T*>(r.z) + b * r.zb + pos * r.zs;
  T* out = r.dz ? static_cast<T*>(r.dz) + b * r.db + pos * r.ds : nullptr;
  const float k = MODE == MODE_DISTILL ? LOG2E * a.inv_tau : LOG2E;

  if constexpr (MODE == MODE_DISTILL) {
    const bool off = ld_idx(a.top_ids, t * a.K, a.idx64) < 0;
    if (off) {
      if (tid == 0) { a.logp[t] = 0.f; a.terms[t] = 0.f; }
      if (out) row_zero(out, r.V, tid, nt);
      return;
    }
    const int places = row_table(WARP, a.K);
    float* q = reinterpret_cast<float*>(dyn) + (WARP ? warp * (2 * a.K + places) : 0);
    int *id = reinterpret_cast<int*>(q + a.K), *table = id + a.K;
    for (int i = tid; i < places; i += nt) table[i] = -1;
    float m, s;
    row_stats<T, 2>(row, r.V, k, m, s, tid, nt);
    join_all(m, s, k);
    sync();
    // the teacher's weights: soft-max over the row's entries
    float tm = -INFINITY, ts = 0.f;
    for (int j = tid; j < a.K; j += nt) {
      const long long y = ld_idx(a.top_ids, t * a.K + j, a.idx64);
      TFB_BOUNDS(y < r.V, 3, y, r.V);
      const bool have = y >= 0 && y < r.V;
      const float z = have ? ld_z(a.top_z, t * a.K + j, a.top_f32) : -INFINITY;
      q[j] = z;
      id[j] = y >= r.V ? -2 : (have ? int(y) : -1);
      join(tm, ts, z, 1.f, k);
    }
    join_all(tm, ts, k);
    const float tr = tm == -INFINITY ? 0.f : tm;
    float kl = 0.f;
    bool bad = false, twice = places == 0;
    const float mr = m == -INFINITY ? 0.f : m, ls = logf(s), lts = logf(ts);
    for (int j = tid; j < a.K; j += nt) {
      if (id[j] == -2) bad = true;
      const float lq = (q[j] - tr) * a.inv_tau - lts, w = ex2((q[j] - tr) * k) / ts;
      q[j] = id[j] >= 0 ? w : 0.f;
      if (places && out && id[j] >= 0) twice |= seen_before(table, places, id[j]);
      if (id[j] >= 0 && q[j] != 0.f) kl += q[j] * (lq - ((Vec<T>::get(row[id[j]]) - mr) * a.inv_tau - ls));
    }
    int any_bad;
    if constexpr (WARP) { any_bad = __any_sync(~0u, bad); twice = __any_sync(~0u, twice); __syncwarp(); } else { any_bad = __syncthreads_or(bad); twice = __syncthreads_or(twice); }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) kl += __shfl_xor_sync(~0u, kl, o);
    if constexpr (!WARP) {
      if ((threadIdx.x & 31) == 0) sh[warp].x = kl;
      __syncthreads();
    }
    const float w = any_bad ? NAN : weight_of(a, t, r.S);
    if (tid == 0) {
      if constexpr (!WARP) {
        kl = 0.f;
        for (int i = 0; i < ROW_THREADS / 32; ++i) kl += sh[i].x;
      }
      if (any_bad) kl = NAN;
      a.logp[t] = kl;
      a.terms[t] = kl * a.tau * a.tau * w;
    }
    if (!out) return;
    // the entries' own gradients, each from its value of z, before the row is written (it may be written in place)
    const float c = a.tau * w;
    constexpr int PER = WARP ? WARP_TOP / 32 : TL_MAX_TOP / ROW_THREADS;
    float g[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int j = tid + u * nt;
      g[u] = 0.f;
      if (j < a.K && id[j] >= 0) {
        float sum = twice ? 0.f : q[j];
        for (int i = 0; twice && i < a.K; ++i) sum += id[i] == id[j] ? q[i] : 0.f;
        g[u] = c * (ex2((Vec<T>::get(row[id[j]]) - mr) * k) / s - sum);
      }
    }
    sync();
    row_grad(row, out, r.V, k, mr, c / s, -1, 0.f, tid, nt);
    sync();
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int j = tid + u * nt;
      if (j < a.K && id[j] >= 0) out[id[j]] = Vec<T>::put(g[u]);
    }
    return;
  } else {
    const long long y = ld_idx(a.targets, t, a.idx64);
    if (y == a.ignore) {
      if (tid == 0) {
        put_stats<MODE>(a, r.T, t, 0.f, 0.0, 0.0);
        if (MODE == MODE_POLICY) a.terms[t] = a.terms[r.T + t] = a.terms[2ll * r.T + t] = 0.f;
      }
      if (MODE != MODE_STATS && out) row_zero(out, r.V, tid, nt);
      return;
    }
    if (tid == 0) TFB_BOUNDS(y >= 0 && y < r.V, 3, y, r.V);
    const bool in = y >= 0 && y < r.V;       // a target outside the vocabulary makes its row NaN
    if constexpr (MODE == MODE_GRAD) {
      const float m = a.stats[t], mr = m == -INFINITY ? 0.f : m, p = ex2(-a.stats[r.T + t] * k);       // 1 / S
      const float c = !in ? NAN : (a.per_seq ? a.dlogp[b] : a.dlogp[t]);
      row_grad(row, out, r.V, k, mr, -c * p, y, -c, tid, nt);
    } else {
      const float zy = in ? Vec<T>::get(row[y]) : NAN;
      float m, s;
      row_stats<T, 2>(row, r.V, k, m, s, tid, nt);
      join_all(m, s, k);
      const double ls = log64(s), lp64 = double(zy) - double(m) - ls;
      if (MODE == MODE_SCORE) {
        if (tid == 0) put_score(a, t, in, m, s);
        return;
      }
      float g = 0.f, w = 0.f, l = 0.f, kl = 0.f, clipped = 0.f;
      if constexpr (MODE == MODE_POLICY) {
        w = weight_of(a, t, r.S);
        policy_row(a, lp64, t, b, l, kl, clipped, g);
      }
      if (tid == 0) {
        put_stats<MODE>(a, r.T, t, m, ls, lp64);
        if constexpr (MODE == MODE_POLICY) {
          a.terms[t] = w * l;
          a.terms[r.T + t] = w * kl;
          a.terms[2ll * r.T + t] = w * clipped;
        }
      }
      if (MODE == MODE_POLICY && out) {
        const float c = w * g;
        sync();                        // everyone has read the target's logit (the row may be written in place)
        row_grad(row, out, r.V, k, m == -INFINITY ? 0.f : m, -c / s, y, -c, tid, nt);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// The pipelined form: a cluster of C blocks takes a row, each a slice of it that passes through shared memory once, so the row is read once and its
// gradient written once.  One persistent block per SM, whose warps work on different rows at a time:
//   producers (2 warps)  bulk copies of 16 KB chunks into a ring, as far ahead as the ring is free; a chunk to each in turn, since one warp takes ~400 ns for a
//                        chunk beside twenty busy ones
//   statistics (2 groups of 4 warps, 4 groups where no gradient follows)   (m, s) of the slice; the groups take chunks in turn, so that one's loads and joins
//                        run beside another's exponentials
//   control (4 warps)    rows in turn: joins the warps' and the cluster's (m, s), computes the loss, leaves the two scalars of the gradient
//   gradient (2 groups)  reads the slice again from the ring, exp2 by exp2, and stores it, 16 bytes per lane; frees the chunks
// The steps of one row wait for one another for microseconds (copy, joins, the exchange between SMs, the loss's arithmetic), which is why several
// rows have to be under way.  A block whose warps take the steps together (values kept in registers in between, one exponential each, two blocks per SM)
// reached 2.3 - 3.6 TB/s of reads and writes where this form reaches 5.0 - 5.6; without the statistics' arithmetic it copies at 6.1.  What bounds it: two
// exponentials per value keep the special function units 60 % busy, the issue slots 57 %.
//
// Values in front of a row's first 16-byte boundary and behind its last one, which a bulk copy cannot address, are put into the ring by the producer's
// lanes, and their vectors filled up with -inf; of the gradient they are stored one by one.  The blocks of a cluster exchange (m, s) through distributed shared memory: every block stores its own into all of
// them (st.async, which signals their barriers).
//
// Buffers of a row (PIPE_ROWS of each) are used again when they can be: a slot's partial sums after control is done with the row that had them before
// (statistics wait for that); the exchange's entries because the warp that sends for row n has finished row n - PIPE_C, for which every block's warp of the
// same number had sent, after it had read all its rows before (PIPE_ROWS >= 2 PIPE_C); the scalars because the ring holds fewer than PIPE_ROWS chunks.
//
// Sums over rows: every control warp adds up its own rows in their order, and the cluster that ends last adds the clusters' sums in theirs, so a
// result depends on the shapes alone (and the GPU).
// ---------------------------------------------------------------------------------------------------------------------
constexpr int PIPE_W = 4, PIPE_SG = 2, PIPE_GG = 2;                      // warps of a group, groups of statistics, of gradients
constexpr int PIPE_S = PIPE_SG * PIPE_W, PIPE_G = PIPE_GG * PIPE_W, PIPE_C = 4, PIPE_P = 2, PIPE_WARPS = PIPE_S + PIPE_G + PIPE_C + PIPE_P, PIPE_CLUSTERS = 148 * 2;
constexpr int CHUNK_VECS = 1024, CHUNK_BYTES = CHUNK_VECS * 16, PIPE_CHUNKS = 12, PIPE_ROWS = 16, TOP_LOADS = 2, LANE_VECS = 4, HALVES = CHUNK_VECS / (PIPE_W * 32 * LANE_VECS);

struct PipeArg {
  int vs, chunks, clusters, csize, nsums;
  double* partial;                     // [clusters, 3]
  int* counter;                        // 0 before the launch
  float* out;                          // [nsums]
};

__device__ __forceinline__ void st_async_v4(uint32_t addr, uint32_t bar, float4 v) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%2, %3, %4, %5}, [%1];" ::"r"(addr), "r"(bar), "f"(v.x), "f"(v.y), "f"(v.z),
               "f"(v.w)
               : "memory");
}

// The rows of a cluster, 32 at a time: every lane looks one up.
struct RowBlock {
  long long t, y, z, d;                // row, its index (target or first id), byte addresses of its logits and gradient
  unsigned valid, on;                  // lanes with a row; with one that counts
};

// One row as seen from a block: vector g of the row's 16-byte frame is whole for fv <= g < lv; this block's are [v0, v0 + n).
struct Slice {
  const char* frame;                   // 16-byte boundary at or before the first value
  int eoff, fv, lv, n;
  bool tail;                           // vector lv is there, in part
};
template <class T>
__device__ __forceinline__ Slice slice_of(long long z, int V, int v0, int vs) {
  Slice s;
  const int off = int(z & 15);
  s.frame = reinterpret_cast<const char*>(z - off);
  s.eoff = off / int(sizeof(T));
  s.fv = off ? 1 : 0;
  const long long bytes = off + (long long)V * int(sizeof(T));
  s.lv = int(bytes >> 4);
  s.tail = (bytes & 15) != 0;
  s.n = min(vs, int((bytes + 15) >> 4) - v0);
  return s;
}

// place in the ring: slot, and how often it has been used before (mod 2)
// The group of a role that takes a chunk is slot % groups, and the ring is a multiple of both roles' groups: a slot is always the same group's.  (With
// another group's use of the slot in between, a group ahead of that one would see the parity of the use before it and take it for its own.)
struct Cursor {
  uint32_t slot = 0, use = 0;
  __device__ __forceinline__ void next(uint32_t n) {
    if (++slot == n) { slot = 0; use ^= 1u; }
  }
};
static_assert(PIPE_CHUNKS % (PIPE_SG + PIPE_GG) == 0 && (PIPE_SG + PIPE_GG) % PIPE_SG == 0 && (PIPE_SG + PIPE_GG) % PIPE_GG == 0, "a slot belongs to one group of each role");
static_assert(PIPE_ROWS > PIPE_CHUNKS && PIPE_ROWS >= 2 * PIPE_C && PIPE_ROWS % PIPE_C == 0, "buffers of a row are free when they come round");

template <class T, int MODE, bool GRAD>
__global__ void __launch_bounds__(PIPE_WARPS * 32, 1) row_pipe_kernel(const RowsArg r, const LossArg a, const PipeArg q) {
  constexpr int N = Vec<T>::N, ES = int(sizeof(T)), LV = LANE_VECS, SGS = GRAD ? PIPE_SG : PIPE_SG + PIPE_GG, SW = SGS * PIPE_W;      // groups and warps of the statistics
  extern __shared__ __align__(128) char dyn[];       // ring of chunks; of a teacher's row, per control warp: weights, ids, gradients, table of ids
  __shared__ __align__(8) uint64_t bars[2 * PIPE_CHUNKS + 3 * PIPE_ROWS + PIPE_C];
  __shared__ float2 part[PIPE_ROWS][PIPE_S + PIPE_G];
  __shared__ __align__(16) float4 xch[PIPE_ROWS][8];
  __shared__ float4 coef[PIPE_ROWS];                 // m, scale, hot: dz = scale exp2((z - m) k) + hot onehot
  __shared__ double acc[PIPE_C][3];
  __shared__ __align__(16) uint4 lowest;             // a vector of -inf
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, C = q.csize, NCH = q.chunks;
  const int rank = C > 1 ? int(cluster_ctarank()) : 0, cl = int(blockIdx.x) / C, v0 = rank * q.vs;
  const uint32_t full = smem_u32(bars), empty = full + 8 * PIPE_CHUNKS, sdone = empty + 8 * PIPE_CHUNKS, cready = sdone + 8 * PIPE_ROWS,
                 xbar = cready + 8 * PIPE_ROWS, gdone = xbar + 8 * PIPE_ROWS;
  const float k = MODE == MODE_DISTILL ? LOG2E * a.inv_tau : LOG2E;
  const int K4 = MODE == MODE_DISTILL ? (a.K + 3) & ~3 : 0, table = MODE == MODE_DISTILL && GRAD ? top_table(a.K) : 0;
  auto entries = [&](int w) { return reinterpret_cast<float*>(dyn + NCH * CHUNK_BYTES) + w * (3 * K4 + table); };

  if (threadIdx.x == 0) {
    for (int i = 0; i < PIPE_CHUNKS; ++i) {
      mbar_init(full + i * 8, 1);
      mbar_init(empty + i * 8, PIPE_W);
    }
    for (int i = 0; i < PIPE_ROWS; ++i) {
      mbar_init(sdone + i * 8, SW);
      mbar_init(cready + i * 8, 1);
      mbar_init(xbar + i * 8, 1);
    }
    for (int i = 0; i < PIPE_C; ++i) mbar_init(gdone + i * 8, PIPE_G);
    *abort_flag = 0;
    const uint32_t inf = ES == 4 ? 0xff800000u : 0xff80ff80u;
    lowest = make_uint4(inf, inf, inf, inf);
    mbar_fence_init();
  }
  __syncthreads();
  if (C > 1) cluster_sync();           // the others' barriers are set up
  // Behind row_count_kernel, which has waited for everything before it when it lets this kernel start, only its own results have to be waited for: the
  // denominators (control warps) and the counter (at the end).  Rows are under way meanwhile.  (That kernel itself starts after its predecessor: placed early, its block kept
  // an SM from the rows; distillation at 12500 x 32000 344 us instead of 322.)
  constexpr bool COUNTED = MODE == MODE_POLICY || MODE == MODE_DISTILL;
  if (!COUNTED || (warp >= PIPE_S + PIPE_G && warp < PIPE_WARPS - PIPE_P)) tfb::pdl_sync();
  if (a.zero && blockIdx.x == 0 && threadIdx.x == 0) *a.zero = 0;

  auto rows_from = [&](long long base) {
    RowBlock b = {};
    b.t = cl + (base + lane) * q.clusters;
    const bool valid = b.t < r.T;
    if (valid) {
      b.y = MODE == MODE_DISTILL ? ld_idx(a.top_ids, b.t * a.K, a.idx64) : ld_idx(a.targets, b.t, a.idx64);
      const unsigned seq = unsigned(b.t) / unsigned(r.S), pos = unsigned(b.t) - seq * unsigned(r.S);
      b.z = reinterpret_cast<long long>(r.z) + (seq * r.zb + pos * r.zs) * ES;
      if (GRAD) b.d = reinterpret_cast<long long>(r.dz) + (seq * r.db + pos * r.ds) * ES;
    }
    b.valid = __ballot_sync(~0u, valid);
    b.on = __ballot_sync(~0u, valid && (MODE == MODE_DISTILL ? b.y >= 0 : b.y != a.ignore));
    return b;
  };
  auto lane_of = [&](long long v, int l) { return __shfl_sync(~0u, v, l); };
  const long long nrows = (r.T - cl + q.clusters - 1) / q.clusters;      // of this cluster (cl < T)
  // waits of a whole warp; `use`: how often the barrier has been waited for before
  auto wait = [&](uint32_t bar, unsigned use, int code) { return mbar_wait_warp(bar, use & 1u, abort_flag, r.status, code); };

  if (warp >= PIPE_WARPS - PIPE_P) {
    // ------------------------------ producers ------------------------------
    unsigned cc = 0;                   // chunks issued
    Cursor c;
    bool ok = true;
    // vectors that are not whole: the row's first (lanes 0 - 7) and last (8 - 15), filled up with -inf.  Loaded a row ahead.
    const int xe = lane & 7;
    auto edge_of = [&](const Slice& s) {
      const int g = lane < 8 ? (s.fv ? 0 : -1) : lane < 16 && s.tail ? s.lv : -1;
      return xe < N && g >= v0 && g < v0 + s.n ? g - v0 : -1;
    };
    auto edge_value = [&](const Slice& s, int ge) {
      const long long x = (long long)(v0 + ge) * N + xe - s.eoff;
      return ge >= 0 && x >= 0 && x < r.V ? (reinterpret_cast<const T*>(s.frame) + s.eoff)[x] : Vec<T>::put(-INFINITY);
    };
    for (long long base = 0; base < nrows && ok; base += 32) {
      const RowBlock b = rows_from(base);
      if (!b.on) continue;
      Slice s = slice_of<T>(lane_of(b.z, __ffs(b.on) - 1), r.V, v0, q.vs);
      int ge = edge_of(s);
      T ve = edge_value(s, ge);
      for (unsigned left = b.on; left && ok;) {
        left &= left - 1;
        const Slice next = slice_of<T>(lane_of(b.z, left ? __ffs(left) - 1 : 0), r.V, v0, q.vs);
        const int ge_next = left ? edge_of(next) : -1;
        const T ve_next = edge_value(next, ge_next);
        for (int c0 = 0; c0 < s.n; c0 += CHUNK_VECS, ++cc, c.next(NCH)) {
          const uint32_t slot = c.slot;
          if (int(slot % PIPE_P) != warp - (PIPE_WARPS - PIPE_P)) continue;
          if (cc >= unsigned(NCH) && !(ok = wait(empty + slot * 8, c.use ^ 1u, ST_TIMEOUT_EMPTY))) break;
          if (__any_sync(~0u, ge >= c0 && ge < c0 + CHUNK_VECS)) {
            if (ge >= c0 && ge < c0 + CHUNK_VECS) reinterpret_cast<T*>(dyn + slot * CHUNK_BYTES)[(ge - c0) * N + xe] = ve;
            __syncwarp();
          }
          if (lane == 0) {
            const int g0 = max(v0 + c0, s.fv), g1 = min(v0 + min(s.n, c0 + CHUNK_VECS), s.lv);
            if (g1 > g0) {
              mbar_expect_tx(full + slot * 8, uint32_t(g1 - g0) * 16);
              bulk_load(smem_u32(dyn) + slot * CHUNK_BYTES + uint32_t(g0 - v0 - c0) * 16, s.frame + (long long)g0 * 16, uint32_t(g1 - g0) * 16, full + slot * 8);
            } else {
              mbar_arrive(full + slot * 8);
            }
          }
        }
        s = next;
        ge = ge_next;
        ve = ve_next;
      }
    }
    if (!ok && lane == 0) {
      // unwinding: copies in flight land before shared memory goes away
      const uint64_t t0 = globaltimer_ns();
      for (unsigned i = cc > unsigned(NCH) ? cc - NCH : 0; i < cc; ++i)
        while (int(i % NCH % PIPE_P) == warp - (PIPE_WARPS - PIPE_P) && !mbar_try_wait(full + (i % NCH) * 8, (i / NCH) & 1u) && globaltimer_ns() - t0 < 2000000ull) {}
    }
  } else if (warp < SW) {
    // ------------------------------ statistics ------------------------------
    unsigned n = 0;
    Cursor c;
    bool ok = true;
    for (long long base = 0; base < nrows && ok; base += 32) {
      const RowBlock b = rows_from(base);
      for (unsigned left = b.on; left && ok; left &= left - 1, ++n) {
        const Slice s = slice_of<T>(lane_of(b.z, __ffs(left) - 1), r.V, v0, q.vs);
        float m = -INFINITY, sum = 0.f;
        for (int c0 = 0; c0 < s.n; c0 += CHUNK_VECS, c.next(NCH)) {
          if (int(c.slot % SGS) != warp / PIPE_W) continue;
          if (!(ok = wait(full + c.slot * 8, c.use, ST_TIMEOUT_FULL))) break;
#pragma unroll 1
          for (int h = 0; h < HALVES; ++h) {
            const int w0 = (h * PIPE_W + warp % PIPE_W) * LV * 32 + lane, left_vecs = s.n - c0;
            const uint4* src = reinterpret_cast<const uint4*>(dyn + c.slot * CHUNK_BYTES) + w0;
            float f[LV][N];
#pragma unroll
            for (int j = 0; j < LV; ++j) Vec<T>::unpack(w0 + j * 32 < left_vecs ? src[j * 32] : lowest, f[j]);      // what lies behind a slice is of other rows
            if (!GRAD && h == HALVES - 1) {    // in registers: the chunk is free
              __syncwarp();
              if (lane == 0) mbar_arrive(empty + c.slot * 8);
            }
            batch_stats<LV, N>(f, k, m, sum);
          }
        }
        if (!ok) break;
        warp_join(m, sum, k);
        const unsigned rs = n % PIPE_ROWS;
        if (n >= PIPE_ROWS && !(ok = wait(cready + rs * 8, n / PIPE_ROWS - 1, ST_TIMEOUT_TMEM_EMPTY))) break;
        if (lane == 0) {
          part[rs][warp] = make_float2(m, sum);
          mbar_arrive(sdone + rs * 8);
        }
      }
    }
  } else if (warp >= PIPE_S + PIPE_G) {
    // ------------------------------ control ------------------------------
    const int w = warp - PIPE_S - PIPE_G;
    double sums[3] = {0.0, 0.0, 0.0};
    unsigned n = 0;
    bool ok = true;
    for (long long base = 0; base < nrows && ok; base += 32) {
      const RowBlock b = rows_from(base);
      const bool live = (b.on >> lane) & 1u;
      if (w == 0 && rank == 0 && !live && ((b.valid >> lane) & 1u)) put_stats<MODE>(a, r.T, b.t, 0.f, 0.0, 0.0);
      // what the rows need from memory, all of them at once
      float zy = 0.f, adv = 0.f, old_lp = 0.f, ref_lp = 0.f, wt = 0.f;
      if (live && MODE != MODE_DISTILL) {
        const bool in = b.y >= 0 && b.y < r.V;
        TFB_BOUNDS(in, 3, b.y, r.V);
        zy = in ? Vec<T>::get(reinterpret_cast<const T*>(b.z)[b.y]) : NAN;       // a target outside the vocabulary makes its row NaN
      }
      if (live && MODE == MODE_POLICY) {
        adv = a.adv[a.adv_seq ? b.t / r.S : b.t];
        if (a.old_lp) old_lp = a.old_lp[b.t];
        if (a.ref_lp) ref_lp = a.ref_lp[b.t];
      }
      if (live && COUNTED) wt = weight_of(a, b.t, r.S);

      for (unsigned left = b.on; left && ok; left &= left - 1, ++n) {
        if (int(n % PIPE_C) != w) continue;
        const int l = __ffs(left) - 1;
        const long long t = lane_of(b.t, l);
        const unsigned rs = n % PIPE_ROWS, use = n / PIPE_ROWS;
        const Slice s = slice_of<T>(lane_of(b.z, l), r.V, v0, q.vs);
        const T* row = reinterpret_cast<const T*>(s.frame) + s.eoff;
        const float wrow = __shfl_sync(~0u, wt, l);
        float x1 = 0.f, x2 = 0.f, xref = 0.f;      // of a teacher's entries in this slice: sum q (log q - (z - xref) / tau), sum q
        bool bad = false;
        float *tq = nullptr, *tg = nullptr;
        int* tid = nullptr;
        if constexpr (MODE == MODE_DISTILL) {
          tq = entries(w);
          tid = reinterpret_cast<int*>(tq + K4);
          tg = tq + 2 * K4;
          if (GRAD && n >= PIPE_C && !(ok = wait(gdone + w * 8, n / PIPE_C - 1, ST_TIMEOUT_TMEM_EMPTY))) break;      // the entries of its last row are written
          float tm = -INFINITY, ts = 0.f, zm = -INFINITY;
          // two entries of a lane at a time, since the student's logits can be asked for only when the ids are there.  us at 12500 x 32000, one / two / four: 20 entries 310 / 312 /
          // 315, 128 360 / 342 / 339, 256 520 / 466 / 425
          for (int j0 = lane; j0 < K4; j0 += TOP_LOADS * 32) {
            long long y[TOP_LOADS];
            float z[TOP_LOADS], zs[TOP_LOADS], mx = tm;
#pragma unroll
            for (int u = 0; u < TOP_LOADS; ++u) y[u] = j0 + u * 32 < a.K ? ld_idx(a.top_ids, t * a.K + j0 + u * 32, a.idx64) : -1;
#pragma unroll
            for (int u = 0; u < TOP_LOADS; ++u) {
              TFB_BOUNDS(y[u] < r.V, 3, y[u], r.V);
              bad |= y[u] >= r.V;
              if (y[u] < 0 || y[u] >= r.V) y[u] = -1;
              z[u] = y[u] >= 0 ? ld_z(a.top_z, t * a.K + j0 + u * 32, a.top_f32) : -INFINITY;
              const int g = y[u] >= 0 ? int((y[u] + s.eoff) / N) - v0 : -1;
              zs[u] = g >= 0 && g < q.vs ? Vec<T>::get(row[y[u]]) : -INFINITY;
            }
#pragma unroll
            for (int u = 0; u < TOP_LOADS; ++u) {
              mx = fmaxf(mx, z[u]);
              zm = fmaxf(zm, zs[u]);
              if (j0 + u * 32 < K4) {
                tid[j0 + u * 32] = int(y[u]);
                tq[j0 + u * 32] = z[u];
                tg[j0 + u * 32] = zs[u];
              }
            }
            const float ref = mx == -INFINITY ? 0.f : mx;
            ts *= ex2((tm - ref) * k);
#pragma unroll
            for (int u = 0; u < TOP_LOADS; ++u) ts += ex2((z[u] - ref) * k);
            tm = mx;
          }
          warp_join(tm, ts, k);
          zm = warp_max(zm);
          bad = __any_sync(~0u, bad);
          const float tr = tm == -INFINITY ? 0.f : tm, lts = logf(ts);
          xref = zm == -INFINITY ? 0.f : zm;
          for (int j = lane; j < K4; j += 32) {
            const int y = tid[j];
            const float z = tq[j], wq = y >= 0 ? ex2((z - tr) * k) / ts : 0.f;
            const int g = y >= 0 ? int((y + s.eoff) / N) - v0 : -1;
            tq[j] = wq;
            if (g >= 0 && g < q.vs && wq != 0.f) {
              x1 += wq * ((z - tr) * a.inv_tau - lts - (tg[j] - xref) * a.inv_tau);
              x2 += wq;
            }
          }
          x1 = warp_sum(x1);
          x2 = warp_sum(x2);
          if (GRAD) {
            // the weights of each entry's id, before the row's statistics are there: the ring holds fewer than two rows of 50257, so what comes after them is waited for.
            // 7959 x 50257 with 64, 256 and 1024 entries: 332, 402 and 1450 us; after the statistics and without the table 357, 738 and 6340.
            int* seen = tid + 2 * K4;
            for (int i = lane * 4; i < table; i += 128) *reinterpret_cast<int4*>(seen + i) = make_int4(-1, -1, -1, -1);
            __syncwarp();
            bool twice = false;
            for (int j = lane; j < K4; j += 32) {
              const int y = tid[j], g = y >= 0 ? int((y + s.eoff) / N) - v0 : -1;
              if (g < 0 || g >= q.vs) continue;
              twice |= seen_before(seen, table, y);
            }
            if (__any_sync(~0u, twice)) {
              float* sums_of = reinterpret_cast<float*>(seen);
              __syncwarp();
              for (int j = lane; j < K4; j += 32) {
                float back = 0.f;
                for (int i = 0; i < K4; i += 4) {
                  const int4 o = *reinterpret_cast<const int4*>(tid + i);
                  const float4 u = *reinterpret_cast<const float4*>(tq + i);
                  back += o.x == tid[j] ? u.x : 0.f;
                  back += o.y == tid[j] ? u.y : 0.f;
                  back += o.z == tid[j] ? u.z : 0.f;
                  back += o.w == tid[j] ? u.w : 0.f;
                }
                sums_of[j] = back;
              }
              __syncwarp();
              for (int j = lane; j < K4; j += 32) tq[j] = sums_of[j];
            }
          }
        }
        if (!(ok = wait(sdone + rs * 8, use, ST_TIMEOUT_TMEM_FULL))) break;
        const float2 p = lane < SW ? part[rs][lane] : make_float2(-INFINITY, 0.f);
        float M = p.x, S = p.y;
        warp_join(M, S, k);
        // a teacher's terms refer to the slice's maximum from here on
        if (MODE == MODE_DISTILL && x2 != 0.f) x1 += x2 * ((M == -INFINITY ? 0.f : M) - xref) * a.inv_tau;
        if (C > 1) {
          if (lane == 0) mbar_expect_tx(xbar + rs * 8, uint32_t(C) * 16);
          if (lane < C) st_async_v4(map_cta(smem_u32(&xch[rs][rank]), lane), map_cta(xbar + rs * 8, lane), make_float4(M, S, x1, x2));
          if (!(ok = wait(xbar + rs * 8, use, ST_TIMEOUT_FLAG))) break;
          const float4 o = lane < C ? xch[rs][lane] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
          M = o.x;
          S = o.y;
          warp_join(M, S, k);
          if (MODE == MODE_DISTILL) {
            x1 = warp_sum(o.w != 0.f ? o.z + o.w * (M - (o.x == -INFINITY ? 0.f : o.x)) * a.inv_tau : o.z);
            x2 = warp_sum(o.w);
          }
        }
        const float Mr = M == -INFINITY ? 0.f : M;
        const double ls = log64(S);
        float scale = 0.f, hot = 0.f;
        if constexpr (MODE == MODE_DISTILL) {
          const float wk = bad ? NAN : wrow;
          hot = a.tau * wk;
          scale = hot / S;
          if (rank == 0 && lane == 0) {
            const float kl = bad ? NAN : x1 + x2 * float(ls);
            a.logp[t] = kl;
            sums[0] += double(kl * a.tau * a.tau * wk);
          }
          if (GRAD) {
            // the entries' own gradients, each from its value of z; the gradient warps store them over what their vectors have written
            for (int j = lane; j < K4; j += 32) tg[j] = scale * ex2((tg[j] - Mr) * k) - hot * tq[j];
            __syncwarp();
          }
        } else {
          const float z = __shfl_sync(~0u, zy, l);
          const double lp = double(z) - double(M) - ls;
          if (rank == 0 && lane == 0) {
            if constexpr (MODE == MODE_SCORE) {
              const long long y = ld_idx(a.targets, t, a.idx64);
              put_score(a, t, y >= 0 && y < r.V, M, S);
            } else {
              put_stats<MODE>(a, r.T, t, M, ls, lp);
            }
          }
          if constexpr (MODE == MODE_POLICY) {
            float loss, kl, clipped, g;
            const double from = a.old_lp ? double(__shfl_sync(~0u, old_lp, l)) : lp;
            policy_terms(a, float(lp), float(lp - from),
                         a.ref_lp ? float(double(__shfl_sync(~0u, ref_lp, l)) - lp) : 0.f, __shfl_sync(~0u, adv, l), loss, kl, clipped, g);
            hot = wrow * g;
            scale = -hot / S;
            sums[0] += double(wrow * loss);
            sums[1] += double(wrow * kl);
            sums[2] += double(wrow * clipped);
          }
        }
        if (lane == 0) {
          coef[rs] = make_float4(Mr, scale, hot, 0.f);
          mbar_arrive(cready + rs * 8);
        }
      }
    }
    if (lane == 0)
      for (int j = 0; j < 3; ++j) acc[w][j] = sums[j];
  } else if (GRAD) {
    // ------------------------------ gradient ------------------------------
    const int gw = warp - PIPE_S;
    unsigned n = 0;
    Cursor c;
    bool ok = true;
    for (long long base = 0; base < nrows && ok; base += 32) {
      const RowBlock b = rows_from(base);
      for (int l = 0; l < 32 && ((b.valid >> l) & 1u) && ok; ++l) {
        const Slice s = slice_of<T>(lane_of(b.z, l), r.V, v0, q.vs);
        char* dst = reinterpret_cast<char*>(lane_of(b.d, l)) - s.eoff * ES;      // the gradient's rows start at the same place of a vector
        T* out = reinterpret_cast<T*>(dst) + s.eoff;
        auto store = [&](int g, const float (&f)[N]) {
          if (g >= s.fv && g < s.lv) {
            *reinterpret_cast<uint4*>(dst + (long long)g * 16) = Vec<T>::pack(f);
          } else {
            const long long x0 = (long long)g * N - s.eoff;
#pragma unroll
            for (int x = 0; x < N; ++x)
              if (x0 + x >= 0 && x0 + x < r.V) out[x0 + x] = Vec<T>::put(f[x]);
          }
        };
        if (!((b.on >> l) & 1u)) {
          float f[N] = {};
          for (int v = gw * 32 + lane; v < s.n; v += PIPE_G * 32) store(v0 + v, f);
          continue;
        }
        const unsigned rs = n % PIPE_ROWS, first = c.slot % PIPE_GG;      // group that has the slice's first chunk
        if (!(ok = wait(cready + rs * 8, n / PIPE_ROWS, ST_TIMEOUT_TMEM_FULL))) break;
        const float4 cf = coef[rs];
        const float2 neg = make_float2(-cf.x, -cf.x), k2 = make_float2(k, k), sc = make_float2(cf.y, cf.y);
        const long long y = lane_of(b.y, l);
        const int gy = MODE == MODE_DISTILL || y < 0 || y >= r.V ? -1 : int((y + s.eoff) / N), ey = int((y + s.eoff) % N);
        auto values = [&](float (&f)[N]) {
#pragma unroll
          for (int x = 0; x < N; x += 2) {
            const float2 d = mul2(add2(make_float2(f[x], f[x + 1]), neg), k2), e = mul2(make_float2(ex2(d.x), ex2(d.y)), sc);
            f[x] = e.x;
            f[x + 1] = e.y;
          }
        };
        for (int c0 = 0; c0 < s.n; c0 += CHUNK_VECS, c.next(NCH)) {
          if (int(c.slot % PIPE_GG) != gw / PIPE_W) continue;
          if (!(ok = wait(full + c.slot * 8, c.use, ST_TIMEOUT_FULL))) break;      // (it has landed; this makes it visible here)
#pragma unroll 1
          for (int h = 0; h < HALVES; ++h) {
          const int w0 = (h * PIPE_W + gw % PIPE_W) * LV * 32, g0 = v0 + c0 + w0;
          const uint4* src = reinterpret_cast<const uint4*>(dyn + c.slot * CHUNK_BYTES) + w0 + lane;
          if (g0 >= s.fv && g0 + LV * 32 <= min(s.lv, v0 + s.n) && (gy < g0 || gy >= g0 + LV * 32)) {
            uint4* to = reinterpret_cast<uint4*>(dst) + g0 + lane;
            float f[LV][N];
#pragma unroll
            for (int j = 0; j < LV; ++j) Vec<T>::unpack(src[j * 32], f[j]);
#pragma unroll
            for (int j = 0; j < LV; ++j) {
              values(f[j]);
              to[j * 32] = Vec<T>::pack(f[j]);
            }
          } else {
            for (int j = 0; j < LV; ++j) {
              const int g = g0 + j * 32 + lane;
              if (g >= v0 + s.n) continue;
              float f[N];
              Vec<T>::unpack(src[j * 32], f);
              values(f);
              if (g == gy) {
#pragma unroll
                for (int x = 0; x < N; ++x)
                  if (x == ey) f[x] += cf.z;
              }
              store(g, f);
            }
          }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(empty + c.slot * 8);
        }
        if (!ok) break;
        if constexpr (MODE == MODE_DISTILL) {
          // every warp those of the vectors that it has stored itself
          __syncwarp();
          const float* tq = entries(n % PIPE_C);
          const int* tid = reinterpret_cast<const int*>(tq + K4);
          for (int j = lane; j < K4; j += 32) {
            const int yj = tid[j], g = yj >= 0 ? int((yj + s.eoff) / N) - v0 : -1;
            if (g >= 0 && g < q.vs && int((first + g / CHUNK_VECS) % PIPE_GG * PIPE_W + g / (LV * 32) % PIPE_W) == gw) out[yj] = Vec<T>::put(tq[2 * K4 + j]);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(gdone + (n % PIPE_C) * 8);
        }
        ++n;
      }
    }
  }
  __syncthreads();
  if (q.nsums && rank == 0 && warp == 0) {
    tfb::pdl_wait();
    int last = 0;
    if (lane == 0) {
      for (int j = 0; j < q.nsums; ++j) {
        double v = 0.0;
        for (int w = 0; w < PIPE_C; ++w) v += acc[w][j];
        q.partial[cl * 3 + j] = v;
      }
      __threadfence();
      last = atomicAdd(q.counter, 1) == q.clusters - 1;
    }
    if (__shfl_sync(~0u, last, 0)) {
      __threadfence();
      for (int j = 0; j < q.nsums; ++j) {
        double v = 0.0;
        for (int c = lane; c < q.clusters; c += 32) v += __ldcg(q.partial + c * 3 + j);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
        if (lane == 0) q.out[j] = float(v);
      }
    }
  }
  if (C > 1) cluster_sync();           // no block leaves while another may still store into its shared memory
}

// denom[0] = number of rows that count (at least 1), or denom[i] = that of sequence i.  `stride`: distance between the indices that say so (targets: 1,
// a teacher's ids: K); a row counts where its index is not `ignore` (targets) or not negative (first id).  Clears *zero; without idx nothing else.
__global__ void __launch_bounds__(1024) row_count_kernel(const void* idx, int idx64, long long stride, long long ignore, int negative, int N, int S, int per_seq,
                                                         float* denom, int* zero) {
  tfb::pdl_sync();
  __shared__ int sh[32];
  if (blockIdx.x == 0 && threadIdx.x == 0) *zero = 0;
  if (!idx) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto counts = [&](long long t) {
    const long long y = ld_idx(idx, t * stride, idx64);
    return negative ? y >= 0 : y != ignore;
  };
  if (per_seq) {
    for (int n = blockIdx.x * 32 + warp; n < N; n += gridDim.x * 32) {
      int c = 0;
#pragma unroll 8
      for (int i = lane; i < S; i += 32) c += counts((long long)n * S + i);
      c = __reduce_add_sync(~0u, c);
      if (lane == 0) denom[n] = float(max(c, 1));
    }
    return;
  }
  int c = 0;
#pragma unroll 8
  for (int t = threadIdx.x; t < N * S; t += 1024) c += counts(t);
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

// out[i] = sum of terms[i * T ...], i < n <= 3, in 64 bits and always in the same order: every block a share of the rows, the block that ends last the shares.
constexpr int TERM_BLOCKS = 32;
__global__ void __launch_bounds__(512) term_sum_kernel(const float* terms, int T, int n, double* partial, int* counter, float* out) {
  tfb::pdl_sync();
  __shared__ double sh[32];
  __shared__ int last;
  const int share = (T + gridDim.x - 1) / gridDim.x, t0 = blockIdx.x * share, t1 = min(T, t0 + share);
  for (int i = 0; i < n; ++i) {
    double v = 0.0;
#pragma unroll 4
    for (int t = t0 + threadIdx.x; t < t1; t += 512) v += double(terms[(long long)i * T + t]);
    v = block_sum(v, sh);
    if (threadIdx.x == 0) partial[blockIdx.x * 3 + i] = v;
  }
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(counter, 1) == int(gridDim.x) - 1;
  }
  __syncthreads();
  if (!last || threadIdx.x >= n) return;
  __threadfence();
  double v = 0.0;
  for (int b = 0; b < int(gridDim.x); ++b) v += __ldcg(partial + b * 3 + threadIdx.x);
  out[threadIdx.x] = float(v);
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
  float* loss;
  int* counter;                        // 0 before the launch
};
// the block that ends last adds up the pairs' terms, always in the same order
__device__ void pair_mean(const PairArg& a, double* sh) {
  __shared__ int last;
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(a.counter, 1) == a.N - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double v = 0.0;
  for (int n = threadIdx.x; n < a.N; n += 512) v += double(__ldcg(a.terms + n));
  v = block_sum(v, sh);
  if (threadIdx.x == 0) *a.loss = float(v);
}

__global__ void __launch_bounds__(512) pair_kernel(const PairArg a) {
  tfb::pdl_sync();
  __shared__ double sh[32];
  __shared__ int count[16];
  const int n = blockIdx.x;
  // half of the block to either answer; its sum in 64 bits, in a fixed order
  const int side = threadIdx.x >> 8, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  {
    const long long t0 = (long long)(n + side * a.N) * a.S;
    double v = 0.0;
    int c = 0;
#pragma unroll 4
    for (int i = threadIdx.x & 255; i < a.S; i += 256) {
      v += a.lp[t0 + i];
      c += ld_idx(a.targets, t0 + i, a.idx64) != a.ignore;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    c = __reduce_add_sync(~0u, c);
    if (lane == 0) {
      sh[warp] = v;
      count[warp] = c;
    }
  }
  __syncthreads();
  double L[2], cnt[2];
  if (threadIdx.x == 0)
    for (int h = 0; h < 2; ++h) {
      L[h] = 0.0;
      int c = 0;
      for (int i = 0; i < 8; ++i) {
        L[h] += sh[h * 8 + i];
        c += count[h * 8 + i];
      }
      cnt[h] = a.average ? double(max(1, c)) : 1.0;
      L[h] /= cnt[h];
    }
  if (threadIdx.x == 0) {
    const double h = (L[0] - (a.ref ? double(a.ref[n]) : 0.0)) - (L[1] - (a.ref ? double(a.ref[a.N + n]) : 0.0));
    const double x = double(a.beta) * h;
    double l, dl;                        // of h
    if (a.kind == 0) {
      const double e = exp(-fabs(x)), sneg = x >= 0 ? e / (1.0 + e) : 1.0 / (1.0 + e);      // sigmoid(-x)
      l = log1p(e) + fmax(-x, 0.0);           // -(1 - s) log sig(x) - s log sig(-x)
      if (a.smooth != 0.f) l += double(a.smooth) * x;      // (x may be infinite)
      if (x != x) l = x;
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
  pair_mean(a, sh);
}

// The general form's launch.
template <class T, int MODE>
static void launch_rows_t(const RowsArg& r, const LossArg& a, bool warp, bool pdl, cudaStream_t st) {
  const size_t smem = MODE == MODE_DISTILL ? size_t(2 * a.K + row_table(warp, a.K)) * 4 : 0;
  if (warp) return tfb::launch_attr(pdl, row_loss_kernel<T, MODE, true>, (r.T + WARP_ROWS - 1) / WARP_ROWS, WARP_ROWS * 32, smem * WARP_ROWS, st, r, a);
  LossArg q = a;
  if (MODE == MODE_GRAD) {
    // Few rows: several blocks to one, up to two waves of the four that an SM holds, two vectors to a thread at least.  us, so / a block to a row: 10 x 128256
    // 3.6 / 13.7, 61 x 128256 8.9 / 14.4, 200 x 32000 7.3 / 6.9; with more waves the blocks' starts show (1280 x 32000 37 / 35, 1400 x 50257 59 / 56).
    const int blocks = 2 * 4 * sm_count(), most = r.V / (Vec<T>::N * ROW_THREADS * 2);
    q.split = max(1, min((blocks + r.T - 1) / r.T, most));
  }
  tfb::launch_attr(pdl, row_loss_kernel<T, MODE, false>, r.T * max(1, q.split), ROW_THREADS, smem, st, r, q);
}
// `behind_small`: the kernel before is a small one of this file, so that early-placed blocks take no room from it (see PDL_ROWS otherwise)
template <int MODE>
static int launch_rows(const RowsArg& r, const LossArg& a, bool warp, bool behind_small, cudaStream_t st) {
  const bool pdl = pdl_mode() == 2 || (pdl_mode() == 1 && (behind_small || r.T <= PDL_ROWS));
  if constexpr (MODE == MODE_SCORE) launch_rows_t<float, MODE>(r, a, warp, pdl, st);
  else if (r.f32) launch_rows_t<float, MODE>(r, a, warp, pdl, st);
  else launch_rows_t<__nv_bfloat16, MODE>(r, a, warp, pdl, st);
  return int(cudaGetLastError());
}

// Rows for a warp each: the pipelined form takes 1.3 us for a row however short, per SM.  us of the policy loss, warps / that form: 50000 rows of 520 bytes 58 / 409, of 8 KB
// 240 / 409, of 16 KB 509 / 424; 2000 rows of 520 bytes 10.9 / 26, of 8 KB 20 / 26, of 16 KB 30 / 27; 96 rows of 2 KB 8.5 / 9.6, of 4 KB 10.5 / 9.6, of 8 KB 13.3 / 9.9.
static bool short_rows(const RowsArg& r, const LossArg& a) {
  const long long bytes = r.V * (r.f32 ? 4ll : 2ll);
  return a.K <= WARP_TOP && bytes <= (r.T >= 1024 ? 8192 : 2048);
}

// Clusters of C blocks of a kernel that the device holds at a time (0: none; negative: -cudaError_t).  One entry per thread, kernel and size of cluster, since a run repeats its
// shapes.
template <class T, int MODE, bool GRAD>
static int resident_clusters(int C, int smem) {
  struct Entry { int dev, smem, n; };
  static thread_local Entry entries[4] = {{-1}, {-1}, {-1}, {-1}};      // C = 1, 2, 4, 8
  auto kern = row_pipe_kernel<T, MODE, GRAD>;
  constexpr int threads = PIPE_WARPS * 32;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  Entry& e = entries[C == 1 ? 0 : C == 2 ? 1 : C == 4 ? 2 : 3];
  if (e.dev == dev && e.smem == smem) return e.n;
  int n = 0;
  if (C == 1) {
    if (cudaError_t err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem)) return -int(err);
    n *= sm_count();
  } else {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.gridDim = C; cfg.blockDim = threads; cfg.dynamicSmemBytes = smem; cfg.attrs = at; cfg.numAttrs = 1;
    if (cudaError_t err = cudaOccupancyMaxActiveClusters(&n, kern, &cfg)) return -int(err);
  }
  e = {dev, smem, n};
  return n;
}

template <class T, int MODE, bool GRAD>
static int launch_pipe_t(const RowsArg& r, const LossArg& a, PipeArg q, long long nvec, cudaStream_t st) {
  static DeviceOnce once;
  auto kern = row_pipe_kernel<T, MODE, GRAD>;
  constexpr int most = 212 << 10;
  // The smallest cluster whose slices are two thirds of the ring, so that the next row's copies go on while a row is finished; larger ones
  // exchange more and leave SMs without a block (33 clusters of 4, 15 of 8, fit on 148 SMs): 3125 x 128256, 4.0 TB/s with 8, 4.9 with 4, 5.0 with 2 (without a gradient
  // 3.2, 4.1, 5.2), 7959 x 50257 3.1 with 4, 4.1 with 2, 5.0 with 1.  Then larger ones while rows are too few to fill the machine.
  const int extra = MODE == MODE_DISTILL ? PIPE_C * (3 * ((a.K + 3) & ~3) + (GRAD ? top_table(a.K) : 0)) * 4 : 0;
  q.chunks = min(PIPE_CHUNKS, (most - extra) / CHUNK_BYTES / (PIPE_SG + PIPE_GG) * (PIPE_SG + PIPE_GG));
  const int slice = q.chunks * 2 / 3 * CHUNK_VECS;
  int C = 1;
  while (C < 8 && (nvec + C - 1) / C > slice) C *= 2;
  if ((nvec + C - 1) / C > slice) return TFB_NOT_TAKEN;
  while (C < 8 && (long long)r.T * C * 2 <= sm_count() && nvec / (2 * C) >= 256) C *= 2;
  q.csize = C;
  q.vs = int((nvec + C - 1) / C);
  const int smem = q.chunks * CHUNK_BYTES + extra;
  if (int e = ensure_dyn_smem(once, kern, most)) return e;
  const int n = resident_clusters<T, MODE, GRAD>(C, smem);
  if (n < 0) return -n;
  if (n == 0) return TFB_NOT_TAKEN;
  q.clusters = min(min(n, PIPE_CLUSTERS), r.T);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.gridDim = q.clusters * C; cfg.blockDim = PIPE_WARPS * 32; cfg.dynamicSmemBytes = smem; cfg.stream = st; cfg.attrs = at;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = pdl_mode() == 2 || (pdl_mode() == 1 && (MODE != MODE_STATS || r.T <= PDL_ROWS));
  cfg.numAttrs = 1;
  if (C > 1) {
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = C; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  (void)cudaLaunchKernelEx(&cfg, kern, r, a, q);
  return int(cudaGetLastError());
}

// The pipelined form where it applies: rows of logits and gradient that start at the same place of a 16-byte vector.
template <int MODE>
static int launch_pipe(const RowsArg& r, const LossArg& a, const PipeArg& q, cudaStream_t st) {
  const int es = r.f32 ? 4 : 2, B = r.T / r.S;
  const uintptr_t z = reinterpret_cast<uintptr_t>(r.z), d = reinterpret_cast<uintptr_t>(r.dz);
  if (r.dz && (((z ^ d) & 15) || (B > 1 && (r.zb - r.db) * es % 16) || (r.S > 1 && (r.zs - r.ds) * es % 16))) return TFB_NOT_TAKEN;
  const bool whole = (z & 15) == 0 && (B == 1 || r.zb * es % 16 == 0) && (r.S == 1 || r.zs * es % 16 == 0);
  const long long bytes = (long long)r.V * es, nvec = whole ? (bytes + 15) / 16 : (bytes + 30) / 16;
  if constexpr (MODE == MODE_SCORE) {
    return launch_pipe_t<float, MODE, false>(r, a, q, nvec, st);
  } else {
    if (r.dz) return r.f32 ? launch_pipe_t<float, MODE, MODE != MODE_STATS>(r, a, q, nvec, st) : launch_pipe_t<__nv_bfloat16, MODE, MODE != MODE_STATS>(r, a, q, nvec, st);
    return r.f32 ? launch_pipe_t<float, MODE, false>(r, a, q, nvec, st) : launch_pipe_t<__nv_bfloat16, MODE, false>(r, a, q, nvec, st);
  }
}

// One of the two, and the sums over the rows: out[i], i < nsums.  ws: the workspace of either form (terms or the clusters' sums); *counter is 0.
template <int MODE>
static int rows_and_sums(const RowsArg& r, LossArg a, int nsums, void* ws, int* counter, float* out, cudaStream_t st) {
  PipeArg q = {};
  q.nsums = nsums; q.partial = static_cast<double*>(ws); q.counter = counter; q.out = out;
  const bool warp = short_rows(r, a);
  int rc = warp ? TFB_NOT_TAKEN : launch_pipe<MODE>(r, a, q, st);
  if (rc != TFB_NOT_TAKEN) return rc;
  a.terms = reinterpret_cast<float*>(static_cast<double*>(ws) + 3 * TERM_BLOCKS);
  rc = launch_rows<MODE>(r, a, warp, MODE != MODE_STATS, st);
  if (rc || !nsums) return rc;
  double* partial = static_cast<double*>(ws);                     // in front of the terms
  const int blocks = min(TERM_BLOCKS, (r.T + 2047) / 2048);
  tfb::launch_k_pdl(term_sum_kernel, blocks, 512, 0, st, a.terms, r.T, nsums, partial, counter, out);
  return int(cudaGetLastError());
}

int row_scores(const float* z, long long ldz, int T, int V, const void* targets, int idx64, long long ignore, const float* zy, float* logp, float* lse, int* status,
               void* stream) {
  RowsArg r = {};
  r.z = z; r.zs = ldz; r.T = r.S = T; r.V = V; r.f32 = 1; r.status = status;
  LossArg a = {};
  a.targets = targets; a.idx64 = idx64; a.ignore = ignore; a.zy = zy; a.logp = logp; a.lse = lse;
  return rows_and_sums<MODE_SCORE>(r, a, 0, nullptr, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

static bool bad_rows(const RowsArg& r) { return !r.z || r.T <= 0 || r.S <= 0 || r.V <= 0 || r.T % r.S; }

}  // namespace tfb

using namespace tfb;

// logp [T], stats [2, T]; 0 where the target is `ignore`.
TFB_API int tfb_token_logprobs(const RowsArg* r, const void* targets, int idx64, long long ignore, float* logp, float* stats, void* stream) {
  if (!r || bad_rows(*r) || !targets || !logp || !stats) return TFB_ERR_ARG;
  LossArg a = {};
  a.targets = targets; a.idx64 = idx64; a.ignore = ignore;
  a.logp = logp; a.stats = stats;
  RowsArg rows = *r;
  rows.dz = nullptr;
  return rows_and_sums<MODE_STATS>(rows, a, 0, nullptr, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

// dz = dlogp (onehot(target) - softmax z)
TFB_API int tfb_token_logprobs_bwd(const RowsArg* r, const void* targets, int idx64, long long ignore, const float* stats, const float* dlogp, void* stream) {
  if (!r || bad_rows(*r) || !targets || !stats || !dlogp || !r->dz) return TFB_ERR_ARG;
  LossArg a = {};
  a.targets = targets; a.idx64 = idx64; a.ignore = ignore;
  a.stats = const_cast<float*>(stats); a.dlogp = dlogp;
  return launch_rows<MODE_GRAD>(*r, a, short_rows(*r, a), false, static_cast<cudaStream_t>(stream));
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
  void* ws;                            // 24 PIPE_CLUSTERS + 12 T bytes, aligned to 8
  float* denom;                        // workspace: [max(1, T / S)], and
  int* counter;                        // one word
};
TFB_API int tfb_policy_loss(const RowsArg* r, const PolicyArg* p, void* stream) {
  if (!r || !p || bad_rows(*r) || !p->targets || !p->adv || !p->logp || !p->out || !p->ws || !p->denom || !p->counter) return TFB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int N = r->T / r->S;
  LossArg a = {};
  a.targets = p->targets; a.idx64 = p->idx64; a.ignore = p->ignore;
  a.logp = p->logp; a.adv = p->adv; a.old_lp = p->old_lp; a.ref_lp = p->ref_lp;
  a.adv_seq = p->adv_seq; a.ratio = p->ratio; a.kl_kind = p->kl_kind;
  a.lo = p->lo; a.hi = p->hi; a.kl_coef = p->kl_coef;
  a.mean = p->mean; a.scale = p->mean == MEAN_SEQUENCES ? float(N) : 1.f;
  a.denom = p->n_valid && p->mean == MEAN_TOKENS ? p->n_valid : p->denom;
  const bool count = a.denom == p->denom && p->mean != MEAN_SUM;
  const int seq = p->mean == MEAN_SEQUENCES;
  tfb::launch_k_rows(r->T, row_count_kernel, seq ? (N + 31) / 32 : 1, 1024, 0, st, count ? p->targets : nullptr, p->idx64, 1ll, p->ignore, 0, N, r->S, seq, p->denom,
                     p->counter);
  return rows_and_sums<MODE_POLICY>(*r, a, 3, p->ws, p->counter, p->out, st);
}

struct PreferenceArg {
  const void* targets;
  int idx64;
  long long ignore;
  const float* ref;
  int kind, average;
  float beta, smooth;
  float *loss, *margins, *logp;        // [1], [N], [2N]
  double* lp64;                        // workspace: [T], [2, T], [2N], [N], one word
  float *stats, *coef, *terms;
  int* counter;
};
TFB_API int tfb_preference_loss(const RowsArg* r, const PreferenceArg* p, void* stream) {
  if (!r || !p || bad_rows(*r) || (r->T / r->S) % 2 || !p->targets || !p->loss || !p->margins || !p->logp || !p->lp64 || !p->stats || !p->coef || !p->terms ||
      !p->counter)
    return TFB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LossArg a = {};
  a.targets = p->targets; a.idx64 = p->idx64; a.ignore = p->ignore;
  a.stats = p->stats; a.logp64 = p->lp64; a.zero = p->counter;
  RowsArg rows = *r;
  rows.dz = nullptr;
  if (int rc = rows_and_sums<MODE_STATS>(rows, a, 0, nullptr, nullptr, nullptr, st)) return rc;
  PairArg q = {p->lp64, p->targets, p->idx64, p->ignore, p->ref, r->T / r->S / 2, r->S, p->kind, p->average, p->beta, p->smooth, p->logp, p->margins, p->coef, p->terms,
               p->loss, p->counter};
  tfb::launch_k_pdl(pair_kernel, q.N, 512, 0, st, q);
  if (!r->dz) return int(cudaGetLastError());
  a.dlogp = p->coef; a.per_seq = 1; a.logp64 = nullptr; a.zero = nullptr;
  return launch_rows<MODE_GRAD>(*r, a, short_rows(*r, a), true, st);
}

struct DistillArg {
  const void *top_ids, *top_z;
  int idx64, top_f32, K;
  float tau;
  const float* n_valid;
  float *kl, *loss;                    // [T], [1]
  void* ws;                            // 24 PIPE_CLUSTERS + 4 T bytes, aligned to 8
  float* denom;                        // workspace: one value, and
  int* counter;                        // one word
};
TFB_API int tfb_distill_loss(const RowsArg* r, const DistillArg* p, void* stream) {
  if (!r || !p || bad_rows(*r) || !p->top_ids || !p->top_z || p->K <= 0 || !(p->tau > 0.f) || !p->kl || !p->loss || !p->ws || !p->denom || !p->counter)
    return TFB_ERR_ARG;
  if (p->K > TL_MAX_TOP) return TFB_ERR_LIMIT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  LossArg a = {};
  a.idx64 = p->idx64; a.logp = p->kl; a.top_ids = p->top_ids; a.top_z = p->top_z; a.K = p->K; a.top_f32 = p->top_f32;
  a.tau = p->tau; a.inv_tau = 1.f / p->tau;
  a.mean = MEAN_TOKENS; a.scale = 1.f; a.denom = p->n_valid ? p->n_valid : p->denom;
  tfb::launch_k_rows(r->T, row_count_kernel, 1, 1024, 0, st, p->n_valid ? nullptr : p->top_ids, p->idx64, (long long)p->K, 0ll, 1, 1, r->T, 0, p->denom, p->counter);
  return rows_and_sums<MODE_DISTILL>(*r, a, 1, p->ws, p->counter, p->loss, st);
}
