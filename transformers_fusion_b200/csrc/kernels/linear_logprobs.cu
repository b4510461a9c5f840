// Log-probabilities of given tokens under a head, from hidden states: lp = x . w[y] - log sum_v exp(x . w[v]), without the [T, V] logits of many rows in
// memory.
//
//   gather   rows that are scored, one behind the other: a prompt's rows take no part in the product
//   product  x W^T on tensor cores (gemm_bf16.cu), whose epilogue keeps (m, sum exp) of every row's columns in half a tile, the target's left out, and drops the rest
//   finish   joins a row's parts, takes the product with its target's row of W by itself, in 32-bit fused multiply-adds, and puts the two together
//
// The target's column is left out of the sum because its logit there is another rounding of the same number: the tensor cores' accumulation is off by a few 2^-24 of the
// partial sums at each of its steps, in one direction (relative error of lp at 4096 terms 1.3e-6 with their value, 2.6e-7 with the multiply-adds').  Where the
// target is most of the sum the difference of the two would be all of lp; so it is the other columns' share that lp is computed from (score_of).
// Few rows (see below) are not gathered: their logits, the rows that are not scored among them, stand in a workspace.
#include "row_losses.cuh"
#include "tfb_host.h"

TFB_BOUNDS_DEFINE(linear_logprobs)

namespace tfb {

struct ScoreArg {
  const __nv_bfloat16 *x, *w;
  long long ldx, ldw;
  const void* targets;
  int idx64;
  long long ignore;
  int M, V, H;
  float *logp, *lse;                   // [M]
  int* rows;                           // one word: rows that are scored
  int *row_of, *col_of;                // [M]: place of a scored row, and its target (-1 outside the vocabulary)
  __nv_bfloat16* xc;                   // [M, ldc]: their hidden states
  long long ldc;
  float2* part;                        // [2 ceil(V / 128), M]
  int parts;                           // of a row; set by the launch
  float* z;                            // few rows, else null: [M, ldz] logits, ldz a multiple of 4
  long long ldz;
  float* zy;                           // few rows: [M] the targets' logits
};

constexpr int GATHER_MOST = 1024;    // rows of a block

// Every block takes `per_block` rows and counts those that are scored before them by itself (the targets of a launch are 256 KB at most), so rows keep
// their order and no counter has to be cleared by a launch of its own.
__global__ void __launch_bounds__(1024) score_gather_kernel(const ScoreArg a, const int per_block) {
  tfb::pdl_sync();
  __shared__ int place[GATHER_MOST], sums[32], count[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r0 = blockIdx.x * per_block, n = min(per_block, a.M - r0);
  int before = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < r0; i += 1024) before += ld_idx(a.targets, i, a.idx64) != a.ignore;
  const bool mine = int(threadIdx.x) < n;
  const long long y = mine ? ld_idx(a.targets, r0 + threadIdx.x, a.idx64) : a.ignore;
  const bool on = y != a.ignore;
  const unsigned mask = __ballot_sync(~0u, on);
  before = __reduce_add_sync(~0u, before);
  if (lane == 0) {
    sums[warp] = before;
    count[warp] = __popc(mask);
  }
  __syncthreads();
  const int c = count[lane], all = __reduce_add_sync(~0u, c), base = __reduce_add_sync(~0u, sums[lane]);
  const int at = base + __reduce_add_sync(~0u, lane < warp ? c : 0) + __popc(mask & ((1u << lane) - 1));
  if (mine) {
    place[threadIdx.x] = on ? at : -1;
    if (on) {
      a.row_of[at] = r0 + threadIdx.x;
      a.col_of[at] = y >= 0 && y < a.V ? int(y) : -1;
    } else {
      a.logp[r0 + threadIdx.x] = a.lse[r0 + threadIdx.x] = 0.f;
    }
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) *a.rows = base + all;
  __syncthreads();
  // a warp takes pieces of a row, four vectors to a lane
  const int vecs = a.H / 8, pieces = (vecs + 127) / 128;
  for (int i = warp; i < n * pieces; i += 32) {
    const int row = i / pieces, v = (i - row * pieces) * 128 + lane, to = place[row];
    if (to < 0) continue;
    const uint4* src = reinterpret_cast<const uint4*>(a.x + (r0 + row) * a.ldx) + v;
    uint4* dst = reinterpret_cast<uint4*>(a.xc + to * a.ldc) + v;
    uint4 w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (v + u * 32 < vecs) w[u] = src[u * 32];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (v + u * 32 < vecs) dst[u * 32] = w[u];
  }
}

// A thread's share of x[row] . w[y], y in the vocabulary.
__device__ __forceinline__ float target_logit(const ScoreArg& a, long long row, long long y, int tid, int nt) {
  const uint4 *p = reinterpret_cast<const uint4*>(a.x + row * a.ldx), *q = reinterpret_cast<const uint4*>(a.w + y * a.ldw);
  float2 t = make_float2(0.f, 0.f), u = t;
#pragma unroll 8
  for (int v = tid; v < a.H / 8; v += nt) {
    const uint4 f = p[v], g = q[v];
    t = fma2(unpack_bf16(f.x), unpack_bf16(g.x), t);
    u = fma2(unpack_bf16(f.y), unpack_bf16(g.y), u);
    t = fma2(unpack_bf16(f.z), unpack_bf16(g.z), t);
    u = fma2(unpack_bf16(f.w), unpack_bf16(g.w), u);
  }
  return (t.x + u.x) + (t.y + u.y);
}

// Eight rows to a block (two sectors of a part's entries), 32 threads to a row's parts with eight loads under way in each: a row of a vocabulary of 128256 has 1002 or 2004
// parts, and one by one they take sixteen threads 75 us.
__global__ void __launch_bounds__(256) score_finish_kernel(const ScoreArg a) {
  tfb::pdl_sync();
  constexpr int R = 8, SHARES = 256 / R, U = 8;
  const int n = *a.rows, r0 = blockIdx.x * R;
  if (r0 >= n) return;
  __shared__ float2 sh[SHARES][R];
  __shared__ float zy[R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  {
    const int i = threadIdx.x % R, share = threadIdx.x / R, at = min(r0 + i, n - 1);
    float m = -INFINITY, s = 0.f;
    for (int p = share; p < a.parts; p += SHARES * U) {
      float2 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = p + u * SHARES < a.parts ? a.part[(long long)(p + u * SHARES) * a.M + at] : make_float2(-INFINITY, 0.f);
      float M = m;
#pragma unroll
      for (int u = 0; u < U; ++u) M = fmaxf(M, v[u].x);
      const float r = M == -INFINITY ? 0.f : M;
      s *= ex2((m - r) * LOG2E);
#pragma unroll
      for (int u = 0; u < U; ++u) s += v[u].y * ex2((v[u].x - r) * LOG2E);
      m = M;
    }
    sh[share][i] = make_float2(m, s);
  }
  for (int i = warp; i < R && r0 + i < n; i += 8) {
    const int y = a.col_of[r0 + i], row = a.row_of[r0 + i];
    if (lane == 0) TFB_BOUNDS(y >= 0, 3, y, a.V);
    const float z = y >= 0 ? warp_sum(target_logit(a, row, y, lane, 32)) : 0.f;
    if (lane == 0) zy[i] = z;
  }
  __syncthreads();
  // one warp to a row: its shares in 64 bits
  for (int i = warp; i < R && r0 + i < n; i += 8) {
    float m = -INFINITY;
    for (int j = lane; j < SHARES; j += 32) m = fmaxf(m, sh[j][i].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    const float r = m == -INFINITY ? 0.f : m;
    double s = 0.0;
    for (int j = lane; j < SHARES; j += 32) s += double(sh[j][i].y * ex2((sh[j][i].x - r) * LOG2E));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (lane) continue;
    const int row = a.row_of[r0 + i];
    score_of(m, s, zy[i], a.col_of[r0 + i] >= 0, a.logp[row], a.lse[row]);
  }
}

// Few rows, whose logits are there: the target's own, and its column out of the row's statistics.  A block to a row.
__global__ void __launch_bounds__(128) score_target_kernel(const ScoreArg a) {
  tfb::pdl_sync();
  __shared__ float sh[4];
  const int row = blockIdx.x;
  const long long y = ld_idx(a.targets, row, a.idx64);
  if (y == a.ignore) return;
  const bool in = y >= 0 && y < a.V;
  if (threadIdx.x == 0) TFB_BOUNDS(in, 3, y, a.V);
  if (!in) return;
  const float z = warp_sum(target_logit(a, row, y, threadIdx.x, 128));
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = z;
  __syncthreads();
  if (threadIdx.x) return;
  a.zy[row] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
  a.z[row * a.ldz + y] = -INFINITY;
}

}  // namespace tfb

using namespace tfb;

// x [M, H] and w [V, H] bf16, pitches multiples of 8, 16-byte aligned; H a multiple of 8.  Writes all of the workspace that it reads.
TFB_API int tfb_linear_logprobs(const ScoreArg* p, int* status, void* stream) {
  if (!p || !p->x || !p->w || !p->targets || !p->logp || !p->lse || !p->rows || !p->row_of || !p->col_of || !p->xc || !p->part || p->M <= 0 || p->V <= 0 || p->H <= 0 || p->H % 8 ||
      p->ldx % 8 || p->ldw % 8 || p->ldc % 8 || ((reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(p->w) | reinterpret_cast<uintptr_t>(p->xc)) & 15))
    return TFB_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Few rows: the weights are streamed once, which the products of a decode step do nearer to the memory's rate than the epilogue's kernel (its tiles are
  // too few rows high to keep enough of W under way), and the logits stay in L2.  us, this way / that kernel, rows x V x H: 1 x 128256 x 4096 165 / 298, 61 x 128256 x 4096
  // 183 / 216, 128 x 128256 x 4096 213 / 222, 61 x 32000 x 512 21.2 / 23.4, but 128 x 32000 x 512 28 / 21 and 128 x 128256 x 512 71 / 45.
  if (p->z && (p->M <= 64 || (p->M <= 128 && p->H >= 2048))) {
    if (!p->zy || p->ldz % 4 || (reinterpret_cast<uintptr_t>(p->z) & 15)) return TFB_ERR_ARG;
    int rc = gemm_skinny(p->x, p->ldx, p->w, p->ldw, p->z, p->ldz, p->M, p->V, p->H, nullptr, nullptr, 0, 1.f, 0, 1, stream);
    if (rc == TFB_NOT_TAKEN)
      rc = gemm_rows(p->x, p->ldx, p->w, p->ldw, nullptr, nullptr, -1, 0, p->z, p->ldz, p->M, p->V, p->H, p->H, nullptr, nullptr, 0, 1.f, 0, 1, 0, status, stream);
    if (rc != TFB_NOT_TAKEN) {
      if (rc) return rc;
      tfb::launch_k_pdl(score_target_kernel, p->M, 128, 0, st, *p);
      return row_scores(p->z, p->ldz, p->M, p->V, p->targets, p->idx64, p->ignore, p->zy, p->logp, p->lse, status, stream);
    }
  }
  const int blocks = max(sm_count(), (p->M + GATHER_MOST - 1) / GATHER_MOST), per_block = (p->M + blocks - 1) / blocks;
  tfb::launch_k(score_gather_kernel, (p->M + per_block - 1) / per_block, 1024, 0, st, *p, per_block);
  ScoreArg a = *p;
  a.parts = gemm_row_stats(p->xc, p->ldc, p->w, p->ldw, p->M, p->V, p->H, p->rows, p->col_of, p->part, status, stream);
  if (a.parts <= 0) return a.parts <= -1000 ? -1000 - a.parts : a.parts;
  tfb::launch_k_pdl(score_finish_kernel, (p->M + 7) / 8, 256, 0, st, a);
  return int(cudaGetLastError());
}
