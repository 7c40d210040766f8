// Attention with capped scores, a bias by distance and a prefix mask: arguments, rows, scores, and the plain
// one-row-per-wave forms, shared by attn_masked.hip's kernels.
//
// Row s of the batch: lq queries, lk keys; query i stands at position p = lk - lq + i (rows end together, so one new
// token over a cache of lk sees all of it). Key j is visible to it when j < lk and, if causal, j <= p or
// j < prefix[s]: always the keys below a number vis(i) that grows with i. Scores of visible keys, natural units:
//   z = scale q.k;  cap > 0: z = cap tanh(z / cap);  z -= slope[head] |p - j|
// P = softmax z, O = P V, lse = ln sum e^z. No visible key: O = 0, lse = -inf, gradients 0. Hidden keys and the
// queries that do not see a key take no part whatever they hold: neither an infinity nor a NaN of theirs gets through
// (see nonfinite rows below).
// Backward, with t = tanh(z / cap): D = sum_j P_j (dO V^T)_j, dS = P (dO V^T - D) (1 - t^2), dQ = scale dS K, dK = scale
// dS^T Q, dV = P^T dO. D is dO.O of the unrounded O; the O at hand is rounded, and the gradients of 16-bit rows would
// carry half again the error that their own roundings give (bf16 0.34% against 0.24%). Since the P of a row sum to 1,
// D' = dO.(rounded O) is off by exactly r = sum_j P_j (dP_j - D'): the dQ blocks sum r as they go, and leave D' + r for
// the blocks of dK and dV and dQ = scale (sum dS' K - r sum P (1 - t^2) K), dS' with D'.
#pragma once

#include <math.h>

#include "common.h"

namespace rus {
namespace {

typedef __bf16 bf16;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct MaskedArgs {
  const void *q, *k, *v, *o, *dout;
  void *out, *dk, *dv;         // out: O, in the backward dQ (both [n_q, h_q, HD] contiguous); dk, dv contiguous
  float* lse;                  // [h_q, n_q] natural log
  float *dk_part, *dv_part;    // [h_q, n_k, HD] where query heads share keys
  float* dsum;                 // [h_q, n_q] D
  float* part;                 // parts of a split over keys
  const int32_t *cu_q, *cu_k, *prefix;
  const float* slopes;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, do_st, do_sh;  // strides: token, head
  int64_t n_q, n_k;
  int n_seq, h_q, h_kv, causal;
  int n_blocks;    // blocks of 128 queries, bound over all rows
  int n_kblocks;   // blocks of 128 keys
  int splits, split_tiles;
  float scale;
  float sl2;        // scale log2 e
  float kc;         // scale / cap
  float k2;         // 2 log2 e scale / cap
  float cap2;       // cap log2 e
};

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

// Row s, clamped into the token arrays. Rows n_seq and n_seq + 1 stand for the tokens behind the last row and before
// the first: queries without keys, keys without queries, so that their results are zeros.
struct MaskedRow {
  int qa, lq, ka, lk, pre;
  __device__ __forceinline__ int off() const { return lk - lq; }
  __device__ __forceinline__ int vis(int i, int causal) const {
    return causal ? min(lk, max(pre, off() + i + 1)) : lk;
  }
  // First query that sees key j (lq: none).
  __device__ __forceinline__ int first(int j, int causal) const {
    return !causal || j < pre ? 0 : min(lq, max(0, j - off()));
  }
};

__device__ __forceinline__ void row_span(const int32_t* cu, int s, int n_seq, int n, int& a, int& e) {
  if (s < n_seq) {
    a = min(max(cu[s], 0), n);
    e = min(max(cu[s + 1], a), n);
  } else if (s == n_seq) {
    a = min(max(cu[n_seq], 0), n);
    e = n;
  } else {
    a = 0;
    e = min(max(cu[0], 0), n);
  }
}

__device__ __forceinline__ MaskedRow masked_row(const MaskedArgs& a, int s) {
  MaskedRow r;
  int e;
  row_span(a.cu_q, s, a.n_seq, static_cast<int>(a.n_q), r.qa, e);
  r.lq = e - r.qa;
  row_span(a.cu_k, s, a.n_seq, static_cast<int>(a.n_k), r.ka, e);
  r.lk = e - r.ka;
  r.pre = 0;
  if (s < a.n_seq) {
    if (a.prefix) r.pre = min(max(a.prefix[s], 0), r.lk);
  }
  return r;
}

// What a pseudo-row's tokens get: as queries no keys, as keys no queries.
__device__ __forceinline__ MaskedRow as_queries(MaskedRow r, int s, int n_seq) {
  if (s >= n_seq) r.lk = 0;
  return r;
}
__device__ __forceinline__ MaskedRow as_keys(MaskedRow r, int s, int n_seq) {
  if (s >= n_seq) r.lq = 0;
  return r;
}

// Block id -> (row, block within it) for blocks of kb tokens, over rows 0 .. n_seq + 1 in order; false past the last.
// Uniform over the block.
__device__ __forceinline__ bool find_span_block(const int32_t* cu, int n_seq, int n, int blk, int kb, int& s, int& b,
                                                int& nb) {
  const int lane = threadIdx.x & 63;
  for (int c = 0; c < n_seq + 2; c += 64) {
    int a = 0, e = 0;
    if (c + lane < n_seq + 2) row_span(cu, c + lane, n_seq, n, a, e);
    const int mine = (e - a + kb - 1) / kb;
    int sum = mine;  // inclusive over the lanes
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o, 64);
      sum += lane >= o ? v : 0;
    }
    const int total = __shfl(sum, 63, 64);
    if (blk < total) {
      const int src = __ffsll(static_cast<unsigned long long>(__ballot(sum > blk))) - 1;
      s = c + src;
      nb = __shfl(mine, src, 64);
      b = blk - (__shfl(sum, src, 64) - nb);
      return true;
    }
    blk -= total;
  }
  return false;
}

// The row that query t belongs to.
__device__ __forceinline__ int row_of(const MaskedArgs& a, int t) {
  if (t < a.cu_q[0]) return a.n_seq + 1;
  if (t >= a.cu_q[a.n_seq]) return a.n_seq;
  int lo = 0, hi = a.n_seq;  // cu_q[lo] <= t < cu_q[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.cu_q[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// ---------------------------------------------------------------------------------------------
// Scores, in log2 units. tanh x = 1 - 2 / (1 + e^{2x}) is good to 2^-22 absolute, i.e. to that part of the cap, which
// counts where the cap is far above the scores: up to |x| = 1/4 the odd polynomial to x^9, 9e-9 of x away.
// ---------------------------------------------------------------------------------------------
constexpr float kSmallTanh = 0.25f;

__device__ __forceinline__ float tanh_small(float x) {
  const float z = x * x;
  float p = __builtin_fmaf(z, 2.1869489e-2f, -5.3968254e-2f);
  p = __builtin_fmaf(z, p, 1.3333333e-1f);
  p = __builtin_fmaf(z, p, -3.3333333e-1f);
  return __builtin_fmaf(z * p, x, x);
}

template <bool CAP, bool BIAS>
struct Scorer {
  float slope2;  // slope log2 e of the head
  float slope;   // slope / scale: in the products' unit
  __device__ __forceinline__ Scorer(const MaskedArgs& a, int head)
      : slope2(BIAS ? a.slopes[head] * kLog2e : 0.0f), slope(BIAS ? a.slopes[head] / a.scale : 0.0f) {}

  // Score of the product st at distance d, and (1 - t^2) of the cap.
  __device__ __forceinline__ float score(const MaskedArgs& a, float st, float d, float& factor) const {
    float y;
    factor = 1.0f;
    if constexpr (CAP) {
      const float x = st * a.kc;
      const float r = __builtin_amdgcn_rcpf(1.0f + exp2_raw(st * a.k2));
      const float ts = tanh_small(x);
      const bool small = fabsf(x) <= kSmallTanh;
      const float t = small ? ts : __builtin_fmaf(-2.0f, r, 1.0f);
      factor = small ? __builtin_fmaf(-ts, ts, 1.0f) : 4.0f * __builtin_fmaf(-r, r, r);
      y = t * a.cap2;
    } else {
      y = st * a.sl2;
    }
    if constexpr (BIAS) y = __builtin_fmaf(-slope2, fabsf(d), y);
    return y;
  }
};

// ---------------------------------------------------------------------------------------------
// One row per wave, products on the vector ALUs, P and dS in 32 bits: keys (or queries) one to a lane for the
// products, head dims over the lanes for the sums. Hidden elements are not read into any sum.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, kWave));
  return v;
}

__device__ __forceinline__ float lane_value(float x, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}

template <typename T, int HD>
__device__ __forceinline__ float dot_rows(const T* x, const T* y) {
  float acc = 0.0f;
#pragma unroll 4
  for (int c = 0; c < HD; c += 8) {
    float u[8], w[8];
    load_f32<T, 8>(x + c, u);
    load_f32<T, 8>(y + c, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = __builtin_fmaf(u[e], w[e], acc);
  }
  return acc;
}

template <typename T>
__device__ __forceinline__ const T* token(const void* x, int64_t t, int64_t st, int head, int64_t sh) {
  return static_cast<const T*>(x) + t * st + head * sh;
}

template <typename T, int HD, bool CAP, bool BIAS>
__device__ void plain_fwd_row(const MaskedArgs& a, const MaskedRow& r, int i, int head) {
  constexpr int N = HD / 64;
  const int lane = threadIdx.x & 63, g = head / (a.h_q / a.h_kv);
  const Scorer<CAP, BIAS> sc(a, head);
  const int64_t t = r.qa + i;
  const T* q = token<T>(a.q, t, a.q_st, head, a.q_sh);
  const int vis = r.vis(i, a.causal), p0 = r.off() + i;
  float m = -INFINITY, l = 0.0f, o[N] = {};
  for (int jb = 0; jb < vis; jb += 64) {
    const int j = min(jb + lane, vis - 1), n = min(64, vis - jb);
    float f;
    float y = sc.score(a, dot_rows<T, HD>(q, token<T>(a.k, r.ka + j, a.k_st, g, a.k_sh)),
                       static_cast<float>(p0 - j), f);
    if (lane >= n) y = -INFINITY;
    const float mn = fmaxf(m, wave_max(y));
    const float ref = mn == -INFINITY ? 0.0f : mn;
    const float alpha = exp2_raw(m - ref), p = exp2_raw(y - ref);
    m = mn;
    l = l * alpha + wave_sum(p);
#pragma unroll
    for (int d = 0; d < N; ++d) o[d] *= alpha;
    for (int jj = 0; jj < n; ++jj) {
      const float pj = lane_value(p, jj);
      const T* v = token<T>(a.v, r.ka + jb + jj, a.v_st, g, a.v_sh) + lane * N;
#pragma unroll
      for (int d = 0; d < N; ++d) o[d] = __builtin_fmaf(pj, static_cast<float>(v[d]), o[d]);
    }
  }
  float x[N];
#pragma unroll
  for (int d = 0; d < N; ++d) x[d] = vis > 0 ? o[d] / l : 0.0f;
  store_from_f32<T, N>(static_cast<T*>(a.out) + (t * a.h_q + head) * HD + lane * N, x);
  if (lane == 0) a.lse[head * a.n_q + t] = vis > 0 ? (m + log2f(l)) * kLn2 : -INFINITY;
}

template <typename T, int HD, bool CAP, bool BIAS>
__device__ void plain_dq_row(const MaskedArgs& a, const MaskedRow& r, int i, int head) {
  constexpr int N = HD / 64;
  const int lane = threadIdx.x & 63, g = head / (a.h_q / a.h_kv);
  const Scorer<CAP, BIAS> sc(a, head);
  const int64_t t = r.qa + i;
  const T* q = token<T>(a.q, t, a.q_st, head, a.q_sh);
  const T* go = token<T>(a.dout, t, a.do_st, head, a.do_sh);
  const int vis = r.vis(i, a.causal), p0 = r.off() + i;
  float dq[N] = {}, dsum = 0.0f;
  const float lse2 = a.lse[head * a.n_q + t] * kLog2e;
  for (int pass = 0; pass < 2; ++pass) {  // D first
    float sum = 0.0f;
    for (int jb = 0; jb < vis; jb += 64) {
      const int j = min(jb + lane, vis - 1), n = min(64, vis - jb);
      float f;
      const float y = sc.score(a, dot_rows<T, HD>(q, token<T>(a.k, r.ka + j, a.k_st, g, a.k_sh)),
                               static_cast<float>(p0 - j), f);
      const float dp = dot_rows<T, HD>(go, token<T>(a.v, r.ka + j, a.v_st, g, a.v_sh));
      const float p = exp2_raw(y - lse2);
      if (pass == 0) {
        sum += lane < n ? p * dp : 0.0f;
        continue;
      }
      const float ds = p * (dp - dsum) * f;
      for (int jj = 0; jj < n; ++jj) {
        const float dj = lane_value(ds, jj);
        const T* k = token<T>(a.k, r.ka + jb + jj, a.k_st, g, a.k_sh) + lane * N;
#pragma unroll
        for (int d = 0; d < N; ++d) dq[d] = __builtin_fmaf(dj, static_cast<float>(k[d]), dq[d]);
      }
    }
    if (pass == 0) dsum = wave_sum(sum);
  }
  if (lane == 0) a.dsum[head * a.n_q + t] = dsum;
#pragma unroll
  for (int d = 0; d < N; ++d) dq[d] *= a.scale;
  store_from_f32<T, N>(static_cast<T*>(a.out) + (t * a.h_q + head) * HD + lane * N, dq);
}

// dK and dV of key j over query heads h0 .. h1 - 1 (of one KV group): in 32 bits at pk, pv where these are given
// (one head's part), rounded into dk, dv otherwise.
template <typename T, int HD, bool CAP, bool BIAS>
__device__ void plain_dkv_row(const MaskedArgs& a, const MaskedRow& r, int j, int h0, int h1, float* pk, float* pv) {
  constexpr int N = HD / 64;
  const int lane = threadIdx.x & 63, g = h0 / (a.h_q / a.h_kv);
  const int64_t t = r.ka + j;
  const T* k = token<T>(a.k, t, a.k_st, g, a.k_sh);
  const T* v = token<T>(a.v, t, a.v_st, g, a.v_sh);
  const int i0 = r.first(j, a.causal);
  float dk[N] = {}, dv[N] = {};
  for (int head = h0; head < h1; ++head) {
    const Scorer<CAP, BIAS> sc(a, head);
    for (int ib = i0; ib < r.lq; ib += 64) {
      const int i = min(ib + lane, r.lq - 1), n = min(64, r.lq - ib);
      const int64_t tq = r.qa + i;
      const T* go = token<T>(a.dout, tq, a.do_st, head, a.do_sh);
      float f;
      const float y = sc.score(a, dot_rows<T, HD>(token<T>(a.q, tq, a.q_st, head, a.q_sh), k),
                               static_cast<float>(r.off() + i - j), f);
      const float dsum = a.dsum[head * a.n_q + tq];
      const float p = exp2_raw(y - a.lse[head * a.n_q + tq] * kLog2e);
      const float ds = p * (dot_rows<T, HD>(go, v) - dsum) * f;
      for (int ii = 0; ii < n; ++ii) {
        const float pi = lane_value(p, ii), di = lane_value(ds, ii);
        const T* q1 = token<T>(a.q, r.qa + ib + ii, a.q_st, head, a.q_sh) + lane * N;
        const T* g1 = token<T>(a.dout, r.qa + ib + ii, a.do_st, head, a.do_sh) + lane * N;
#pragma unroll
        for (int d = 0; d < N; ++d) {
          dk[d] = __builtin_fmaf(di, static_cast<float>(q1[d]), dk[d]);
          dv[d] = __builtin_fmaf(pi, static_cast<float>(g1[d]), dv[d]);
        }
      }
    }
  }
#pragma unroll
  for (int d = 0; d < N; ++d) dk[d] *= a.scale;
  if (pk) {
#pragma unroll
    for (int d = 0; d < N; ++d) {
      pk[lane * N + d] = dk[d];
      pv[lane * N + d] = dv[d];
    }
  } else {
    store_from_f32<T, N>(static_cast<T*>(a.dk) + (t * a.h_kv + g) * HD + lane * N, dk);
    store_from_f32<T, N>(static_cast<T*>(a.dv) + (t * a.h_kv + g) * HD + lane * N, dv);
  }
}

}  // namespace
}  // namespace rus
