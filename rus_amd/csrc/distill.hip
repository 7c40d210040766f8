// Distillation from a teacher's top logits over the lm_head, on fp16 MFMA for gfx950: the KL divergence of the
// student's softmax over the whole vocabulary from the teacher's over its K entries, and its hidden gradient, with no
// [N, V] logits.
//
//   q = softmax over the token's entries of (teacher logit / T)        p = softmax over the vocabulary of h W^T / T
//   KL = sum_k q_k (ln q_k - ln p_id(k))     loss = T^2 sum KL / denom     dH = T / denom (p W - sum_k q_k W_id(k))
//
// An entry whose id lies outside the vocabulary, or whose logit is -inf, is none; a token without entries has no
// teacher: KL and gradient 0, not counted in denom. An id that comes twice adds its q.
//
// Chunk by chunk of the vocabulary, as the cross-entropy's single pass (lmhead.hip): a GEMM whose epilogue keeps each
// token's maximum and sum per 256 rows and stores P = 2^(z log2 e - ref) in fp16, the rescaling of the half tiles whose
// reference moved, and the split-K product P . W_chunk into fp32 partials. What differs: the logits stay in 32 bits
// (divided by T, not rounded to fp16 first), and the teacher's entries are taken out of P before the product. They come
// back in 32 bits as (p_k - q_k) W_id(k), z_k from a product of its own: where the student has learnt its teacher p_k
// and q_k cancel, and p_k's rounding in fp16 (2^-12 of it) would be all that is left. These products come first, since
// their maximum is a good reference for P from the first chunk on (707 tokens x 87,296 rows: what a first chunk without
// one costs in rescaling is 35 us).
//
// Bound by the two GEMMs from some hundred tokens on, by reading W and W^T below. 151,936 rows of 1,536: 2,048 tokens
// 1,050 us statistics and P (910 TFLOP/s), 1,155 us gradient (830), 140 us all others; 707 tokens 404, 443 and 75 us; 64
// tokens 141 us each (3.3 TB/s) and 50 us.
#include <math.h>

#include "common.h"
#include "lmhead_tile.h"
#include "mfma_gemm.h"

namespace rus {
namespace {

typedef __bf16 bf16;

constexpr float kPrescale = 65536.0f;
constexpr int kMaxEntries = 1024;

struct DistillStats {
  float* part_m;
  float* part_s;
  int64_t part_stride;
  int part_base;
  float inv_t;
  f16* p;  // [n_tok][ld_p], columns up to kpad (0 past M)
  int64_t ld_p;
  int kpad;
  const float* ref;     // [n_tok] reference from the entries and the chunks before (-inf: none yet)
  float* half_ref;      // [2 * parts of the chunk][part_stride] the reference each half tile used
};

// A = W rows (vocabulary), B = H rows (tokens): a block's 256 x 256 tile of logits in registers, a token in each lane
// pair (l, l ^ 32). Maximum and sum over the tile's rows, and P.
template <bool PROBS>
__global__ __launch_bounds__(kThreads8) __attribute__((amdgpu_waves_per_eu(2, 2))) void
distill_stats_kernel(GemmArgs g, DistillStats p) {
  __shared__ __attribute__((aligned(16))) char smem[kSmemBytes];
  Tile tl;
  if (!tile_of(g, tl)) return;
  f32x16 acc[kMT][2];
  mainloop(g, tl, smem, acc);
  constexpr int RW = kBN / 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int wm = wave8_m(wave), wn = wave8_n(g, tl, wave);
  const int rows_left = g.M - (tl.m0 + wm * kWM);  // rows at or past this are padding
  float rm[2], rs[2];
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) {
    const int tok = tl.n0 + wn * RW + nt * 32 + (lane & 31);
    rm[nt] = -INFINITY, rs[nt] = 0.0f;
    if (tl.n0 + wn * RW + nt * 32 >= g.N) continue;  // no token here
    float m = -INFINITY;
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = mt * 32 + 8 * (r >> 2) + (r & 3) + 4 * h;
        const float z = row < rows_left ? acc[mt][nt][r] * p.inv_t : -INFINITY;
        acc[mt][nt][r] = z;
        m = fmaxf(m, z);
      }
    m = fmaxf(m, __shfl_xor(m, 32, kWave));
    float ref = m * kLog2e;
    if constexpr (PROBS) {
      const float given = tok < g.N ? p.ref[tok] : -INFINITY;
      ref = ref > given + kRefWindow ? own_ref(ref) : given;
      if (!(m > -INFINITY)) ref = given > -INFINITY ? given : 0.0f;
      if (h == 0 && tok < g.N) p.half_ref[static_cast<int64_t>(2 * (tl.m0 / kBM) + wm) * p.part_stride + tok] = ref;
    } else {
      if (!(m > -INFINITY)) ref = 0.0f;
    }
    float s = 0.0f;
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float e = exp2_fast(__builtin_fmaf(acc[mt][nt][r], kLog2e, -ref));
        s += e;
        acc[mt][nt][r] = e;
      }
    s += __shfl_xor(s, 32, kWave);
    if constexpr (PROBS) {
      // The partial's sum is relative to its maximum; 2^-100 below the reference any bounded sum will do, but a NaN
      // stays one.
      const float up = ref - m * kLog2e;
      s = up > 100.0f ? s * 0.0f + 1.0f : s * exp2_fast(up);
    }
    if (!(m > -INFINITY)) s = s != s ? s : 0.0f;
    rm[nt] = m;
    rs[nt] = s;
  }
  if constexpr (PROBS) {
    store_tile_tv<8>(smem, g, tl, p.p, p.ld_p, p.kpad, [&](int mt, int nt, int r, int) { return acc[mt][nt][r]; });
    __syncthreads();  // the staging reads of the LDS are done
  }
  // The two vocabulary halves of the tile meet in the LDS.
  float* xm = reinterpret_cast<float*>(smem);
  if (wm == 1 && h == 0) {
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const int o = wn * RW + nt * 32 + lane;
      xm[o] = rm[nt];
      xm[kBN + o] = rs[nt];
    }
  }
  __syncthreads();
  if (wm == 0 && h == 0) {
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const int o = wn * RW + nt * 32 + lane, tok = tl.n0 + o;
      if (tok >= g.N) continue;
      const float M = fmaxf(rm[nt], xm[o]);
      const float ref = M > -INFINITY ? M : 0.0f;
      const float s = rs[nt] * exp2_fast((rm[nt] - ref) * kLog2e) + xm[kBN + o] * exp2_fast((xm[o] - ref) * kLog2e);
      const int64_t at = static_cast<int64_t>(p.part_base + tl.m0 / kBM) * p.part_stride + tok;
      p.part_m[at] = M;
      p.part_s[at] = s;
    }
  }
}

struct Entries {
  const void* ids;     // [n_tok][k] int64 or int32
  const void* logits;  // [n_tok][k] fp32, fp16 or bf16
  int k, ids32, logits_type;
  int64_t n_vocab;
  float inv_t;
  __device__ __forceinline__ int64_t id(int64_t i) const {  // -1: outside the vocabulary
    const int64_t v = ids32 ? static_cast<const int32_t*>(ids)[i] : static_cast<const int64_t*>(ids)[i];
    return v >= 0 && v < n_vocab ? v : -1;
  }
  __device__ __forceinline__ float scaled_logit(int64_t i) const { return logit(i) * inv_t; }
  __device__ __forceinline__ float logit(int64_t i) const {
    if (logits_type == RUS_DTYPE_F32) return static_cast<const float*>(logits)[i];
    if (logits_type == RUS_DTYPE_F16) return static_cast<float>(static_cast<const f16*>(logits)[i]);
    return static_cast<float>(static_cast<const bf16*>(logits)[i]);
  }
};

// Sum and maximum over a block of 64 W threads, the same in every thread.
template <int W>
__device__ __forceinline__ float block_sum(float x, float* buf) {
  x = wave_sum(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = x;
  __syncthreads();
  float s = buf[0];
#pragma unroll
  for (int w = 1; w < W; ++w) s += buf[w];
  return s;
}
template <int W>
__device__ __forceinline__ float block_max(float x, float* buf) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, kWave));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = x;
  __syncthreads();
  float m = buf[0];
#pragma unroll
  for (int w = 1; w < W; ++w) m = fmaxf(m, buf[w]);
  return m;
}

// Between a chunk's two GEMMs, one token a block: the token's reference for the chunk is the one it came with, or, past
// the window, the one of the chunk's maximum; half tiles that used another are brought to it (by a power of two, exact
// but for values below fp16's range), and P = 0 at the teacher's entries. state: of the accumulated partials' reference
// (run), the next chunk's (ref); alpha = 2^(run before - run).
struct DistillState {
  const float *ref_in, *run_in;  // run_in nullptr: the first chunk
  float *ref_out, *run_out, *alpha, *m_run;
};

// Threads: with few tokens a block moves a row alone (64 tokens x 131,072 rows, some of them past the window: 34 us with
// 256 threads, 14 with 1,024), with many it mostly has nothing to move (2,048 tokens: 7 us with 256, 16 with 1,024).
template <int kFixThreads>
__global__ __launch_bounds__(kFixThreads) void distill_fix_kernel(f16* p, int64_t ld, int n, int64_t start,
                                                          const float* __restrict__ part_m,
                                                          const float* __restrict__ half_ref, int64_t stride,
                                                          DistillState st, Entries e) {
  __shared__ float buf[kFixThreads / 64], ks[kFixThreads];
  const int tok = blockIdx.x, t = threadIdx.x, parts = (n + kBM - 1) / kBM;
  float m = -INFINITY;
  for (int q = t; q < parts; q += kFixThreads) m = fmaxf(m, part_m[q * stride + tok]);
  m = block_max<kFixThreads / 64>(m, buf);
  const float y = m * kLog2e, given = st.ref_in[tok];
  const bool past = y > given + kRefWindow;
  float run = past ? own_ref(y) : given;
  if (!(run > -INFINITY)) run = 0.0f;  // no finite logit yet
  if (t == 0) {
    st.run_out[tok] = run;
    st.ref_out[tok] = y > -INFINITY ? fmaxf(run, own_ref(y)) : run;
    st.alpha[tok] = st.run_in ? exp2_fast(st.run_in[tok] - run) : 0.0f;
    st.m_run[tok] = run * 0.6931471805599453f;
  }
  f16* row = p + static_cast<int64_t>(tok) * ld;
  if (past) {  // a thread finds the half tiles, 16 threads move one
    for (int q0 = 0; q0 < 2 * parts; q0 += kFixThreads) {
      const float k = q0 + t < 2 * parts ? half_ref[(q0 + t) * stride + tok] : run;
      __syncthreads();
      ks[t] = k;
      __syncthreads();
      constexpr int kDepth = 8;  // half tiles that a group has in flight
      for (int q = t >> 4; q < min(kFixThreads, 2 * parts - q0); q += kFixThreads / 16 * kDepth) {
        f16x8 v[kDepth];
        float f[kDepth];
#pragma unroll
        for (int j = 0; j < kDepth; ++j) {
          const int qq = q + kFixThreads / 16 * j, c = 128 * (q0 + qq) + 8 * (t & 15);
          f[j] = qq < min(kFixThreads, 2 * parts - q0) && c < n ? ks[qq & (kFixThreads - 1)] : run;
          if (f[j] != run) v[j] = *reinterpret_cast<const f16x8*>(row + c);
        }
#pragma unroll
        for (int j = 0; j < kDepth; ++j) {
          if (f[j] == run) continue;
          const float by = exp2_fast(fminf(f[j] - run, 0.0f));  // above run only where P is all zero
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] = from_f32<f16>(static_cast<float>(v[j][i]) * by);
          *reinterpret_cast<f16x8*>(row + 128 * (q0 + q + kFixThreads / 16 * j) + 8 * (t & 15)) = v[j];
        }
      }
    }
    __builtin_amdgcn_s_waitcnt(0);  // before the zeros below
    __syncthreads();
  }
  for (int k = t; k < e.k; k += kFixThreads) {
    const int64_t i = static_cast<int64_t>(tok) * e.k + k, v = e.id(i), c = v - start;
    if (v >= 0 && c >= 0 && c < n && e.scaled_logit(i) != -INFINITY) row[c] = static_cast<f16>(0.0f);
  }
}

constexpr int kEntryWaves = 8, kEntryDepth = 8;  // rows of W that a wave has in flight

// The logits of a token's entries (a block each), products h . W_id in 32 bits, and the reference that their maximum
// gives.
__global__ __launch_bounds__(64 * kEntryWaves) void distill_logits_kernel(const f16* __restrict__ hidden, int64_t ld_h,
                                                                          const f16* __restrict__ w, int64_t ld_w,
                                                                          int d, Entries e, float* __restrict__ z,
                                                                          float* __restrict__ ref) {
  __shared__ int32_t id[kMaxEntries];
  __shared__ float buf[kEntryWaves];
  const int tok = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t base = static_cast<int64_t>(tok) * e.k;
  float any = 0.0f;
  for (int k = t; k < e.k; k += 64 * kEntryWaves) {
    id[k] = e.scaled_logit(base + k) == -INFINITY ? -1 : static_cast<int32_t>(e.id(base + k));
    any = fmaxf(any, id[k] >= 0 ? 1.0f : 0.0f);
  }
  any = block_max<kEntryWaves>(any, buf);  // (its barriers also close id)
  if (any == 0.0f) {  // no teacher: P = 0 for every token of the vocabulary, nothing of it is read
    if (t == 0 && ref) ref[tok] = INFINITY;
    return;
  }
  const f16* h = hidden + tok * ld_h;
  float top = -INFINITY;
  for (int k0 = kEntryDepth * wave; k0 < e.k; k0 += kEntryDepth * kEntryWaves) {
    float acc[kEntryDepth] = {};
    const f16* row[kEntryDepth];
#pragma unroll
    for (int j = 0; j < kEntryDepth; ++j)
      row[j] = w + static_cast<int64_t>(max(id[min(k0 + j, e.k - 1)], 0)) * ld_w;
    for (int c = 8 * lane; c < d; c += 512) {
      float x[8];
      load_f32<f16, 8>(h + c, x);
      Pack<f16, 8> y[kEntryDepth];
#pragma unroll
      for (int j = 0; j < kEntryDepth; ++j) y[j] = load_pack<f16, 8>(row[j] + c);
#pragma unroll
      for (int j = 0; j < kEntryDepth; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[j] = __builtin_fmaf(x[i], static_cast<float>(y[j].v[i]), acc[j]);
    }
#pragma unroll
    for (int j = 0; j < kEntryDepth; ++j) {
      const float v = wave_sum(acc[j]) * e.inv_t;
      if (k0 + j >= e.k) continue;
      if (lane == 0) z[base + k0 + j] = v;
      if (id[k0 + j] >= 0) top = fmaxf(top, v);
    }
  }
  if (!ref) return;
  top = block_max<kEntryWaves>(top, buf);
  if (t == 0) ref[tok] = top > -INFINITY && top < INFINITY ? floorf(top * kLog2e) : -INFINITY;
}

// lse of 16 tokens a block from the partials, 64 threads to a token.
constexpr int kLseTok = 16, kLseSub = 64;

__global__ __launch_bounds__(kLseTok * kLseSub) void distill_lse_kernel(const float* __restrict__ part_m,
                                                                        const float* __restrict__ part_s, int n_parts,
                                                                        int n_tok, float* __restrict__ lse) {
  __shared__ float ms[kLseSub][kLseTok + 1], ss[kLseSub][kLseTok + 1];
  const int col = threadIdx.x % kLseTok, sub = threadIdx.x / kLseTok, tok = blockIdx.x * kLseTok + col;
  float m = -INFINITY, s = 0.0f;
  auto add = [&](float m2, float s2) {
    const float mn = fmaxf(m, m2), ref = mn > -INFINITY ? mn : 0.0f;
    s = s * exp2_fast((m - ref) * kLog2e) + s2 * exp2_fast((m2 - ref) * kLog2e);
    m = mn;
  };
  constexpr int kDepth = 8;
  if (tok < n_tok)
    for (int q = sub; q < n_parts; q += kLseSub * kDepth) {
      float x[kDepth], y[kDepth];
#pragma unroll
      for (int j = 0; j < kDepth; ++j) {
        const int64_t o = static_cast<int64_t>(min(q + kLseSub * j, n_parts - 1)) * n_tok + tok;
        x[j] = part_m[o];
        y[j] = part_s[o];
      }
#pragma unroll
      for (int j = 0; j < kDepth; ++j)
        if (q + kLseSub * j < n_parts) add(x[j], y[j]);
    }
  ms[sub][col] = m;
  ss[sub][col] = s;
  __syncthreads();
  for (int half = kLseSub / 2; half >= 1; half /= 2) {
    if (sub < half) {
      add(ms[sub + half][col], ss[sub + half][col]);
      ms[sub][col] = m;
      ss[sub][col] = s;
    }
    __syncthreads();
  }
  if (sub == 0 && tok < n_tok) lse[tok] = m + logf(s);
}

// One token per block: KL, and in the place of each entry's logit what its row of W is worth in dH: p - q (p where an
// id comes first).
__global__ __launch_bounds__(256) void distill_entries_kernel(Entries e, const float* __restrict__ lse,
                                                              float* __restrict__ z, float* __restrict__ kl,
                                                              float* __restrict__ taught) {
  __shared__ int32_t id[kMaxEntries];
  __shared__ float buf[4];
  const int tok = blockIdx.x, t = threadIdx.x;
  const int64_t base = static_cast<int64_t>(tok) * e.k;
  float top = -INFINITY, any = 0.0f;
  for (int k = t; k < e.k; k += 256) {
    const float x = e.scaled_logit(base + k);
    const int32_t v = x == -INFINITY ? -1 : static_cast<int32_t>(e.id(base + k));
    id[k] = v;
    if (v >= 0) {
      top = fmaxf(top, x);
      any = 1.0f;
    }
  }
  any = block_max<4>(any, buf);
  if (any == 0.0f) {  // no teacher
    if (t == 0) kl[tok] = taught[tok] = 0.0f;
    return;
  }
  top = block_max<4>(top, buf);
  const float L = lse[tok];
  float total = 0.0f;
  for (int k = t; k < e.k; k += 256)
    if (id[k] >= 0) total += exp2_fast((e.scaled_logit(base + k) - top) * kLog2e);
  total = block_sum<4>(total, buf);
  const float log_total = logf(total);
  float sum = 0.0f;
  for (int k = t; k < e.k; k += 256) {
    float c = 0.0f;
    if (id[k] >= 0) {
      const float x = e.scaled_logit(base + k) - top, y = z[base + k] - L;  // ln q + ln total, ln p
      const float q = exp2_fast(x * kLog2e) / total;
      sum = __builtin_fmaf(q, (x - log_total) - y, sum);
      bool first = true;
      for (int j = 0; j < k; ++j) first = first && id[j] != id[k];
      c = (first ? exp2_fast(y * kLog2e) : 0.0f) - q;
    }
    z[base + k] = c;
  }
  sum = block_sum<4>(sum, buf);
  if (t == 0) {
    kl[tok] = sum;
    taught[tok] = 1.0f;
  }
}

__global__ __launch_bounds__(1024) void distill_loss_kernel(const float* __restrict__ kl,
                                                            const float* __restrict__ taught, int n_tok, float t2,
                                                            const float* __restrict__ num_items,
                                                            float* __restrict__ loss, float* __restrict__ denom) {
  __shared__ double s_sum[16];
  __shared__ float s_cnt[16];
  double sum = 0.0;
  float cnt = 0.0f;
  for (int i = threadIdx.x; i < n_tok; i += 1024) {
    sum += kl[i];
    cnt += taught[i];
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, kWave);
  cnt = wave_sum(cnt);
  if (threadIdx.x % kWave == 0) {
    s_sum[threadIdx.x / kWave] = sum;
    s_cnt[threadIdx.x / kWave] = cnt;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    float c = 0.0f;
    for (int w = 0; w < 16; ++w) {
      t += s_sum[w];
      c += s_cnt[w];
    }
    const float d = fmaxf(num_items ? *num_items : c, 1.0f);
    denom[0] = d;
    loss[0] = static_cast<float>(t * t2 / d);
  }
}

// dH of 512 columns of one token (times 2^16) a block: the partials' sum brought to the token's lse, and the entries' rows.
constexpr int kFinishThreads = 128;

__global__ __launch_bounds__(kFinishThreads) void distill_finish_kernel(
    const float* __restrict__ parts, int n_parts, int n_tok, int d, const float* __restrict__ m_run,
    const float* __restrict__ lse, const float* __restrict__ taught, const float* __restrict__ coef, Entries e,
    const f16* __restrict__ w, int64_t ld_w, const float* __restrict__ denom, float temperature,
    float* __restrict__ out) {
  __shared__ int32_t id[kMaxEntries];
  __shared__ float cf[kMaxEntries];
  const int tok = blockIdx.x, t = threadIdx.x;
  const bool on = taught[tok] != 0.0f;
  if (on)
    for (int k = t; k < e.k; k += kFinishThreads) {
      const int64_t i = static_cast<int64_t>(tok) * e.k + k;
      const float c = coef[i];
      id[k] = c == 0.0f ? -1 : static_cast<int32_t>(e.id(i));  // 0: an entry that is none
      cf[k] = c;
    }
  __syncthreads();
  const int c = 4 * (blockIdx.y * kFinishThreads + t);
  if (c >= d) return;
  const int64_t n = static_cast<int64_t>(n_tok) * d, at = static_cast<int64_t>(tok) * d + c;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (on) {
    constexpr int kDepth = 8;  // loads in flight together; the sum goes in order
    for (int q = 0; q < n_parts; q += kDepth) {
      f32x4 x[kDepth];
#pragma unroll
      for (int j = 0; j < kDepth; ++j) x[j] = *reinterpret_cast<const f32x4*>(parts + min(q + j, n_parts - 1) * n + at);
#pragma unroll
      for (int j = 0; j < kDepth; ++j)
        if (q + j < n_parts) o += x[j];
    }
    o *= exp2_fast((m_run[tok] - lse[tok]) * kLog2e);
    for (int k = 0; k < e.k; k += kDepth) {
      float y[kDepth][4];
#pragma unroll
      for (int j = 0; j < kDepth; ++j) {
        const int32_t v = id[min(k + j, e.k - 1)];
        load_f32<f16, 4>(w + static_cast<int64_t>(max(v, 0)) * ld_w + c, y[j]);
      }
#pragma unroll
      for (int j = 0; j < kDepth; ++j) {
        const int kk = min(k + j, e.k - 1);
        if (k + j >= e.k || id[kk] < 0) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(cf[kk], y[j][i], o[i]);
      }
    }
    o *= temperature * kPrescale / *denom;
  }
  *reinterpret_cast<f32x4*>(out + at) = o;
}

int check_entries(const char* fn, const void* ids, int32_t ids32, const void* logits, int32_t logits_type,
                  int32_t n_entries, int64_t n_tok, int64_t n_vocab) {
  if (n_entries <= 0 || n_entries > kMaxEntries)
    return fail(RUS_ERR_UNSUPPORTED, "%s: %d entries per token (1 to %d)", fn, n_entries, kMaxEntries);
  if (n_tok < 0 || n_tok >= (1 << 22) || n_vocab <= 0 || n_vocab >= (1 << 30))
    return fail(RUS_ERR_INVALID, "%s: bad sizes n_tok=%lld n_vocab=%lld", fn, (long long)n_tok, (long long)n_vocab);
  if (logits_type != RUS_DTYPE_F32 && logits_type != RUS_DTYPE_F16 && logits_type != RUS_DTYPE_BF16)
    return fail(RUS_ERR_INVALID, "%s: unknown dtype %d of the teacher's logits", fn, logits_type);
  if (n_tok > 0 && (!ids || !logits || !aligned(ids, ids32 ? 4 : 8)))
    return fail(RUS_ERR_INVALID, "%s: null or misaligned entries", fn);
  return RUS_OK;
}

int check_temperature(const char* fn, float t) {
  if (!(t >= 1e-6f) || !(t <= 1e6f))
    return fail(RUS_ERR_INVALID, "%s: temperature %g outside [1e-6, 1e6]", fn, static_cast<double>(t));
  return RUS_OK;
}

int check_width(const char* fn, int64_t d) {
  if (d <= 0 || d % kBK || d >= (1 << 24))
    return fail(RUS_ERR_INVALID, "%s: d=%lld must be a multiple of %d", fn, (long long)d, kBK);
  return RUS_OK;
}

}  // namespace
}  // namespace rus

using namespace rus;

namespace {

// The floats of a pass, one after another in the caller's workspace.
struct DistillLayout {
  float *part_m, *part_s;  // [parts of the vocabulary][n_tok]
  float *lse, *taught;     // [n_tok]
  float* coef;             // [n_tok][n_entries] the entries' logits, then what their rows are worth
  float* rows;             // [7][n_tok]: ref and run of the even chunks, of the odd ones, alpha, m_run, the first ref
  float* half_ref;         // [2 * parts of a chunk][n_tok]
  float* dparts;           // [n_split][n_tok][d]
  f16* p;                  // [n_tok][ld_p]
  int64_t ld_p, floats;
};

DistillLayout distill_layout(float* base, int64_t n_tok, int64_t d, int64_t n_vocab, int64_t chunk, int32_t n_entries,
                             int32_t n_split) {
  DistillLayout l;
  int64_t at = 0;
  auto take = [&](int64_t n) {
    float* p = base ? base + at : nullptr;
    at += (n + 3) / 4 * 4;  // every piece 16-byte aligned
    return p;
  };
  const int64_t parts = (n_vocab + kBM - 1) / kBM, cols = chunk < n_vocab ? chunk : n_vocab;
  l.part_m = take(parts * n_tok);
  l.part_s = take(parts * n_tok);
  l.lse = take(n_tok);
  l.taught = take(n_tok);
  l.coef = take(n_tok * n_entries);
  l.rows = l.half_ref = l.dparts = nullptr;
  l.p = nullptr;
  l.ld_p = (cols + kBK - 1) / kBK * kBK;
  if (n_split > 0) {
    l.rows = take(7 * n_tok);
    l.half_ref = take(2 * ((cols + kBM - 1) / kBM) * n_tok);
    l.dparts = take(n_split * n_tok * d);
    l.p = reinterpret_cast<f16*>(take(n_tok * l.ld_p / 2));
  }
  l.floats = at;
  return l;
}

int check_pass(const char* fn, int64_t n_tok, int64_t d, int64_t n_vocab, int64_t chunk, int32_t n_entries,
               int32_t n_split) {
  if (int e = check_width(fn, d)) return e;
  if (n_entries <= 0 || n_entries > kMaxEntries)
    return fail(RUS_ERR_UNSUPPORTED, "%s: %d entries per token (1 to %d)", fn, n_entries, kMaxEntries);
  if (n_tok <= 0 || n_tok >= (1 << 22) || n_vocab <= 0 || n_vocab >= (1 << 30) || chunk <= 0 ||
      (chunk < n_vocab && chunk % kBM) || n_split < 0 || n_split > 64)
    return fail(RUS_ERR_INVALID, "%s: bad sizes n_tok=%lld n_vocab=%lld chunk=%lld n_split=%d", fn, (long long)n_tok,
                (long long)n_vocab, (long long)chunk, n_split);
  return RUS_OK;
}

int check_workspace(const char* fn, const DistillLayout& l, const float* workspace, int64_t n_workspace) {
  if (!workspace || n_workspace < l.floats || !aligned(workspace, 16))
    return fail(RUS_ERR_INVALID, "%s: workspace of %lld floats, %lld needed", fn, (long long)n_workspace,
                (long long)l.floats);
  return RUS_OK;
}

}  // namespace

extern "C" int rus_lmhead_distill_workspace(int64_t n_tok, int64_t d, int64_t n_vocab, int64_t chunk,
                                            int32_t n_entries, int32_t n_split, int64_t* floats) {
  const char* fn = "rus_lmhead_distill_workspace";
  if (!floats) return fail(RUS_ERR_INVALID, "%s: null result", fn);
  if (int e = check_pass(fn, n_tok, d, n_vocab, chunk, n_entries, n_split)) return e;
  *floats = distill_layout(nullptr, n_tok, d, n_vocab, chunk, n_entries, n_split).floats;
  return RUS_OK;
}

extern "C" int rus_lmhead_distill_chunk(const void* hidden, int64_t ld_h, const void* weight_rows, int64_t ld_w,
                                        const void* weight_t, int64_t ld_wt, const void* weight, int64_t ld_all,
                                        int64_t n_tok, int64_t d, int64_t n_rows, int64_t vocab_start,
                                        int64_t n_vocab, int64_t chunk, const void* ids, int32_t ids32, const void* logits, int32_t logits_dtype, int32_t n_entries,
                                        float temperature, int32_t n_split, float* workspace, int64_t n_workspace,
                                        void* stream) {
  const char* fn = "rus_lmhead_distill_chunk";
  if (int e = check_pass(fn, n_tok, d, n_vocab, chunk, n_entries, n_split)) return e;
  if (int e = check_entries(fn, ids, ids32, logits, logits_dtype, n_entries, n_tok, n_vocab)) return e;
  if (int e = check_temperature(fn, temperature)) return e;
  if (vocab_start < 0 || vocab_start % chunk || n_rows <= 0 || n_rows > chunk || vocab_start + n_rows > n_vocab ||
      (n_rows < chunk && vocab_start + n_rows != n_vocab))
    return fail(RUS_ERR_INVALID, "%s: rows [%lld, + %lld) are no chunk of %lld in %lld", fn, (long long)vocab_start,
                (long long)n_rows, (long long)chunk, (long long)n_vocab);
  if (ld_h < d || ld_w < d || (vocab_start == 0 && ld_all < d))
    return fail(RUS_ERR_INVALID, "%s: row strides smaller than d", fn);
  const DistillLayout l = distill_layout(workspace, n_tok, d, n_vocab, chunk, n_entries, n_split);
  if (n_tok * ld_h * 2 >= (int64_t(1) << 32) || n_rows * ld_w * 2 >= (int64_t(1) << 32) ||
      (n_split && (n_tok * l.ld_p * 2 >= (int64_t(1) << 32) || d * ld_wt * 2 >= (int64_t(1) << 32))))
    return fail(RUS_ERR_UNSUPPORTED, "%s: an operand of 4 GiB or more", fn);
  if (int e = check_operand(fn, hidden, ld_h, "hidden")) return e;
  if (int e = check_operand(fn, weight_rows, ld_w, "weight_rows")) return e;
  if (vocab_start == 0)
    if (int e = check_operand(fn, weight, ld_all, "weight")) return e;
  if (int e = check_workspace(fn, l, workspace, n_workspace)) return e;
  GemmArgs g;
  g.A = static_cast<const f16*>(weight_rows);
  g.lda = ld_w;
  g.M = static_cast<int>(n_rows);
  g.B = static_cast<const f16*>(hidden);
  g.ldb = ld_h;
  g.N = static_cast<int>(n_tok);
  g.K = static_cast<int>(d);
  g.k_per_split = g.K;
  g.splits = 1;
  g.tiles_m = (g.M + kBM - 1) / kBM;
  g.tiles_n = (g.N + kBN - 1) / kBN;
  if (static_cast<int64_t>(g.tiles_m) * g.tiles_n >= (1 << 22))
    return fail(RUS_ERR_UNSUPPORTED, "%s: %d x %d tiles beyond one dispatch", fn, g.tiles_m, g.tiles_n);
  const int64_t index = vocab_start / chunk;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Entries e{ids, logits, n_entries, ids32, logits_dtype, n_vocab, 1.0f / temperature};
  float* first_ref = n_split ? l.rows + 6 * n_tok : nullptr;
  if (index == 0) {
    hipLaunchKernelGGL(distill_logits_kernel, dim3(static_cast<unsigned>(n_tok)), dim3(64 * kEntryWaves), 0, st,
                       static_cast<const f16*>(hidden), ld_h, static_cast<const f16*>(weight), ld_all, g.K, e, l.coef,
                       first_ref);
    if (int err = check_launch(fn)) return err;
  }
  const int part_base = static_cast<int>(vocab_start / kBM);
  DistillStats p{l.part_m, l.part_s, n_tok, part_base, 1.0f / temperature, l.p, l.ld_p,
                 static_cast<int>((n_rows + kBK - 1) / kBK * kBK), nullptr, l.half_ref};
  if (!n_split) {
    hipLaunchKernelGGL(distill_stats_kernel<false>, dim3(launch_grid(g)), dim3(kThreads8), 0, st, g, p);
    return check_launch(fn);
  }
  // (the chunks take turns in two states, so that none is updated in place)
  float* after = l.rows + index % 2 * 2 * n_tok;
  const float* before = l.rows + (index + 1) % 2 * 2 * n_tok;
  const DistillState state{index ? before : first_ref, index ? before + n_tok : nullptr, after, after + n_tok,
                           l.rows + 4 * n_tok, l.rows + 5 * n_tok};
  p.ref = state.ref_in;
  hipLaunchKernelGGL(distill_stats_kernel<true>, dim3(launch_grid(g)), dim3(kThreads8), 0, st, g, p);
  if (int err = check_launch(fn)) return err;
  auto fix = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(n_tok)), dim3(threads), 0, st, l.p, l.ld_p, g.M, vocab_start,
                       l.part_m + static_cast<int64_t>(part_base) * n_tok, l.half_ref, n_tok, state, e);
  };
  if (n_tok <= 256)
    fix(distill_fix_kernel<1024>, 1024);
  else
    fix(distill_fix_kernel<256>, 256);
  if (int err = check_launch(fn)) return err;
  return rus_lmhead_ce_grad_hidden_scaled(l.p, l.ld_p, weight_t, ld_wt, n_tok, d, n_rows, l.dparts, n_split, index > 0,
                                          state.alpha, stream);
}

extern "C" int rus_lmhead_distill_finish(const void* weight, int64_t ld_w, int64_t n_tok, int64_t d, int64_t n_vocab,
                                         int64_t chunk, const void* ids, int32_t ids32, const void* logits,
                                         int32_t logits_dtype, int32_t n_entries, float temperature, int32_t n_split,
                                         const float* num_items, float* kl,
                                         float* loss, float* denom, float* dh, float* workspace, int64_t n_workspace,
                                         void* stream) {
  const char* fn = "rus_lmhead_distill_finish";
  if (int e = check_pass(fn, n_tok, d, n_vocab, chunk, n_entries, n_split)) return e;
  if (int e = check_entries(fn, ids, ids32, logits, logits_dtype, n_entries, n_tok, n_vocab)) return e;
  if (int e = check_temperature(fn, temperature)) return e;
  if (ld_w < d) return fail(RUS_ERR_INVALID, "%s: row strides smaller than d", fn);
  if (int e = check_operand(fn, weight, ld_w, "weight")) return e;
  if (!kl || !loss || !denom || (n_split && (!dh || !aligned(dh, 16))))
    return fail(RUS_ERR_INVALID, "%s: null or misaligned output", fn);
  const DistillLayout l = distill_layout(workspace, n_tok, d, n_vocab, chunk, n_entries, n_split);
  if (int e = check_workspace(fn, l, workspace, n_workspace)) return e;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Entries e{ids, logits, n_entries, ids32, logits_dtype, n_vocab, 1.0f / temperature};
  const int n = static_cast<int>(n_tok);
  hipLaunchKernelGGL(distill_lse_kernel, dim3((n + kLseTok - 1) / kLseTok), dim3(kLseTok * kLseSub), 0, st, l.part_m,
                     l.part_s, static_cast<int>((n_vocab + kBM - 1) / kBM), n, l.lse);
  if (int err = check_launch(fn)) return err;
  hipLaunchKernelGGL(distill_entries_kernel, dim3(n), dim3(256), 0, st, e, l.lse, l.coef, kl, l.taught);
  if (int err = check_launch(fn)) return err;
  hipLaunchKernelGGL(distill_loss_kernel, dim3(1), dim3(1024), 0, st, kl, l.taught, n, temperature * temperature,
                     num_items, loss, denom);
  if (int err = check_launch(fn)) return err;
  if (!n_split) return RUS_OK;
  hipLaunchKernelGGL(distill_finish_kernel, dim3(n, static_cast<unsigned>((d + 4 * kFinishThreads - 1) /
                                                                          (4 * kFinishThreads))),
                     dim3(kFinishThreads), 0, st, l.dparts, n_split, n, static_cast<int>(d), l.rows + 5 * n_tok, l.lse,
                     l.taught, l.coef, e, static_cast<const f16*>(weight), ld_w, denom, temperature, dh);
  return check_launch(fn);
}
