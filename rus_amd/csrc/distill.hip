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
// and q_k cancel, and p_k's rounding in fp16 (2^-12 of it) would be all that is left.
//
// Bound by the two GEMMs from some hundred tokens on, by reading W and W^T below.
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
  const float* ref;     // [n_tok] reference from the chunks before (nullptr: the first chunk)
  float* half_ref;      // [2 * parts of the chunk][part_stride]
  uint32_t* chunk_max;  // [n_tok] ordered bits of the chunk's maximum (0 before the launch)
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
      const float given = p.ref && tok < g.N ? p.ref[tok] : -INFINITY;
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
      if constexpr (PROBS) atomicMax(p.chunk_max + tok, ordered_bits(M));
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

// P = 0 at the teacher's entries inside [start, start + n).
__global__ __launch_bounds__(256) void distill_blank_kernel(f16* p, int64_t ld, int n_tok, int n, int64_t start,
                                                            Entries e) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<int64_t>(n_tok) * e.k) return;
  const int64_t v = e.id(i), c = v - start;
  if (v >= 0 && c >= 0 && c < n && e.scaled_logit(i) != -INFINITY) p[i / e.k * ld + c] = static_cast<f16>(0.0f);
}

// Sum and maximum over a block of 256 threads, the same in every thread.
__device__ __forceinline__ float block_sum(float x, float* buf) {
  x = wave_sum(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = x;
  __syncthreads();
  return buf[0] + buf[1] + buf[2] + buf[3];
}
__device__ __forceinline__ float block_max(float x, float* buf) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, kWave));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = x;
  __syncthreads();
  return fmaxf(fmaxf(buf[0], buf[1]), fmaxf(buf[2], buf[3]));
}

// One token per block: its lse from the partials, the logits of its entries as products h . W_id in 32 bits, KL, and
// what each entry's row of W is worth in dH: coef = p - q (p where an id comes first).
__global__ __launch_bounds__(256) void distill_entries_kernel(
    const f16* __restrict__ hidden, int64_t ld_h, const f16* __restrict__ w, int64_t ld_w, int d, Entries e,
    const float* __restrict__ part_m, const float* __restrict__ part_s, int n_parts, int64_t stride,
    float* __restrict__ kl, float* __restrict__ lse, float* __restrict__ taught, float* __restrict__ coef) {
  __shared__ int32_t id[kMaxEntries];
  __shared__ float tl[kMaxEntries], z[kMaxEntries];
  __shared__ float buf[4];
  const int tok = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t base = static_cast<int64_t>(tok) * e.k;
  float top = -INFINITY, any = 0.0f;
  for (int k = t; k < e.k; k += 256) {
    int64_t v = e.id(base + k);
    const float x = e.scaled_logit(base + k);
    if (x == -INFINITY) v = -1;
    id[k] = static_cast<int32_t>(v);
    tl[k] = x;
    if (v >= 0) {
      top = fmaxf(top, x);
      any = 1.0f;
    }
  }
  any = block_max(any, buf);
  if (any == 0.0f) {  // no teacher
    if (t == 0) kl[tok] = lse[tok] = taught[tok] = 0.0f;
    return;
  }
  top = block_max(top, buf);
  float m = -INFINITY, s = 0.0f;
  for (int q = t; q < n_parts; q += 256) m = fmaxf(m, part_m[q * stride + tok]);
  m = block_max(m, buf);
  const float ref = m > -INFINITY ? m : 0.0f;
  for (int q = t; q < n_parts; q += 256)
    s += part_s[q * stride + tok] * exp2_fast((part_m[q * stride + tok] - ref) * kLog2e);
  s = block_sum(s, buf);
  const float L = m + logf(s);
  // Products of the entries' rows, four to a wave at a time so that their loads are in flight together.
  const f16* h = hidden + tok * ld_h;
  for (int k0 = 4 * wave; k0 < e.k; k0 += 16) {
    float acc[4] = {};
    for (int c = 8 * lane; c < d; c += 512) {
      float x[8];
      load_f32<f16, 8>(h + c, x);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int32_t v = id[min(k0 + j, e.k - 1)];
        if (v < 0) continue;
        float y[8];
        load_f32<f16, 8>(w + static_cast<int64_t>(v) * ld_w + c, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[j] = __builtin_fmaf(x[i], y[i], acc[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc[j] = wave_sum(acc[j]);
      if (lane == 0 && k0 + j < e.k) z[k0 + j] = acc[j] * e.inv_t;
    }
  }
  float total = 0.0f;
  for (int k = t; k < e.k; k += 256)
    if (id[k] >= 0) total += exp2_fast((tl[k] - top) * kLog2e);
  total = block_sum(total, buf);  // (its barriers also close z)
  const float log_total = logf(total);
  float sum = 0.0f;
  for (int k = t; k < e.k; k += 256) {
    float c = 0.0f;
    if (id[k] >= 0) {
      const float q = exp2_fast((tl[k] - top) * kLog2e) / total;
      sum = __builtin_fmaf(q, (tl[k] - top - log_total) - (z[k] - L), sum);
      bool first = true;
      for (int j = 0; j < k; ++j) first = first && id[j] != id[k];
      c = (first ? exp2_fast((z[k] - L) * kLog2e) : 0.0f) - q;
    }
    if (coef) coef[base + k] = c;
  }
  sum = block_sum(sum, buf);
  if (t == 0) {
    kl[tok] = sum;
    lse[tok] = L;
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

// dH of one token (times 2^16), one block: the partials' sum brought to the token's lse, and the entries' rows.
__global__ __launch_bounds__(256) void distill_finish_kernel(
    const float* __restrict__ parts, int n_parts, int n_tok, int d, const float* __restrict__ m_run,
    const float* __restrict__ lse, const float* __restrict__ taught, const float* __restrict__ coef, Entries e,
    const f16* __restrict__ w, int64_t ld_w, const float* __restrict__ denom, float temperature,
    float* __restrict__ out) {
  __shared__ int32_t id[kMaxEntries];
  __shared__ float cf[kMaxEntries];
  const int tok = blockIdx.x, t = threadIdx.x;
  const bool on = taught[tok] != 0.0f;
  if (on)
    for (int k = t; k < e.k; k += 256) {
      const int64_t i = static_cast<int64_t>(tok) * e.k + k;
      id[k] = static_cast<int32_t>(e.id(i));
      cf[k] = coef[i];
      if (cf[k] == 0.0f) id[k] = -1;  // an entry that is none
    }
  __syncthreads();
  const float f = on ? exp2_fast((m_run[tok] - lse[tok]) * kLog2e) : 0.0f;
  const float scale = temperature * kPrescale / *denom;
  const int64_t n = static_cast<int64_t>(n_tok) * d;
  for (int c = 4 * t; c < d; c += 1024) {
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    const int64_t at = static_cast<int64_t>(tok) * d + c;
    if (on) {
      f32x4 a = *reinterpret_cast<const f32x4*>(parts + at);
      for (int q = 1; q < n_parts; ++q) a += *reinterpret_cast<const f32x4*>(parts + q * n + at);
      o = a * f;
#pragma unroll 4
      for (int k = 0; k < e.k; ++k) {
        if (id[k] < 0) continue;
        float y[4];
        load_f32<f16, 4>(w + static_cast<int64_t>(id[k]) * ld_w + c, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(cf[k], y[i], o[i]);
      }
      o *= scale;
    }
    *reinterpret_cast<f32x4*>(out + at) = o;
  }
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

extern "C" int rus_lmhead_distill_fwd(const void* hidden, const void* weight, int64_t n_tok, int64_t d, int64_t ld_h,
                                      int64_t ld_w, int64_t n_vocab, float temperature, float* part_m, float* part_s,
                                      int64_t part_base, int64_t part_stride, void* probs, int64_t ld_p,
                                      const float* ref, float* half_ref, uint32_t* chunk_max, void* stream) {
  const char* fn = "rus_lmhead_distill_fwd";
  if (int e = check_width(fn, d)) return e;
  if (n_tok < 0 || n_tok >= (1 << 22) || n_vocab < 0 || n_vocab >= (1 << 30))
    return fail(RUS_ERR_INVALID, "%s: bad sizes n_tok=%lld n_vocab=%lld", fn, (long long)n_tok, (long long)n_vocab);
  if (int e = check_temperature(fn, temperature)) return e;
  if (n_tok == 0 || n_vocab == 0) return RUS_OK;
  if (ld_h < d || ld_w < d) return fail(RUS_ERR_INVALID, "%s: row strides smaller than d", fn);
  if (n_tok * ld_h * 2 >= (int64_t(1) << 32) || n_vocab * ld_w * 2 >= (int64_t(1) << 32))
    return fail(RUS_ERR_UNSUPPORTED, "%s: an operand of 4 GiB or more", fn);
  if (int e = check_operand(fn, hidden, ld_h, "hidden")) return e;
  if (int e = check_operand(fn, weight, ld_w, "weight")) return e;
  if (!part_m || !part_s || part_base < 0 || part_base >= (1 << 24) || part_stride < n_tok)
    return fail(RUS_ERR_INVALID, "%s: null output or bad partial layout", fn);
  const int64_t kpad = (n_vocab + kBK - 1) / kBK * kBK;
  if (probs) {
    if (ld_p < kpad) return fail(RUS_ERR_INVALID, "%s: ld_p must be >= %lld", fn, (long long)kpad);
    if (int e = check_operand(fn, probs, ld_p, "probs")) return e;
    if (!half_ref || !chunk_max) return fail(RUS_ERR_INVALID, "%s: null buffer", fn);
  }
  GemmArgs g;
  g.A = static_cast<const f16*>(weight);
  g.lda = ld_w;
  g.M = static_cast<int>(n_vocab);
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
  DistillStats p{part_m,   part_s, part_stride, static_cast<int>(part_base), 1.0f / temperature, static_cast<f16*>(probs),
                 ld_p,     static_cast<int>(kpad), ref, half_ref, chunk_max};
  if (probs)
    hipLaunchKernelGGL(distill_stats_kernel<true>, dim3(launch_grid(g)), dim3(kThreads8), 0,
                       static_cast<hipStream_t>(stream), g, p);
  else
    hipLaunchKernelGGL(distill_stats_kernel<false>, dim3(launch_grid(g)), dim3(kThreads8), 0,
                       static_cast<hipStream_t>(stream), g, p);
  return check_launch(fn);
}

extern "C" int rus_lmhead_distill_blank(void* probs, int64_t ld_p, int64_t n_tok, int64_t n_rows, int64_t vocab_start,
                                        const void* ids, int32_t ids32, const void* logits, int32_t logits_dtype,
                                        int32_t n_entries, int64_t n_vocab, float temperature, void* stream) {
  const char* fn = "rus_lmhead_distill_blank";
  if (int e = check_entries(fn, ids, ids32, logits, logits_dtype, n_entries, n_tok, n_vocab)) return e;
  if (int e = check_temperature(fn, temperature)) return e;
  if (n_tok == 0) return RUS_OK;
  if (!probs || n_rows <= 0 || n_rows > ld_p || vocab_start < 0 || vocab_start + n_rows > n_vocab)
    return fail(RUS_ERR_INVALID, "%s: rows [%lld, + %lld) of %lld, ld_p=%lld", fn, (long long)vocab_start,
                (long long)n_rows, (long long)n_vocab, (long long)ld_p);
  const Entries e{ids, logits, n_entries, ids32, logits_dtype, n_vocab, 1.0f / temperature};
  hipLaunchKernelGGL(distill_blank_kernel, dim3(static_cast<unsigned>((n_tok * n_entries + 255) / 256)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), static_cast<f16*>(probs), ld_p, static_cast<int>(n_tok),
                     static_cast<int>(n_rows), vocab_start, e);
  return check_launch(fn);
}

extern "C" int rus_lmhead_distill_entries(const void* hidden, int64_t ld_h, const void* weight, int64_t ld_w,
                                          int64_t n_vocab, int64_t n_tok, int64_t d, const void* ids, int32_t ids32,
                                          const void* logits, int32_t logits_dtype, int32_t n_entries,
                                          float temperature, const float* part_m, const float* part_s, int64_t n_parts,
                                          int64_t part_stride, const float* num_items, float* kl, float* lse,
                                          float* taught, float* coef, float* loss, float* denom, void* stream) {
  const char* fn = "rus_lmhead_distill_entries";
  if (int e = check_width(fn, d)) return e;
  if (int e = check_entries(fn, ids, ids32, logits, logits_dtype, n_entries, n_tok, n_vocab)) return e;
  if (int e = check_temperature(fn, temperature)) return e;
  if (!loss || !denom) return fail(RUS_ERR_INVALID, "%s: null pointer argument", fn);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (n_tok > 0) {
    if (ld_h < d || ld_w < d) return fail(RUS_ERR_INVALID, "%s: row strides smaller than d", fn);
    if (int e = check_operand(fn, hidden, ld_h, "hidden")) return e;
    if (int e = check_operand(fn, weight, ld_w, "weight")) return e;
    if (!part_m || !part_s || n_parts <= 0 || n_parts >= (1 << 24) || part_stride < n_tok || !kl || !lse || !taught)
      return fail(RUS_ERR_INVALID, "%s: null pointer or bad partial layout", fn);
    const Entries e{ids, logits, n_entries, ids32, logits_dtype, n_vocab, 1.0f / temperature};
    hipLaunchKernelGGL(distill_entries_kernel, dim3(static_cast<unsigned>(n_tok)), dim3(256), 0, st,
                       static_cast<const f16*>(hidden), ld_h, static_cast<const f16*>(weight), ld_w,
                       static_cast<int>(d), e, part_m, part_s, static_cast<int>(n_parts),
                       part_stride, kl, lse, taught, coef);
    if (int err = check_launch(fn)) return err;
  }
  hipLaunchKernelGGL(distill_loss_kernel, dim3(1), dim3(1024), 0, st, kl, taught, static_cast<int>(n_tok),
                     temperature * temperature, num_items, loss, denom);
  return check_launch(fn);
}

extern "C" int rus_lmhead_distill_finish(const float* parts, int32_t n_parts, int64_t n_tok, int64_t d,
                                         const float* m_run, const float* lse, const float* taught, const float* coef,
                                         const void* ids, int32_t ids32, int32_t n_entries, const void* weight,
                                         int64_t ld_w, int64_t n_vocab, const float* denom, float temperature,
                                         float* out, void* stream) {
  const char* fn = "rus_lmhead_distill_finish";
  if (int e = check_width(fn, d)) return e;
  if (int e = check_entries(fn, ids, ids32, ids, RUS_DTYPE_F32, n_entries, n_tok, n_vocab)) return e;
  if (int e = check_temperature(fn, temperature)) return e;
  if (n_tok == 0) return RUS_OK;
  if (ld_w < d) return fail(RUS_ERR_INVALID, "%s: row strides smaller than d", fn);
  if (int e = check_operand(fn, weight, ld_w, "weight")) return e;
  if (!parts || n_parts <= 0 || !m_run || !lse || !taught || !coef || !denom || !out || !aligned(parts, 16) ||
      !aligned(out, 16))
    return fail(RUS_ERR_INVALID, "%s: null or misaligned pointer", fn);
  const Entries e{ids, nullptr, n_entries, ids32, RUS_DTYPE_F32, n_vocab, 1.0f};
  hipLaunchKernelGGL(distill_finish_kernel, dim3(static_cast<unsigned>(n_tok)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), parts, n_parts, static_cast<int>(n_tok), static_cast<int>(d),
                     m_run, lse, taught, coef, e, static_cast<const f16*>(weight), ld_w, denom, temperature, out);
  return check_launch(fn);
}
