// Products of microscaled rows: y = x W^T (+ bias), and the gated feed-forward's first half
// silu(x Wg^T) (x Wu^T) with its backward, on v_mfma_scale_f32_32x32x64_f8f6f4.
//
// The instruction takes 64 of the contraction at a time: two blocks of 32, whose scales it applies
// itself. A lane (row l % 32, half g = l / 32) of an fp4 operand holds block g's 32 codes; of an fp8
// operand bytes 16 g .. +16 of block 0 and of block 1; its scale byte is block g's. W is the first
// operand (the rows of the result), x the second (its columns): register r of lane l holds row
// 8 (r / 4) + 4 (l / 32) + r % 4 and token l % 32. Row i of a tile is feature 16 ((i / 4) % 2) +
// 4 (i / 8) + i % 4, so that a lane's 16 registers are 16 neighbouring features.
// The instruction's sums are fp32; within the 16 products of an fp8 operand that it adds first it
// keeps about 13 bits below the largest (fp4 by fp4 loses nothing), so results are 16-bit types.
#include "mx.h"
#include "swiglu_math.h"

namespace rus {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

enum { kPlain = 0, kGluFwd = 1, kGluBwd = 2 };

struct MxArgs {
  const uint8_t *xc, *xs;  // x: codes and scales, [m] rows
  const uint8_t *wc, *ws;  // W: [n] rows, or [2 n] (gate rows, then up rows)
  int m, n, nb;            // tokens, output features, blocks of the contraction (multiple of 4)
  const void* bias;        // kPlain: [n] or null
  const void* dh;          // kGluBwd: [m, n]
  int64_t ld_dh;
  void* y;                 // [m, n], or [m, 2 n] for kGluBwd
  int64_t ldy;
  bool vec;                // rows of y (and dh, bias) allow aligned packs
};

template <int FMT>
constexpr int kMfmaFmt = FMT == kFp4 ? 4 : 0;

__device__ __forceinline__ int feature_of(int i) {
  return 16 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3);
}

// One operand row of one group of four blocks: the two MFMA steps' fragments and their scales.
template <int FMT>
struct Frag {
  u32x4s v[FMT == kFp4 ? 2 : 4];
  uint32_t s;
  __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* scales, int g) {
    if constexpr (FMT == kFp4) {
      const u32x4s* p = reinterpret_cast<const u32x4s*>(codes + g * 32);
      v[0] = p[0];
      v[1] = p[1];
    } else {
      const u32x4s* p = reinterpret_cast<const u32x4s*>(codes + g * 16);
      v[0] = p[0];
      v[1] = p[4];
      v[2] = p[2];
      v[3] = p[6];
    }
    s = *reinterpret_cast<const uint32_t*>(scales) >> (16 * g);
  }
  template <int S>
  __device__ __forceinline__ i32x8 get() const {
    if constexpr (FMT == kFp4)
      return i32x8{(int)v[S].x, (int)v[S].y, (int)v[S].z, (int)v[S].w, 0, 0, 0, 0};
    else
      return i32x8{(int)v[2 * S].x,     (int)v[2 * S].y,     (int)v[2 * S].z,     (int)v[2 * S].w,
                   (int)v[2 * S + 1].x, (int)v[2 * S + 1].y, (int)v[2 * S + 1].z, (int)v[2 * S + 1].w};
  }
};

template <int FW, int FX>
__device__ __forceinline__ void mma(const Frag<FW>& w, const Frag<FX>& x, f32x16& acc) {
  acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w.template get<0>(), x.template get<0>(), acc,
                                                        kMfmaFmt<FW>, kMfmaFmt<FX>, 0, (int)w.s, 0,
                                                        (int)x.s);
  acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w.template get<1>(), x.template get<1>(), acc,
                                                        kMfmaFmt<FW>, kMfmaFmt<FX>, 1, (int)w.s, 1,
                                                        (int)x.s);
}

// N neighbouring values from / to a row, from feature f on of `n`.
template <typename T, int N>
__device__ __forceinline__ void load_n(const T* row, int f, int n, bool vec, float (&v)[N]) {
  if (vec && f + N <= n) {
    load_f32<T, N>(row + f, v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = f + i < n ? static_cast<float>(row[f + i]) : 0.0f;
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T* row, int f, int n, bool vec, const float (&v)[N]) {
  if (vec && f + N <= n) {
    store_from_f32<T, N>(row + f, v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (f + i < n) row[f + i] = from_f32<T>(v[i]);
  }
}

// What becomes of N neighbouring features f.. of token t: a = x W^T (or the gate's), u the up's.
template <int EPI, typename T, int N>
__device__ __forceinline__ void finish(const MxArgs& g, int t, int f, const float (&a)[N],
                                       const float (&u)[N]) {
  T* y = static_cast<T*>(g.y) + t * g.ldy;
  float o[N];
  if constexpr (EPI == kPlain) {
    float b[N] = {};
    if (g.bias) load_n<T, N>(static_cast<const T*>(g.bias), f, g.n, g.vec, b);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = a[i] + b[i];
    store_n<T, N>(y, f, g.n, g.vec, o);
  } else if constexpr (EPI == kGluFwd) {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = a[i] * glu_sigmoid(a[i]) * u[i];
    store_n<T, N>(y, f, g.n, g.vec, o);
  } else {
    float d[N], du[N];
    load_n<T, N>(static_cast<const T*>(g.dh) + t * g.ld_dh, f, g.n, g.vec, d);
#pragma unroll
    for (int i = 0; i < N; ++i) glu_bwd(d[i], a[i], u[i], o[i], du[i]);
    store_n<T, N>(y, f, g.n, g.vec, o);
    store_n<T, N>(y + g.n, f, g.n, g.vec, du);
  }
}

// 32 features x 32 tokens per workgroup, the contraction's groups of four blocks dealt to the four
// waves, operands straight from memory to registers; the waves' sums meet in LDS.
constexpr int kRowsWaves = 4;

template <int FX, int FW, int EPI, typename T>
__global__ __launch_bounds__(kRowsWaves* kWave) void mx_rows_kernel(MxArgs g) {
  constexpr int NA = EPI == kPlain ? 1 : 2;
  __shared__ float red[kRowsWaves][NA][16][kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int f0 = blockIdx.x * 32, t0 = blockIdx.y * 32;
  // rows past the edge re-read the last one; what they give is not stored
  const int64_t tok = min(t0 + (lane & 31), g.m - 1);
  const int64_t feat = min(f0 + feature_of(lane & 31), g.n - 1);
  const uint8_t* xc = g.xc + tok * g.nb * kCodeBytes<FX>;
  const uint8_t* xs = g.xs + tok * g.nb;
  const uint8_t *wc[NA], *ws[NA];
#pragma unroll
  for (int a = 0; a < NA; ++a) {
    wc[a] = g.wc + (feat + static_cast<int64_t>(a) * g.n) * g.nb * kCodeBytes<FW>;
    ws[a] = g.ws + (feat + static_cast<int64_t>(a) * g.n) * g.nb;
  }
  f32x16 acc[NA] = {};
  for (int b = 4 * wave; b < g.nb; b += 4 * kRowsWaves) {
    Frag<FX> x;
    x.load(xc + b * kCodeBytes<FX>, xs + b, half);
#pragma unroll
    for (int a = 0; a < NA; ++a) {
      Frag<FW> w;
      w.load(wc[a] + b * kCodeBytes<FW>, ws[a] + b, half);
      mma(w, x, acc[a]);
    }
  }
#pragma unroll
  for (int a = 0; a < NA; ++a)
#pragma unroll
    for (int r = 0; r < 16; ++r) red[wave][a][r][lane] = acc[a][r];
  __syncthreads();
  const int t = t0 + (lane & 31), f = f0 + 16 * half + 4 * wave;
  if (t >= g.m || f >= g.n) return;
  float v[2][4] = {};
#pragma unroll
  for (int a = 0; a < NA; ++a)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 0; w < kRowsWaves; ++w) v[a][i] += red[w][a][4 * wave + i][lane];
  finish<EPI, T, 4>(g, t, f, v[0], v[1]);
}

template <int EPI, typename T, int FX, int FW>
int launch(const char* fn, const MxArgs& g, hipStream_t st) {
  const dim3 grid((g.n + 31) / 32, (g.m + 31) / 32);
  hipLaunchKernelGGL((mx_rows_kernel<FX, FW, EPI, T>), grid, dim3(kRowsWaves * kWave), 0, st, g);
  return check_launch(fn);
}

template <int EPI>
int dispatch(const char* fn, const MxArgs& g, int32_t x_fmt, int32_t w_fmt, int32_t dtype,
             hipStream_t st) {
  auto types = [&](auto t) -> int {
    typedef decltype(t) T;
    if (x_fmt == RUS_MX_FP8)
      return w_fmt == RUS_MX_FP4 ? launch<EPI, T, kFp8, kFp4>(fn, g, st)
                                 : launch<EPI, T, kFp8, kFp8>(fn, g, st);
    return w_fmt == RUS_MX_FP4 ? launch<EPI, T, kFp4, kFp4>(fn, g, st)
                               : launch<EPI, T, kFp4, kFp8>(fn, g, st);
  };
  return dtype == RUS_DTYPE_BF16 ? types(bf16{}) : types(f16{});
}

// Checks shared by the three entry points; fills what they share.
int prepare(const char* fn, MxArgs& g, const void* xc, const void* xs, int32_t x_fmt, const void* wc,
            const void* ws, int32_t w_fmt, int64_t m, int64_t n, int64_t k, void* y,
            int64_t ldy, int64_t y_cols, int32_t dtype) {
  if (m < 0 || n <= 0 || k <= 0 || m >= (1 << 30) || n >= (1 << 28) || k > (1 << 28))
    return fail(RUS_ERR_INVALID, "%s: bad sizes m=%lld n=%lld k=%lld", fn, (long long)m,
                (long long)n, (long long)k);
  if (dtype != RUS_DTYPE_F16 && dtype != RUS_DTYPE_BF16)
    return fail(RUS_ERR_UNSUPPORTED, "%s: results are fp16 or bf16, not dtype %d", fn, (int)dtype);
  if (ldy < y_cols && m > 1)
    return fail(RUS_ERR_INVALID, "%s: output row stride %lld smaller than %lld columns", fn,
                (long long)ldy, (long long)y_cols);
  if (m == 0) return RUS_OK;
  if (int e = check_mx(fn, xc, xs, x_fmt, "x")) return e;
  if (int e = check_mx(fn, wc, ws, w_fmt, "w")) return e;
  if (!y || !aligned(y, 2)) return fail(RUS_ERR_INVALID, "%s: output is null or misaligned", fn);
  if ((m + 31) / 32 > 65535)
    return fail(RUS_ERR_UNSUPPORTED, "%s: m=%lld is beyond 65535 tiles of 32 tokens", fn, (long long)m);
  g = MxArgs{};
  g.xc = static_cast<const uint8_t*>(xc);
  g.xs = static_cast<const uint8_t*>(xs);
  g.wc = static_cast<const uint8_t*>(wc);
  g.ws = static_cast<const uint8_t*>(ws);
  g.m = static_cast<int>(m);
  g.n = static_cast<int>(n);
  g.nb = static_cast<int>(mx_blocks(k));
  g.y = y;
  g.ldy = ldy;
  g.vec = aligned(y, 16) && ldy % 8 == 0 && n % 8 == 0;
  return RUS_OK;
}

}  // namespace
}  // namespace rus

using namespace rus;

extern "C" int rus_mx_gemm(const void* x_codes, const void* x_scales, int32_t x_fmt,
                           const void* w_codes, const void* w_scales, int32_t w_fmt, int64_t m,
                           int64_t n, int64_t k, const void* bias, void* y, int64_t stride_y,
                           int32_t dtype, void* stream) {
  const char* fn = "rus_mx_gemm";
  MxArgs g;
  if (int e = prepare(fn, g, x_codes, x_scales, x_fmt, w_codes, w_scales, w_fmt, m, n, k, y, stride_y,
                      n, dtype))
    return e;
  if (m == 0) return RUS_OK;
  if (bias && !aligned(bias, 2)) return fail(RUS_ERR_INVALID, "%s: misaligned bias", fn);
  g.bias = bias;
  g.vec = g.vec && (!bias || aligned(bias, 16));
  return dispatch<kPlain>(fn, g, x_fmt, w_fmt, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int rus_mx_glu_fwd(const void* x_codes, const void* x_scales, int32_t x_fmt,
                              const void* w_codes, const void* w_scales, int32_t w_fmt, int64_t m,
                              int64_t n, int64_t k, void* h, int64_t stride_h, int32_t dtype,
                              void* stream) {
  const char* fn = "rus_mx_glu_fwd";
  MxArgs g;
  if (int e = prepare(fn, g, x_codes, x_scales, x_fmt, w_codes, w_scales, w_fmt, m, n, k, h, stride_h,
                      n, dtype))
    return e;
  if (m == 0) return RUS_OK;
  return dispatch<kGluFwd>(fn, g, x_fmt, w_fmt, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int rus_mx_glu_bwd(const void* dh, int64_t stride_dh, const void* x_codes,
                              const void* x_scales, int32_t x_fmt, const void* w_codes,
                              const void* w_scales, int32_t w_fmt, int64_t m, int64_t n, int64_t k,
                              void* d_gu, int64_t stride_d_gu, int32_t dtype, void* stream) {
  const char* fn = "rus_mx_glu_bwd";
  MxArgs g;
  if (int e = prepare(fn, g, x_codes, x_scales, x_fmt, w_codes, w_scales, w_fmt, m, n, k, d_gu,
                      stride_d_gu, 2 * n, dtype))
    return e;
  if (m == 0) return RUS_OK;
  if (stride_dh < n && m > 1)
    return fail(RUS_ERR_INVALID, "%s: stride_dh=%lld smaller than a row", fn, (long long)stride_dh);
  if (!dh || !aligned(dh, 2)) return fail(RUS_ERR_INVALID, "%s: dh is null or misaligned", fn);
  g.dh = dh;
  g.ld_dh = stride_dh;
  g.vec = g.vec && aligned(dh, 16) && stride_dh % 8 == 0;
  return dispatch<kGluBwd>(fn, g, x_fmt, w_fmt, dtype, static_cast<hipStream_t>(stream));
}
