// Rows to microscaled blocks and back, and the residual + RMSNorm whose output is such blocks.
#include "mx.h"

namespace rus {
namespace {

// Eight elements of a row from column c on, zeros from `cols` on: 16-byte accesses at whatever
// alignment the elements have (rows of an odd length start anywhere), single ones at the row's end.
typedef u32x4s u32x4u __attribute__((aligned(2)));
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int c, int cols, float (&v)[8]) {
  if (c + 8 <= cols) {
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 8 / E; ++j) {
      const u32x4s w = *reinterpret_cast<const u32x4u*>(row + c + j * E);
      const Pack<T, E> t = __builtin_bit_cast(Pack<T, E>, w);
#pragma unroll
      for (int i = 0; i < E; ++i) v[j * E + i] = static_cast<float>(t.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? static_cast<float>(row[c + i]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ row, int c, int cols, const float (&v)[8]) {
  if (c + 8 <= cols) {
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 8 / E; ++j) {
      Pack<T, E> t;
#pragma unroll
      for (int i = 0; i < E; ++i) t.v[i] = from_f32<T>(v[j * E + i]);
      *reinterpret_cast<u32x4u*>(row + c + j * E) = __builtin_bit_cast(u32x4s, t);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[c + i] = from_f32<T>(v[i]);
  }
}

// A thread's eight scaled elements leave as one 4- or 8-byte store.
template <int FMT>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&v)[8], bool nan) {
  if constexpr (FMT == kFp4) {
    uint32_t w[1];
    to_fp4<8>(v, nan, w);
    *reinterpret_cast<uint32_t*>(p) = w[0];
  } else {
    uint32_t w[2];
    to_fp8<8>(v, nan, w);
    *reinterpret_cast<u32x2s*>(p) = u32x2s{w[0], w[1]};
  }
}

// Thread = eight elements, four neighbouring lanes = one block: a 16-byte load, the block's largest
// element by two lane exchanges, one store of 4 or 8 bytes of codes. Bound by memory: 17920 x 1536
// fp16 to 4 bits 14.5 us and back 12.4 us (70 MB of rows, codes and scales: 4.8 / 5.6 TB/s), fp32 18.8 us
// (125 MB). Rows of an odd length go by the same accesses: 16384 x 1111 fp16 to 4 bits took 24.5 us
// with single-element loads there and takes 13.3, back 26.5 and 10.2; lengths that are multiples of 8
// took the same either way.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, int64_t stride,
                                                          int cols, int nb, int64_t total,
                                                          uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;  // whole blocks leave together: total is a multiple of 16
  const int64_t row = i / (nb * 4);
  const int p = static_cast<int>(i - row * (nb * 4));
  float v[8];
  load8<T>(x + row * stride, p * 8, cols, v);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[j]));
  top = quad_max(top);
  const uint32_t b = scale_byte<FMT>(top);
  const float inv = inv_scale(b);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= inv;
  store_codes<FMT>(codes + i * (kCodeBytes<FMT> / 4), v, b == 255);
  if ((threadIdx.x & 3) == 0) scales[i >> 2] = static_cast<uint8_t>(b);
}

template <typename T, int FMT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales,
                                                            int cols, int nb, int packs,
                                                            int64_t total, T* __restrict__ out,
                                                            int64_t stride) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int64_t row = i / packs;
  const int p = static_cast<int>(i - row * packs);
  const uint8_t* c = codes + (row * nb * 4 + p) * (kCodeBytes<FMT> / 4);
  const float s = mx_scale(scales[row * nb + (p >> 2)]);
  float v[8];
  if constexpr (FMT == kFp4) {
    from_fp4(*reinterpret_cast<const uint32_t*>(c), s, v);
  } else {
    const u32x2s w = *reinterpret_cast<const u32x2s*>(c);
    from_fp8(w.x, w.y, s, v);
  }
  store8<T>(out + row * stride, p * 8, cols, v);
}

// ---- residual + RMSNorm into fp8 blocks ----------------------------------------------------------
//
// h = T(x + res), y = h rstd w, and y's blocks. The normalised value is rounded once, from 64 bits to
// the 8-bit element: the element type has few values, and a sum of squares or a product rounded in
// fp32 first would put a y next to a border between two of them (or next to a power of two that
// changes the block's scale) on either side of it depending on the order of the sum.
//
// The sum is fp64 throughout. The products are fp32 where that cannot be told from fp64
// (fast_blocks): three roundings move y by less than 2^-22 of it, so where y (1 - 2^-21) and
// y (1 + 2^-21) become the same code, so does the fp64 value. A wave in which one element fails that
// test (a few in a thousand do) forms its elements in fp64.

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

// 1 / sqrt(x) to about an ulp: the hardware's estimate is good to 2^-22 or better, and a step of third
// order cubes that. (A square root and a division, each correctly rounded, are ten times as many
// instructions, more than the rest of a thread's work on its eight elements.)
__device__ __forceinline__ double rsqrt64(double x) {
  const double y = __builtin_amdgcn_rsq(x);
  if (!(y > 0.0 && y < __builtin_inf())) return y;
  const double e = __builtin_fma(-x * y, y, 1.0);
  return __builtin_fma(y * e, __builtin_fma(0.375, e, 0.5), y);
}

// fp64 -> fp32 rounded to odd: a later rounding to few bits then gives that of the fp64 value.
__device__ __forceinline__ float to_odd(double d) {
  const float f = static_cast<float>(d);
  const double back = static_cast<double>(f);
  if (back == d || !(__builtin_fabs(d) < 1e30)) return f;
  uint32_t u = __builtin_bit_cast(uint32_t, f);
  if (__builtin_fabs(back) > __builtin_fabs(d)) u -= 1;
  return __builtin_bit_cast(float, u | 1u);
}

// A thread's eight codes and their block's scale byte from fp64 products.
__device__ __forceinline__ void exact_blocks(const float (&h)[8], const float (&w)[8], double r,
                                             uint32_t (&code)[2], int* scale) {
  double y[8];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = static_cast<double>(h[i]) * r * static_cast<double>(w[i]);
    top = max(top, static_cast<uint32_t>(__builtin_bit_cast(uint64_t, y[i]) >> 32) & 0x7fffffffu);
  }
  top = quad_max(top);
  int b = static_cast<int>(top >> 20) - 1023 + 127 - kEmax<kFp8>;
  const bool nan = top >= 0x7ff00000u;
  b = nan ? 255 : min(max(b, 0), 254);
  // 2^(127 - b) in fp64, exact products
  const double inv = __builtin_bit_cast(double, static_cast<uint64_t>(1023 + 127 - b) << 52);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_odd(y[i] * inv);
  to_fp8<8>(v, nan, code);
  *scale = b;
}

// The same from fp32 products; false (for the whole wave) where they do not settle it. `plain`: rstd is
// far from fp32's limits; `inside`: the block holds some of the row's elements (else it is zeros). With
// the block's largest y in [2^-60, 2^100] and |w| up to 2^40, every product that is not far below the
// smallest code is a normal number.
__device__ __forceinline__ bool fast_blocks(const float (&h)[8], const float (&w)[8], float r,
                                            bool plain, bool inside, uint32_t (&code)[2], int* scale) {
  float y[8], wide = 0.0f;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = h[i] * r * w[i];
    top = max(top, abs_bits(y[i]));
    wide = fmaxf(wide, __builtin_fabsf(w[i]));
  }
  top = quad_max(top);
  const float t = __builtin_bit_cast(float, top);
  const float lo = 1.0f - 0x1p-21f, hi = 1.0f + 0x1p-21f;
  bool ok = plain && wide < 0x1p40f && t > 0x1p-60f && t < 0x1p100f &&
            (abs_bits(t * lo) >> 23) == (abs_bits(t * hi) >> 23);
  const int b = static_cast<int>(top >> 23) - kEmax<kFp8>;
  const float inv = inv_scale(b);
  float a[8], z[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = y[i] * inv;
    a[i] = v * lo;
    z[i] = v * hi;
  }
  uint32_t other[2];
  to_fp8<8>(a, false, code);
  to_fp8<8>(z, false, other);
  ok = ok && code[0] == other[0] && code[1] == other[1];
  *scale = b;
  if (!inside) {
    code[0] = code[1] = 0;
    *scale = 0;
    ok = true;
  }
  return __all(ok);
}

// One workgroup per row, eight columns per thread and step; a row of up to 8192 columns stays in
// registers between the two passes, a longer one is read again (from this CU's L2). Bound by memory:
// 16381 x 1536 fp16 with the residual moves 177 MB in 36 us (4.9 TB/s); on the same rows each call, part
// of which the last-level cache holds, 31 us, and there it took 39 us with fp64 products and a correctly
// rounded square root and division, bound by arithmetic. Without a residual, where 76 MB move, arithmetic
// still bounds it: 26 us (33 in fp64).
template <typename T, typename W, bool HAS_RES>
__global__ __launch_bounds__(1024) void rmsnorm_mx_kernel(
    const T* __restrict__ x, const T* __restrict__ res, const W* __restrict__ w, T* sum_out,
    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, float* __restrict__ rstd, int cols,
    int nb, int64_t stride, float eps, double over) {
  __shared__ double red[16];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * stride;
  const T* rr = HAS_RES ? res + row * stride : nullptr;
  T* sr = HAS_RES ? sum_out + row * stride : nullptr;
  const int packs = nb * 4, nt = blockDim.x;
  double ss = 0.0;
  float h[8];
  for (int p = threadIdx.x; p < packs; p += nt) {
    const int c = p * 8;
    load8<T>(xr, c, cols, h);
    if (HAS_RES) {
      float r[8];
      load8<T>(rr, c, cols, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = round_to<T>(h[i] + r[i]);
      store8<T>(sr, c, cols, h);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += static_cast<double>(h[i]) * static_cast<double>(h[i]);
  }
  ss = wave_sum64(ss);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
  __syncthreads();
  double all = 0.0;
  for (int i = 0; i < nt / kWave; ++i) all += red[i];
  const double r = rsqrt64(all * over + static_cast<double>(eps));
  const float r32 = static_cast<float>(r);
  if (threadIdx.x == 0) rstd[row] = r32;
  const bool plain = r32 > 0x1p-100f && r32 < 0x1p100f;
  const bool kept = packs <= nt;  // the row is still in h
  for (int p = threadIdx.x; p < packs; p += nt) {
    const int c = p * 8;
    if (!kept) load8<T>(HAS_RES ? sr : xr, c, cols, h);  // this thread wrote these itself
    float wv[8];
    load8<W>(w, c, cols, wv);
    uint32_t code[2];
    int b;
    if (!fast_blocks(h, wv, r32, plain, c - (p & 3) * 8 < cols, code, &b))
      exact_blocks(h, wv, r, code, &b);
    *reinterpret_cast<u32x2s*>(codes + (row * packs + p) * 8) = u32x2s{code[0], code[1]};
    if ((p & 3) == 0) scales[row * nb + (p >> 2)] = static_cast<uint8_t>(b);
  }
}

template <typename F>
int with_type(const char* fn, int32_t dtype, F f) {
  switch (dtype) {
    case RUS_DTYPE_F16:
      return f(f16{});
    case RUS_DTYPE_F32:
      return f(float{});
    case RUS_DTYPE_BF16:
      return f(bf16{});
  }
  return fail(RUS_ERR_INVALID, "%s: unknown dtype %d", fn, (int)dtype);
}

int check_rows(const char* fn, int64_t rows, int64_t cols) {
  if (rows < 0 || cols <= 0 || cols > (1 << 28))
    return fail(RUS_ERR_INVALID, "%s: bad sizes rows=%lld cols=%lld", fn, (long long)rows,
                (long long)cols);
  if (rows > (int64_t(1) << 36) / mx_blocks(cols))
    return fail(RUS_ERR_UNSUPPORTED, "%s: rows=%lld x cols=%lld is beyond 2^36 blocks", fn,
                (long long)rows, (long long)cols);
  return RUS_OK;
}

}  // namespace

int quantize_rows(const char* fn, const void* x, int32_t dtype, int64_t n_rows, int64_t n_cols,
                  int64_t stride_row, int32_t fmt, void* codes, void* scales, hipStream_t stream) {
  if (int e = check_rows(fn, n_rows, n_cols)) return e;
  if (stride_row < n_cols && n_rows > 1)
    return fail(RUS_ERR_INVALID, "%s: stride_row=%lld smaller than a row", fn, (long long)stride_row);
  return with_type(fn, dtype, [&](auto t) -> int {
    typedef decltype(t) T;
    if (n_rows == 0) return RUS_OK;
    if (int e = check_mx(fn, codes, scales, fmt, "output")) return e;
    if (!x || !aligned(x, sizeof(T))) return fail(RUS_ERR_INVALID, "%s: x is null or misaligned", fn);
    const int nb = static_cast<int>(mx_blocks(n_cols));
    auto go = [&](auto k, int64_t bytes) {
      return by_rows(fn, n_rows, nb * 4, [&](int64_t first, int64_t rows) {
        const int64_t total = rows * nb * 4;
        hipLaunchKernelGGL(k, dim3(static_cast<unsigned>((total + 255) / 256)), dim3(256), 0, stream,
                           static_cast<const T*>(x) + first * stride_row, stride_row,
                           static_cast<int>(n_cols), nb, total,
                           static_cast<uint8_t*>(codes) + first * nb * bytes,
                           static_cast<uint8_t*>(scales) + first * nb);
      });
    };
    return fmt == RUS_MX_FP4 ? go(mx_quantize_kernel<T, kFp4>, kCodeBytes<kFp4>)
                             : go(mx_quantize_kernel<T, kFp8>, kCodeBytes<kFp8>);
  });
}

}  // namespace rus

using namespace rus;

extern "C" int rus_mx_quantize(const void* x, int32_t dtype, int64_t n_rows, int64_t n_cols,
                               int64_t stride_row, int32_t fmt, void* codes, void* scales,
                               void* stream) {
  return quantize_rows("rus_mx_quantize", x, dtype, n_rows, n_cols, stride_row, fmt, codes, scales,
                       static_cast<hipStream_t>(stream));
}

extern "C" int rus_mx_dequantize(const void* codes, const void* scales, int32_t fmt, int64_t n_rows,
                                 int64_t n_cols, void* out, int32_t dtype, int64_t stride_row,
                                 void* stream) {
  const char* fn = "rus_mx_dequantize";
  if (int e = check_rows(fn, n_rows, n_cols)) return e;
  if (stride_row < n_cols && n_rows > 1)
    return fail(RUS_ERR_INVALID, "%s: stride_row=%lld smaller than a row", fn, (long long)stride_row);
  return with_type(fn, dtype, [&](auto t) -> int {
    typedef decltype(t) T;
    if (n_rows == 0) return RUS_OK;
    if (int e = check_mx(fn, codes, scales, fmt, "input")) return e;
    if (!out || !aligned(out, sizeof(T)))
      return fail(RUS_ERR_INVALID, "%s: out is null or misaligned", fn);
    const int nb = static_cast<int>(mx_blocks(n_cols));
    const int packs = static_cast<int>((n_cols + 7) / 8);
    auto go = [&](auto k, int64_t bytes) {
      return by_rows(fn, n_rows, packs, [&](int64_t first, int64_t rows) {
        const int64_t total = rows * packs;
        hipLaunchKernelGGL(k, dim3(static_cast<unsigned>((total + 255) / 256)), dim3(256), 0,
                           static_cast<hipStream_t>(stream),
                           static_cast<const uint8_t*>(codes) + first * nb * bytes,
                           static_cast<const uint8_t*>(scales) + first * nb, static_cast<int>(n_cols),
                           nb, packs, total, static_cast<T*>(out) + first * stride_row, stride_row);
      });
    };
    return fmt == RUS_MX_FP4 ? go(mx_dequantize_kernel<T, kFp4>, kCodeBytes<kFp4>)
                             : go(mx_dequantize_kernel<T, kFp8>, kCodeBytes<kFp8>);
  });
}

extern "C" int rus_rmsnorm_mx_fwd(const void* x, const void* residual, const void* weight,
                                  int32_t w_dtype, void* sum_out, void* codes, void* scales,
                                  float* rstd, int64_t n_rows, int64_t n_cols, int64_t stride_row,
                                  float eps, int32_t dtype, void* stream) {
  const char* fn = "rus_rmsnorm_mx_fwd";
  if (int e = check_rows(fn, n_rows, n_cols)) return e;
  if (n_rows >= (int64_t(1) << 31))
    return fail(RUS_ERR_INVALID, "%s: n_rows=%lld must be below 2^31", fn, (long long)n_rows);
  if (stride_row < n_cols && n_rows > 1)
    return fail(RUS_ERR_INVALID, "%s: stride_row=%lld smaller than a row", fn, (long long)stride_row);
  if (dtype == RUS_DTYPE_BF16 || w_dtype == RUS_DTYPE_BF16)
    return fail(RUS_ERR_UNSUPPORTED, "%s: fp16 or fp32 activations and weights (as rus_rmsnorm_bwd)", fn);
  return with_type(fn, dtype, [&](auto t) -> int {
    return with_type(fn, w_dtype, [&](auto wt) -> int {
      typedef decltype(t) T;
      typedef decltype(wt) W;
      if constexpr (sizeof(t) == 2 && !__is_same(T, f16)) return RUS_ERR_UNSUPPORTED;
      else if constexpr (sizeof(wt) == 2 && !__is_same(W, f16)) return RUS_ERR_UNSUPPORTED;
      else {
        if (n_rows == 0) return RUS_OK;
        if (int e = check_mx(fn, codes, scales, RUS_MX_FP8, "output")) return e;
        if (!aligned(codes, 8) || !x || !weight || !rstd || !aligned(x, sizeof(T)) ||
            !aligned(weight, sizeof(W)) || !aligned(rstd, 4))
          return fail(RUS_ERR_INVALID, "%s: null or misaligned pointer", fn);
        if ((residual != nullptr) != (sum_out != nullptr))
          return fail(RUS_ERR_INVALID, "%s: residual and sum_out come together", fn);
        if (residual && (!aligned(residual, sizeof(T)) || !aligned(sum_out, sizeof(T))))
          return fail(RUS_ERR_INVALID, "%s: misaligned residual or sum_out", fn);
        const int nb = static_cast<int>(mx_blocks(n_cols));
        const int packs = nb * 4;
        // as few steps as 1024 threads allow, and equal ones
        const int steps = (packs + 1023) / 1024;
        const int threads = ((packs + steps - 1) / steps + 63) / 64 * 64;
        auto go = [&](auto k) {
          return by_rows(fn, n_rows, threads, [&](int64_t first, int64_t rows) {
            const int64_t at = first * stride_row;
            hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(rows)), dim3(threads), 0,
                               static_cast<hipStream_t>(stream), static_cast<const T*>(x) + at,
                               residual ? static_cast<const T*>(residual) + at : nullptr,
                               static_cast<const W*>(weight),
                               sum_out ? static_cast<T*>(sum_out) + at : nullptr,
                               static_cast<uint8_t*>(codes) + first * nb * kCodeBytes<kFp8>,
                               static_cast<uint8_t*>(scales) + first * nb, rstd + first,
                               static_cast<int>(n_cols), nb, stride_row, eps,
                               1.0 / static_cast<double>(n_cols));
          });
        };
        return residual ? go(rmsnorm_mx_kernel<T, W, true>) : go(rmsnorm_mx_kernel<T, W, false>);
      }
    });
  });
}
