// Rows to microscaled blocks and back, and the residual + RMSNorm whose output is such blocks.
#include "mx.h"

namespace rus {
namespace {

// Eight elements of a row from column c on, zeros from `cols` on.
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int c, int cols, bool vec,
                                      float (&v)[8]) {
  if (vec && c + 8 <= cols) {
    load_f32<T, 8>(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? static_cast<float>(row[c + i]) : 0.0f;
  }
}

// The largest of the four lanes that share a block.
__device__ __forceinline__ uint32_t quad_max(uint32_t m) {
  m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 1, kWave)));
  return max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 2, kWave)));
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

// Thread = eight elements, four neighbouring lanes = one block.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, int64_t stride,
                                                          int cols, int nb, int64_t total,
                                                          bool vec, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;  // whole blocks leave together: total is a multiple of 16
  const int64_t row = i / (nb * 4);
  const int p = static_cast<int>(i - row * (nb * 4));
  float v[8];
  load8<T>(x + row * stride, p * 8, cols, vec, v);
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
                                                            int64_t total, bool vec,
                                                            T* __restrict__ out, int64_t stride) {
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
  T* o = out + row * stride + p * 8;
  if (vec && p * 8 + 8 <= cols) {
    store_from_f32<T, 8>(o, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (p * 8 + j < cols) o[j] = from_f32<T>(v[j]);
  }
}

// ---- residual + RMSNorm into fp8 blocks ----------------------------------------------------------
//
// h = T(x + res), y = h rstd w, and y's blocks. The normalised value is rounded once, from 64 bits to
// the 8-bit element: the element type has few values, and a sum of squares or a product rounded in
// fp32 first would put a y next to a border between two of them (or next to a power of two that
// changes the block's scale) on either side of it depending on the order of the sum. fp64 runs at
// half the fp32 rate on this chip, which a kernel bound by memory does not notice.

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
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

// One workgroup per row, eight columns per thread and step.
template <typename T, typename W, bool HAS_RES>
__global__ __launch_bounds__(1024) void rmsnorm_mx_kernel(
    const T* __restrict__ x, const T* __restrict__ res, const W* __restrict__ w, T* sum_out,
    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, float* __restrict__ rstd, int cols,
    int nb, int64_t stride, float eps, bool vec, bool wvec) {
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
    load8<T>(xr, c, cols, vec, h);
    if (HAS_RES) {
      float r[8];
      load8<T>(rr, c, cols, vec, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = round_to<T>(h[i] + r[i]);
      if (vec && c + 8 <= cols) {
        store_from_f32<T, 8>(sr + c, h);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < cols) sr[c + i] = from_f32<T>(h[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += static_cast<double>(h[i]) * static_cast<double>(h[i]);
  }
  ss = wave_sum64(ss);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
  __syncthreads();
  double all = 0.0;
  for (int i = 0; i < nt / kWave; ++i) all += red[i];
  const double r = 1.0 / __builtin_sqrt(all / cols + static_cast<double>(eps));
  if (threadIdx.x == 0) rstd[row] = static_cast<float>(r);
  const bool kept = packs <= nt;  // the row is still in h
  for (int p = threadIdx.x; p < packs; p += nt) {
    const int c = p * 8;
    if (!kept) load8<T>(HAS_RES ? sr : xr, c, cols, vec, h);  // this thread wrote these itself
    float wv[8];
    load8<W>(w, c, cols, wvec, wv);
    double y[8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = static_cast<double>(h[i]) * r * static_cast<double>(wv[i]);
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
    store_codes<kFp8>(codes + (row * packs + p) * 8, v, nan);
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
    const int64_t total = n_rows * nb * 4;
    const bool vec = aligned(x, 16) && (stride_row * sizeof(T)) % 16 == 0;
    const dim3 grid(static_cast<unsigned>((total + 255) / 256));
    auto go = [&](auto k) {
      hipLaunchKernelGGL(k, grid, dim3(256), 0, stream, static_cast<const T*>(x), stride_row,
                         static_cast<int>(n_cols), nb, total, vec, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales));
    };
    if (fmt == RUS_MX_FP4)
      go(mx_quantize_kernel<T, kFp4>);
    else
      go(mx_quantize_kernel<T, kFp8>);
    return check_launch(fn);
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
    const int64_t total = n_rows * packs;
    const bool vec = aligned(out, 16) && (stride_row * sizeof(T)) % 16 == 0;
    const dim3 grid(static_cast<unsigned>((total + 255) / 256));
    auto go = [&](auto k) {
      hipLaunchKernelGGL(k, grid, dim3(256), 0, static_cast<hipStream_t>(stream),
                         static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales),
                         static_cast<int>(n_cols), nb, packs, total, vec, static_cast<T*>(out),
                         stride_row);
    };
    if (fmt == RUS_MX_FP4)
      go(mx_dequantize_kernel<T, kFp4>);
    else
      go(mx_dequantize_kernel<T, kFp8>);
    return check_launch(fn);
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
        const bool vec = aligned(x, 16) && (stride_row * sizeof(T)) % 16 == 0 &&
                         (!residual || (aligned(residual, 16) && aligned(sum_out, 16)));
        const int packs = nb * 4;
        const int threads = packs >= 1024 ? 1024 : (packs + 63) / 64 * 64;
        auto go = [&](auto k) {
          hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(n_rows)), dim3(threads), 0,
                             static_cast<hipStream_t>(stream), static_cast<const T*>(x),
                             static_cast<const T*>(residual), static_cast<const W*>(weight),
                             static_cast<T*>(sum_out), static_cast<uint8_t*>(codes),
                             static_cast<uint8_t*>(scales), rstd, static_cast<int>(n_cols), nb,
                             stride_row, eps, vec, aligned(weight, 16));
        };
        if (residual)
          go(rmsnorm_mx_kernel<T, W, true>);
        else
          go(rmsnorm_mx_kernel<T, W, false>);
        return check_launch(fn);
      }
    });
  });
}
