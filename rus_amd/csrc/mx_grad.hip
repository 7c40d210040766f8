// The product's gradient with respect to its activations: dx[m, k] = T(sum_n dy[m, n] T(W[n, k])), T
// dy's 16-bit type, W [n, k] in microscaled blocks along k. The contraction runs across W's blocks, so
// their scales cannot be applied by the scaled matrix instruction: W is decoded to T as it is read and
// the product runs on v_mfma_f32_32x32x16_{f16,bf16}.
#include "mx.h"

namespace rus {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct GradArgs {
  const void* dy;
  int64_t ld_dy;
  const uint8_t *wc, *ws;
  int m, n, k, nb;  // tokens, contraction (rows of W), output columns, blocks of a row of W
  void* dx;
  int64_t ld_dx;
};

template <int FMT>
__device__ __forceinline__ float code_value(const uint8_t* row, int c) {
  if constexpr (FMT == kFp4) {
    const uint32_t b = row[c >> 1] >> (4 * (c & 1));
    const f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 1.0f, 0);
    return v.x;
  } else {
    return __builtin_amdgcn_cvt_f32_fp8(row[c], 0);
  }
}

// One wave: 32 tokens x 32 columns.
template <typename T, int FMT>
__global__ __launch_bounds__(kWave) void mx_grad_kernel(GradArgs g) {
  const int lane = threadIdx.x, half = lane >> 5;
  const int c0 = blockIdx.x * 32, t0 = blockIdx.y * 32;
  const int t = min(t0 + (lane & 31), g.m - 1), c = min(c0 + (lane & 31), g.k - 1);
  const T* dy = static_cast<const T*>(g.dy) + t * g.ld_dy;
  f32x16 acc = {};
  for (int n0 = 0; n0 < g.n; n0 += 16) {
    T a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = n0 + 8 * half + i;
      const int64_t r = static_cast<int64_t>(min(n, g.n - 1)) * g.nb;
      const float w = code_value<FMT>(g.wc + r * kCodeBytes<FMT>, c) * mx_scale(g.ws[r + (c >> 5)]);
      a[i] = n < g.n ? dy[n] : static_cast<T>(0.0f);
      b[i] = from_f32<T>(n < g.n ? w : 0.0f);
    }
    if constexpr (__is_same(T, f16))
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, b),
                                                   __builtin_bit_cast(f16x8, a), acc, 0, 0, 0);
    else
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, b),
                                                    __builtin_bit_cast(bf16x8, a), acc, 0, 0, 0);
  }
  if (t0 + (lane & 31) >= g.m) return;
  T* o = static_cast<T*>(g.dx) + t * g.ld_dx;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int col = c0 + 8 * (r >> 2) + 4 * half + (r & 3);
    if (col < g.k) o[col] = from_f32<T>(acc[r]);
  }
}

}  // namespace
}  // namespace rus

using namespace rus;

extern "C" int rus_mx_gemm_t(const void* dy, int64_t stride_dy, int32_t dtype, const void* w_codes,
                             const void* w_scales, int32_t w_fmt, int64_t m, int64_t n, int64_t k,
                             void* dx, int64_t stride_dx, void* stream) {
  const char* fn = "rus_mx_gemm_t";
  if (m < 0 || n <= 0 || k <= 0 || m >= (1 << 30) || n >= (1 << 28) || k > (1 << 28))
    return fail(RUS_ERR_INVALID, "%s: bad sizes m=%lld n=%lld k=%lld", fn, (long long)m,
                (long long)n, (long long)k);
  if (dtype != RUS_DTYPE_F16 && dtype != RUS_DTYPE_BF16)
    return fail(RUS_ERR_UNSUPPORTED, "%s: gradients are fp16 or bf16, not dtype %d", fn, (int)dtype);
  if ((stride_dy < n || stride_dx < k) && m > 1)
    return fail(RUS_ERR_INVALID, "%s: row strides dy=%lld dx=%lld too small", fn,
                (long long)stride_dy, (long long)stride_dx);
  if (m == 0) return RUS_OK;
  if (int e = check_mx(fn, w_codes, w_scales, w_fmt, "w")) return e;
  if (!dy || !dx || !aligned(dy, 2) || !aligned(dx, 2))
    return fail(RUS_ERR_INVALID, "%s: dy / dx null or misaligned", fn);
  if ((m + 31) / 32 > 65535)
    return fail(RUS_ERR_UNSUPPORTED, "%s: m=%lld is beyond 65535 tiles of 32 tokens", fn, (long long)m);
  GradArgs g;
  g.dy = dy;
  g.ld_dy = stride_dy;
  g.wc = static_cast<const uint8_t*>(w_codes);
  g.ws = static_cast<const uint8_t*>(w_scales);
  g.m = static_cast<int>(m);
  g.n = static_cast<int>(n);
  g.k = static_cast<int>(k);
  g.nb = static_cast<int>(mx_blocks(k));
  g.dx = dx;
  g.ld_dx = stride_dx;
  const dim3 grid((g.k + 31) / 32, (g.m + 31) / 32);
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, dim3(kWave), 0, static_cast<hipStream_t>(stream), g);
  };
  if (dtype == RUS_DTYPE_F16) {
    if (w_fmt == RUS_MX_FP4) go(mx_grad_kernel<f16, kFp4>);
    else go(mx_grad_kernel<f16, kFp8>);
  } else {
    if (w_fmt == RUS_MX_FP4) go(mx_grad_kernel<bf16, kFp4>);
    else go(mx_grad_kernel<bf16, kFp8>);
  }
  return check_launch(fn);
}
