// Microscaled blocks: 32 elements along a row share one power-of-two scale (E8M0 byte b: 2^(b-127),
// 255 = NaN), each element in e2m1 (4 bits, two to a byte, the even element in the low half) or e4m3
// (8 bits). A stored row is padded to whole groups of four blocks: [rows, nb] scales and [rows, 16 nb]
// or [rows, 32 nb] code bytes, nb = 4 ceil(cols / 128), codes and scales of the padding zero, so the
// products have no tail along the contraction and read scales as aligned 32-bit words.
//
// Rounding to a block: b = E - emax, E the biased exponent of the block's largest |x| (as fp32) and
// emax that of the format's largest binade (2 / 8), at least 0; the elements are x 2^(127-b), exact in
// fp32, clamped to the format's largest value and rounded to nearest even by the hardware conversion.
// A block that holds an infinity or a NaN is NaN as a whole (scale 255).
#pragma once

#include <type_traits>
#include <utility>

#include "common.h"

namespace rus {

// rus_mx_quantize, for entry points that quantise what they are given.
int quantize_rows(const char* fn, const void* x, int32_t dtype, int64_t n_rows, int64_t n_cols,
                  int64_t stride_row, int32_t fmt, void* codes, void* scales, hipStream_t stream);

// The products' kernel for a few tokens, x in blocks (xc, xs) or rounded to them (x, rows of the result's
// type). few_tokens: whether it takes these sizes; nothing else is checked here.
struct TokenArgs {
  const void* x;
  int64_t ldx;
  const uint8_t *xc, *xs, *wc, *ws;
  int x_fmt, m, n, k, nb;
  const void* bias;
  void* y;
  int64_t ldy;
};
enum { kTokenPlain = 0, kTokenGlu = 1 };
bool few_tokens(int64_t m, int64_t n, int64_t nb);
int token_product(const char* fn, const TokenArgs& g, int w_fmt, bool glu, bool bf, hipStream_t st);

namespace {

constexpr int kFp4 = RUS_MX_FP4, kFp8 = RUS_MX_FP8;
constexpr int kMxBlock = 32;

typedef __bf16 bf16;
typedef float f32x2 __attribute__((ext_vector_type(2)));

template <int FMT>
constexpr int kCodeBytes = FMT == kFp4 ? 16 : 32;  // code bytes of a block
template <int FMT>
constexpr int kEmax = FMT == kFp4 ? 2 : 8;

__host__ __device__ inline int64_t mx_blocks(int64_t cols) { return (cols + 127) / 128 * 4; }

// 2^(b - 127), NaN for 255.
__device__ __forceinline__ float mx_scale(uint32_t b) {
  const uint32_t bits = b == 0 ? 0x00400000u : (b == 255 ? 0x7fc00000u : b << 23);
  return __builtin_bit_cast(float, bits);
}

__device__ __forceinline__ uint32_t abs_bits(float x) {
  return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
}

// The scale byte of a block whose largest |x| has the fp32 bits `top` (255: not finite).
template <int FMT>
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  const int b = static_cast<int>(top >> 23) - kEmax<FMT>;
  return static_cast<uint32_t>(b < 0 ? 0 : b);
}

// 2^(127 - b) for a finite block (b <= 252).
__device__ __forceinline__ float inv_scale(uint32_t b) {
  return __builtin_bit_cast(float, (254u - b) << 23);
}

// The largest of the four lanes that share a block.
__device__ __forceinline__ uint32_t quad_max(uint32_t m) {
  m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 1, kWave)));
  return max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 2, kWave)));
}

// N (a multiple of 4 / 8) scaled elements to codes, in order; `nan`: the block is not finite.
template <int N>
__device__ __forceinline__ void to_fp8(const float (&v)[N], bool nan, uint32_t (&out)[N / 4]) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    float c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = __builtin_amdgcn_fmed3f(v[4 * i + j], -448.0f, 448.0f);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], w, true);
    out[i] = nan ? 0x7f7f7f7fu : static_cast<uint32_t>(w);
  }
}
template <int N>
__device__ __forceinline__ void to_fp4(const float (&v)[N], bool nan, uint32_t (&out)[N / 8]) {
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
    const float* p = &v[8 * i];
    uint32_t w = 0;  // the conversion saturates
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, p[0], p[1], 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, p[2], p[3], 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, p[4], p[5], 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, p[6], p[7], 1.0f, 3);
    out[i] = nan ? 0u : w;
  }
}

// Eight codes to fp32, times `s`.
__device__ __forceinline__ void from_fp8(uint32_t lo, uint32_t hi, float s, float (&v)[8]) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(lo, false);
  const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(lo, true);
  const f32x2 c = __builtin_amdgcn_cvt_pk_f32_fp8(hi, false);
  const f32x2 d = __builtin_amdgcn_cvt_pk_f32_fp8(hi, true);
  const float e[8] = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = e[i] * s;
}
__device__ __forceinline__ void from_fp4(uint32_t w, float s, float (&v)[8]) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
  const float e[8] = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = e[i] * s;
}

// f(0), f(1), .. f(N - 1) as compile-time constants.
template <typename F, int... I>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F f) {
  each_of(f, std::make_integer_sequence<int, N>{});
}

// The sum of `parts` groups of V floats, `step` apart, added in order. DEEP: sixteen loads at a time, for
// few sums of many parts, which take a few rounds of the latency from other XCDs' caches (28 parts of
// 16 x 1,536: 5.4 us by eights, 3.7 by sixteens, as 32 parts take); many sums are better served by more
// waves with fewer registers (5 parts of 4,096 x 1,536: 21 us, by sixteens 27).
template <bool DEEP, int V>
__device__ __forceinline__ void sum_parts(const float* __restrict__ p, int64_t step, int parts, float (&v)[V]) {
  load_f32<float, V>(p, v);
  if constexpr (DEEP) {
    constexpr int N = 16;
    for (int s = 1; s < parts; s += N) {
      float u[N][V];
#pragma unroll
      for (int i = 0; i < N; ++i) load_f32<float, V>(p + min(s + i, parts - 1) * step, u[i]);
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = s + i < parts ? v[j] + u[i][j] : v[j];
    }
  } else {
#pragma unroll 8
    for (int s = 1; s < parts; ++s) {
      float u[V];
      load_f32<float, V>(p + s * step, u);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += u[j];
    }
  }
}
// Whether a sum of that many threads is of the first kind.
inline bool deep_sum(int64_t threads, int64_t parts) { return threads <= 32768 && parts > 8; }

// A dispatch counts its work-items in 32 bits.
constexpr int64_t kMaxItems = int64_t(1) << 32;
inline int check_items(const char* fn, int64_t workgroups, int64_t threads) {
  if (workgroups * threads < kMaxItems) return RUS_OK;
  return fail(RUS_ERR_UNSUPPORTED, "%s: %lld workgroups of %lld are beyond one dispatch", fn,
              (long long)workgroups, (long long)threads);
}

// launch(first, count) for slices of the rows that a dispatch holds: one, below 2^31 work-items.
template <typename F>
int by_rows(const char* fn, int64_t rows, int64_t threads_per_row, F launch) {
  const int64_t most = (kMaxItems / 2 + threads_per_row - 1) / threads_per_row;
  for (int64_t first = 0; first < rows; first += most) {
    launch(first, rows - first < most ? rows - first : most);
    if (int e = check_launch(fn)) return e;
  }
  return RUS_OK;
}

// A thread's last plans by the sizes they are for: finding one goes over all choices, a few us.
template <typename Plan>
class PlanMemo {
 public:
  struct Key {
    int64_t a, b, c, d;
  };
  template <typename F>
  Plan get(const Key& k, F find) {
    const uint64_t h = (static_cast<uint64_t>(k.a) * 0x9e3779b97f4a7c15u + static_cast<uint64_t>(k.b)) *
                           0x9e3779b97f4a7c15u + static_cast<uint64_t>(k.c) * 31u + static_cast<uint64_t>(k.d);
    Slot& s = slots_[(h >> 32) % kSlots];
    if (!s.used || s.key.a != k.a || s.key.b != k.b || s.key.c != k.c || s.key.d != k.d)
      s = {true, k, find()};
    return s.plan;
  }

 private:
  static constexpr int kSlots = 64;
  struct Slot {
    bool used = false;
    Key key{};
    Plan plan{};
  } slots_[kSlots];
};

inline int check_format(const char* fn, int32_t fmt, const char* name) {
  if (fmt == RUS_MX_FP4 || fmt == RUS_MX_FP8) return RUS_OK;
  return fail(RUS_ERR_INVALID, "%s: %s has unknown format %d", fn, name, (int)fmt);
}

// The checks every entry point makes of a block operand.
inline int check_mx(const char* fn, const void* codes, const void* scales, int32_t fmt,
                    const char* name) {
  if (int e = check_format(fn, fmt, name)) return e;
  if (!codes || !scales || !aligned(codes, 16) || !aligned(scales, 4))
    return fail(RUS_ERR_INVALID, "%s: %s codes / scales null or misaligned (16 / 4 bytes)", fn, name);
  return RUS_OK;
}

}  // namespace
}  // namespace rus
