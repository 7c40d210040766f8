// The product's gradient with respect to its activations: dx[m, k] = T(sum_n dy[m, n] T(W[n, k])), T
// dy's 16-bit type, W [n, k] in microscaled blocks along k. The contraction runs across W's blocks, so
// the scaled matrix instruction cannot apply their scales: W is decoded to T on its way into LDS and
// the product runs on v_mfma_f32_32x32x16_{f16,bf16}.
//
// Eight waves form a tile of TM tokens x 256 columns, the contraction staged 64 at a time through two
// LDS buffers. A stage's dy rows and W codes travel through registers one stage ahead: each of the 512
// threads loads one block of W (32 codes, its scale), decodes it with 16 of gfx950's scaled
// conversions and writes it transposed-readable; rows without alignment, and the contraction's end,
// are filled element by element on the same way. W's rows lie along the contraction, so its fragments
// leave LDS through the transposing ds_read_b64_tr_b16.
// A tile count below the chip's 256 CUs splits the contraction; the splits' fp32 sums are added in
// split order by a second launch.
#include <type_traits>

#include "mx.h"

namespace rus {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char* lds_ptr;

typedef u32x4s u32x4u __attribute__((aligned(2)));  // a 16-byte access at any alignment of elements

constexpr int kGradN = 256, kGradK = 64, kGradThreads = 512;
constexpr int kWRow = kGradN * 2;  // bytes of one contraction row of the W stage

struct GradArgs {
  const void* dy;
  int64_t ld_dy;
  const uint8_t *wc, *ws;
  int m, n, k, nb;   // tokens, contraction (rows of W), output columns, blocks of a row of W
  int tiles_m, tiles_k, splits, stages;  // stages of 64 rows of W, dealt evenly to the splits
  void* dx;          // [m, k], or the splits' fp32 sums [splits, m, k]
  int64_t ld_dx;
};

template <typename T>
struct Half8 {
  typedef T type __attribute__((ext_vector_type(8)));
};

template <typename T>
__device__ __forceinline__ f32x16 mma16(const u32x4s& a, const u32x4s& b, const f32x16& c) {
  typedef typename Half8<T>::type V;
  if constexpr (__is_same(T, f16))
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c,
                                                  0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b),
                                                   c, 0, 0, 0);
}

// Eight codes (one word of fp4, two of fp8) times 2^(scale - 127) as eight T, rounded once.
template <typename T, int FMT>
__device__ __forceinline__ u32x4s decode8(uint32_t lo, uint32_t hi, float s) {
  u32x4s o;
#define RUS_PAIR(W, I) \
  if constexpr (__is_same(T, f16)) { \
    if constexpr (FMT == kFp4) o[I] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(W, s, I)); \
    else o[I] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(W, s, I & 1)); \
  } else { \
    if constexpr (FMT == kFp4) o[I] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(W, s, I)); \
    else o[I] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(W, s, I & 1)); \
  }
  RUS_PAIR(lo, 0)
  RUS_PAIR(lo, 1)
  RUS_PAIR((FMT == kFp4 ? lo : hi), 2)
  RUS_PAIR((FMT == kFp4 ? lo : hi), 3)
#undef RUS_PAIR
  return o;
}

template <typename T, int FMT, int TM>
__global__ __launch_bounds__(kGradThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void
mx_grad_kernel(GradArgs g) {
  constexpr int WM = TM >= 128 ? 2 : 1, WN = 8 / WM;           // waves along tokens and columns
  constexpr int MT = TM / WM / 32, NT = kGradN / WN / 32;      // 32 x 32 results of a wave
  constexpr int AC = TM * 8 / kGradThreads;                    // 16-byte pieces of dy per thread
  constexpr int kABytes = TM * 128, kBBytes = kGradK * kWRow;
  constexpr int WV = FMT == kFp4 ? 1 : 2;
  __shared__ __attribute__((aligned(16))) char smem[2 * (kABytes + kBBytes)];
  const int total = g.tiles_m * g.tiles_k * g.splits;
  // Each XCD takes a run of work items: its tiles share rows of W (and of dy) in one L2.
  const int per = (total + 7) >> 3, work = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (static_cast<int>(blockIdx.x >> 3) >= per || work >= total) return;
  const int m0 = work % g.tiles_m * TM;
  const int c0 = work / g.tiles_m % g.tiles_k * kGradN;
  const int split = work / (g.tiles_m * g.tiles_k);
  const int s0 = static_cast<int>(static_cast<int64_t>(g.stages) * split / g.splits);
  const int s1 = static_cast<int>(static_cast<int64_t>(g.stages) * (split + 1) / g.splits);
  const int t = threadIdx.x, lane = t & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // dy: piece i of thread t is row (512 i + t) / 8, columns 8 (t % 8) of the stage, stored at chunk
  // (t % 8) ^ ((row / 2) % 8) of its 128-byte row: 16 neighbouring rows read at one chunk then cover
  // all banks once. Rows past the last re-read it.
  const T* dy = static_cast<const T*>(g.dy);
  int64_t arow[AC > 0 ? AC : 1];
  uint32_t aat[AC > 0 ? AC : 1];
  const bool has_a = AC > 0 || t < TM * 8;
#pragma unroll
  for (int i = 0; i < (AC > 0 ? AC : 1); ++i) {
    const int row = (512 * i + t) >> 3;
    arow[i] = static_cast<int64_t>(min(m0 + row, g.m - 1)) * g.ld_dy;
    aat[i] = row * 128 + (((t & 7) ^ ((row >> 1) & 7)) << 4);
  }
  // W: thread t's block is t % 8 of contraction row t / 8; its chunks of 8 columns j = 0..3 lie at chunk
  // (4 b + j) ^ ((row % 4) * 4) of the 512-byte row, written in an order that spreads 16 lanes over all
  // banks (chunk j ^ spread first).
  const int brow = t >> 3, bblk = t & 7;
  const int blk = min((c0 >> 5) + bblk, g.nb - 1);
  const int spread = (bblk >> 2) | ((brow & 1) << 1);
  const uint32_t bat = brow * kWRow + (((4 * bblk) ^ ((brow & 3) << 2)) << 4);

  u32x4s ra[AC > 0 ? AC : 1], rb[WV];
  uint32_t rs = 0;
  const int ragged = g.n & 7;
  auto load = [&](int s) {
    const int n0 = s * kGradK, n = n0 + 8 * (t & 7);
    if (has_a) {
      if (n0 + kGradK <= g.n || !ragged) {  // whole pieces, at any alignment (those past the end: `store`)
#pragma unroll
        for (int i = 0; i < (AC > 0 ? AC : 1); ++i)
          ra[i] = *reinterpret_cast<const u32x4u*>(dy + arow[i] + (n < g.n ? n : 0));
      } else {
#pragma unroll
        for (int i = 0; i < (AC > 0 ? AC : 1); ++i) {
          Pack<T, 8> p;
#pragma unroll
          for (int j = 0; j < 8; ++j) p.v[j] = n + j < g.n ? dy[arow[i] + n + j] : static_cast<T>(0.0f);
          ra[i] = __builtin_bit_cast(u32x4s, p);
        }
      }
    }
    const int64_t at = static_cast<int64_t>(min(n0 + brow, g.n - 1)) * g.nb + blk;
    const u32x4s* src = reinterpret_cast<const u32x4s*>(g.wc + at * kCodeBytes<FMT>);
#pragma unroll
    for (int v = 0; v < WV; ++v) rb[v] = src[v];
    rs = g.ws[at];
  };
  auto store = [&](int s, int buf) {  // stage s, in registers, to LDS; zeros past the contraction's end
    char* base = smem + buf * (kABytes + kBBytes);
    const bool a_in = s * kGradK + 8 * (t & 7) < g.n, b_in = s * kGradK + brow < g.n;
    if (has_a) {
#pragma unroll
      for (int i = 0; i < (AC > 0 ? AC : 1); ++i)
        *reinterpret_cast<u32x4s*>(base + aat[i]) = a_in ? ra[i] : u32x4s{0, 0, 0, 0};
    }
    const float scale = b_in ? mx_scale(rs) : 1.0f;
#pragma unroll
    for (int v = 0; v < WV; ++v) rb[v] = b_in ? rb[v] : u32x4s{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int q = j ^ spread;
      uint32_t lo, hi = 0;
      if constexpr (FMT == kFp4) {
        lo = q & 2 ? (q & 1 ? rb[0].w : rb[0].z) : (q & 1 ? rb[0].y : rb[0].x);
      } else {
        const u32x4s w = q & 2 ? rb[WV - 1] : rb[0];
        lo = q & 1 ? w.z : w.x;
        hi = q & 1 ? w.w : w.y;
      }
      *reinterpret_cast<u32x4s*>(base + kABytes + bat + q * 16) = decode8<T, FMT>(lo, hi, scale);
    }
  };

  // Fragments. dy: row wm * (TM / WM) + 32 mt + l % 32, chunk 2 kk + l / 32. W: lane l (j = l % 16)
  // points at row 16 kk + 8 (l / 32) + j / 4 (+ 4 for the upper half), columns 16 ((l / 16) % 2) +
  // 4 (j % 4) of its 32; the transposing read hands lane i column i of the 16.
  const int arow_f = wm * (TM / WM) + (lane & 31);
  const uint32_t af = arow_f * 128, asw = (arow_f >> 1) & 7;
  const int j16 = lane & 15;
  uint32_t bf[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int col = wn * (kGradN / WN) + nt * 32 + 16 * ((lane >> 4) & 1) + 4 * (j16 & 3);
    bf[nt] = (8 * half + (j16 >> 2)) * kWRow + (((col >> 3) ^ ((j16 >> 2) << 2)) << 4) + (col & 7) * 2;
  }
  f32x16 acc[MT][NT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = f32x16{};

  // Two sets of fragments: one step's are read while the other's products run.
  struct Frags {
    u32x4s a[MT], b[NT];
  };
  auto read = [&](Frags& f, int buf, int kk) {
    const char* base = smem + buf * (kABytes + kBBytes);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      f.a[mt] = *reinterpret_cast<const u32x4s*>(base + af + mt * 4096 + (((2 * kk + half) ^ asw) << 4));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      lds_ptr p = (lds_ptr)(base + kABytes) + bf[nt] + kk * 16 * kWRow;
      typedef __attribute__((address_space(3))) s16x4* vec_ptr;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((vec_ptr)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((vec_ptr)(p + 4 * kWRow));
      const u32x2s l2 = __builtin_bit_cast(u32x2s, lo), h2 = __builtin_bit_cast(u32x2s, hi);
      f.b[nt] = u32x4s{l2.x, l2.y, h2.x, h2.y};
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto mma = [&](const Frags& f) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = mma16<T>(f.a[mt], f.b[nt], acc[mt][nt]);
    __builtin_amdgcn_sched_barrier(0);
  };

  load(s0);
  store(s0, 0);
  if (s0 + 1 < s1) load(s0 + 1);
  __syncthreads();
  Frags f0, f1;
  read(f0, 0, 0);
  for (int s = s0; s < s1; ++s) {
    const int buf = (s - s0) & 1;
    read(f1, buf, 1);
    mma(f0);
    read(f0, buf, 2);
    // Stage s + 1 goes into the buffer whose last reads the barrier of stage s - 1 ended.
    if (s + 1 < s1) store(s + 1, buf ^ 1);
    if (s + 2 < s1) load(s + 2);
    mma(f1);
    read(f1, buf, 3);
    mma(f0);
    __syncthreads();
    if (s + 1 < s1) read(f0, buf ^ 1, 0);
    mma(f1);
  }

  auto write = [&](auto put) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = c0 + wn * (kGradN / WN) + nt * 32 + (lane & 31);
      if (col >= g.k) continue;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = m0 + wm * (TM / WM) + mt * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
          if (row < g.m) put(row, col, acc[mt][nt][r]);
        }
    }
  };
  if (g.splits > 1) {
    float* parts = static_cast<float*>(g.dx) + static_cast<int64_t>(split) * g.m * g.k;
    write([&](int row, int col, float v) { parts[static_cast<int64_t>(row) * g.k + col] = v; });
  } else {
    T* dx = static_cast<T*>(g.dx);
    write([&](int row, int col, float v) { dx[row * g.ld_dx + col] = from_f32<T>(v); });
  }
}

// dx = T(the splits' sums, added in order), V columns per thread.
template <typename T, int V>
__global__ __launch_bounds__(256) void mx_grad_sum_kernel(const float* __restrict__ parts, int splits,
                                                          int64_t m, int packs, int k,
                                                          T* __restrict__ dx, int64_t ld_dx) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= m * packs) return;
  const int64_t row = i / packs;
  const int c = static_cast<int>(i - row * packs) * V;
  const float* p = parts + row * k + c;
  float v[V];
  load_f32<float, V>(p, v);
#pragma unroll 8
  for (int s = 1; s < splits; ++s) {
    float u[V];
    load_f32<float, V>(p + s * m * k, u);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += u[j];
  }
  store_from_f32<T, V>(dx + row * ld_dx + c, v);
}

// The tile height and the number of splits for a shape. A stage of a 256-token tile takes about 2 us on
// a CU, of a lower tile in proportion to its tokens but at least 0.5 (the decode); a split's sums cost
// 8 bytes per value written and read again.
struct GradPlan {
  int tm, splits;
};

GradPlan grad_plan(int64_t m, int64_t n, int64_t k) {
  const int64_t stages = (n + kGradK - 1) / kGradK, tk = (k + kGradN - 1) / kGradN;
  GradPlan best{256, 1};
  double least = 1e30;
  for (int tm : {256, 128, 64, 32}) {
    const int64_t tiles = (m + tm - 1) / tm * tk;
    const double stage = tm == 256 ? 2.0 : tm == 128 ? 1.1 : tm == 64 ? 0.7 : 0.5;
    for (int64_t s = 1; s <= 64 && s <= stages; ++s) {
      const double rounds = static_cast<double>((tiles * s + 255) / 256);
      const double us = rounds * (static_cast<double>((stages + s - 1) / s) * stage + 3.0) +
                        (s > 1 ? 4.0 + 8e-6 * static_cast<double>(s * m * k) / 4.0 : 0.0);
      if (us < least) {
        least = us;
        best = {tm, static_cast<int>(s)};
      }
    }
  }
  return best;
}

}  // namespace
}  // namespace rus

using namespace rus;

extern "C" int rus_mx_gemm_t_workspace(int64_t m, int64_t n, int64_t k, int64_t* floats) {
  const char* fn = "rus_mx_gemm_t_workspace";
  if (!floats) return fail(RUS_ERR_INVALID, "%s: null result", fn);
  if (m < 0 || n <= 0 || k <= 0 || m >= (1 << 30) || n >= (1 << 28) || k > (1 << 28))
    return fail(RUS_ERR_INVALID, "%s: bad sizes m=%lld n=%lld k=%lld", fn, (long long)m,
                (long long)n, (long long)k);
  const GradPlan p = grad_plan(m, n, k);
  *floats = p.splits > 1 ? p.splits * m * k : 0;
  return RUS_OK;
}

extern "C" int rus_mx_gemm_t(const void* dy, int64_t stride_dy, int32_t dtype, const void* w_codes,
                             const void* w_scales, int32_t w_fmt, int64_t m, int64_t n, int64_t k,
                             void* dx, int64_t stride_dx, float* workspace, int64_t n_workspace,
                             void* stream) {
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
  const GradPlan plan = grad_plan(m, n, k);
  const bool split = plan.splits > 1;
  if (split && (n_workspace < plan.splits * m * k || !workspace || !aligned(workspace, 16)))
    return fail(RUS_ERR_INVALID, "%s: workspace holds %lld floats (16-byte aligned), needs %lld", fn,
                (long long)n_workspace, (long long)(plan.splits * m * k));
  GradArgs g;
  g.dy = dy;
  g.ld_dy = stride_dy;
  g.wc = static_cast<const uint8_t*>(w_codes);
  g.ws = static_cast<const uint8_t*>(w_scales);
  g.m = static_cast<int>(m);
  g.n = static_cast<int>(n);
  g.k = static_cast<int>(k);
  g.nb = static_cast<int>(mx_blocks(k));
  const int64_t tiles = ((m + plan.tm - 1) / plan.tm) * ((k + kGradN - 1) / kGradN);
  if (tiles * plan.splits >= (int64_t(1) << 30))
    return fail(RUS_ERR_UNSUPPORTED, "%s: m=%lld x k=%lld is beyond 2^30 tiles", fn, (long long)m,
                (long long)k);
  g.tiles_m = static_cast<int>((m + plan.tm - 1) / plan.tm);
  g.tiles_k = static_cast<int>((k + kGradN - 1) / kGradN);
  g.splits = plan.splits;
  g.stages = static_cast<int>((n + kGradK - 1) / kGradK);
  g.dx = split ? static_cast<void*>(workspace) : dx;
  g.ld_dx = stride_dx;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(8 * ((tiles * plan.splits + 7) / 8)));
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(kGradThreads), 0, st, g); };
  auto tile = [&](auto t, auto fmt) {
    typedef decltype(t) T;
    constexpr int F = decltype(fmt)::value;
    switch (plan.tm) {
      case 256:
        return go(mx_grad_kernel<T, F, 256>);
      case 128:
        return go(mx_grad_kernel<T, F, 128>);
      case 64:
        return go(mx_grad_kernel<T, F, 64>);
      default:
        return go(mx_grad_kernel<T, F, 32>);
    }
  };
  auto types = [&](auto t) {
    typedef decltype(t) T;
    if (w_fmt == RUS_MX_FP4)
      tile(t, std::integral_constant<int, kFp4>{});
    else
      tile(t, std::integral_constant<int, kFp8>{});
    if (!split) return;
    const bool wide = k % 4 == 0 && stride_dx % 4 == 0 && aligned(dx, 8);
    const int packs = static_cast<int>(wide ? k / 4 : k);
    const dim3 sum(static_cast<unsigned>((m * packs + 255) / 256));
    if (wide)
      hipLaunchKernelGGL((mx_grad_sum_kernel<T, 4>), sum, dim3(256), 0, st, workspace, plan.splits, m,
                         packs, g.k, static_cast<T*>(dx), stride_dx);
    else
      hipLaunchKernelGGL((mx_grad_sum_kernel<T, 1>), sum, dim3(256), 0, st, workspace, plan.splits, m,
                         packs, g.k, static_cast<T*>(dx), stride_dx);
  };
  if (dtype == RUS_DTYPE_F16)
    types(f16{});
  else
    types(bf16{});
  return check_launch(fn);
}
