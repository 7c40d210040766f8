// The product's gradient with respect to its activations: dx[m, k] = T(sum_n dy[m, n] T(W[n, k])), T
// dy's 16-bit type, W [n, k] in microscaled blocks along k. The contraction runs across W's blocks, so
// the scaled matrix instruction cannot apply their scales: W is decoded to T on its way into LDS and
// the product runs on v_mfma_f32_32x32x16_{f16,bf16}.
//
// Eight waves form a tile of TM tokens x 256 columns, the contraction staged 64 at a time through two
// LDS buffers. A stage's dy rows and W codes travel through registers one stage ahead: each of the 512
// threads loads one block of W (32 codes, its scale), decodes it with 16 of gfx950's scaled
// conversions and writes it transposed-readable; rows of any alignment, and the contraction's end, come
// in on the same way. W's rows lie along the contraction, so its fragments leave LDS through the
// transposing ds_read_b64_tr_b16. Reads, decoding, writes and loads go out between the products: bound by
// the matrix pipe and its clock (2,048 x 17,920 x 1,536 bf16: 96 us on the same operands each call, 113 on
// three sets in turn, 1.17 and 1.0 PFLOP/s, where a library product of 8192^3 reaches 1.2; 11 for the sums).
// A tile count below the chip's 256 CUs splits the contraction; the splits' fp32 sums are added in
// split order by a second launch.
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
  const bool has_a = AC > 0 || t < TM * 8;  // (uniform over a wave)
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

  constexpr int AP = AC > 0 ? AC : 1;  // pieces of dy per thread (a tile of 32 rows: half the threads have one)
  u32x4s ra[AP], rb[WV];
  uint32_t rs = 0;
  // What a thread has of stage s: its pieces of dy (I < AP; columns past the end: `put`), its block of W.
  auto load_piece = [&](int s, int i) {
    const int n = s * kGradK + 8 * (t & 7);
    ra[i] = *reinterpret_cast<const u32x4u*>(dy + arow[i] + (n + 8 <= g.n ? n : 0));
  };
  auto load_block = [&](int s) {
    const int64_t at = static_cast<int64_t>(min(s * kGradK + brow, g.n - 1)) * g.nb + blk;
    const u32x4s* src = reinterpret_cast<const u32x4s*>(g.wc + at * kCodeBytes<FMT>);
#pragma unroll
    for (int v = 0; v < WV; ++v) rb[v] = src[v];
    rs = g.ws[at];
  };
  auto load = [&](int s) {
    if (has_a) {
      if ((s + 1) * kGradK <= g.n) {
#pragma unroll
        for (int i = 0; i < AP; ++i) load_piece(s, i);
      } else {  // the contraction's end inside the stage: element by element
        const int n = s * kGradK + 8 * (t & 7);
#pragma unroll
        for (int i = 0; i < AP; ++i) {
          Pack<T, 8> p;
#pragma unroll
          for (int j = 0; j < 8; ++j) p.v[j] = n + j < g.n ? dy[arow[i] + n + j] : static_cast<T>(0.0f);
          ra[i] = __builtin_bit_cast(u32x4s, p);
        }
      }
    }
    load_block(s);
  };
  // Piece I of stage s, in registers, to LDS: dy's, then the block's four chunks, decoded. WHOLE: the stage
  // does not reach past the contraction's end (else zeros there, on both sides: no value of W matters).
  auto put = [&](int s, int buf, auto I, auto WHOLE) {
    constexpr int i = decltype(I)::value;
    char* base = smem + buf * (kABytes + kBBytes);
    if constexpr (i < AP) {
      if (has_a) *reinterpret_cast<u32x4s*>(base + aat[i]) = ra[i];
    } else {
      constexpr int j = i - AP;
      const bool in = decltype(WHOLE)::value || s * kGradK + brow < g.n;
      const float scale = in ? mx_scale(rs) : 1.0f;
      const int q = j ^ spread;
      uint32_t lo, hi = 0;
      if constexpr (FMT == kFp4) {
        lo = q & 2 ? (q & 1 ? rb[0].w : rb[0].z) : (q & 1 ? rb[0].y : rb[0].x);
      } else {
        const u32x4s w = q & 2 ? rb[WV - 1] : rb[0];
        lo = q & 1 ? w.z : w.x;
        hi = q & 1 ? w.w : w.y;
      }
      if (!in) lo = hi = 0;
      *reinterpret_cast<u32x4s*>(base + kABytes + bat + q * 16) = decode8<T, FMT>(lo, hi, scale);
    }
  };
  constexpr int kPieces = AP + 4;

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
  constexpr int kMma = MT * NT, kReads = MT + NT;
  auto read_one = [&](Frags& f, int buf, int kk, auto R) {
    constexpr int r = decltype(R)::value;
    const char* base = smem + buf * (kABytes + kBBytes);
    if constexpr (r < MT) {
      f.a[r] = *reinterpret_cast<const u32x4s*>(base + af + r * 4096 + (((2 * kk + half) ^ asw) << 4));
    } else {
      lds_ptr p = (lds_ptr)(base + kABytes) + bf[r - MT] + kk * 16 * kWRow;
      typedef __attribute__((address_space(3))) s16x4* vec_ptr;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((vec_ptr)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((vec_ptr)(p + 4 * kWRow));
      const u32x2s l2 = __builtin_bit_cast(u32x2s, lo), h2 = __builtin_bit_cast(u32x2s, hi);
      f.b[r - MT] = u32x4s{l2.x, l2.y, h2.x, h2.y};
    }
  };
  // One step's products; after product j, then(j).
  auto mma = [&](const Frags& f, auto then) {
    each<kMma>([&](auto J) {
      constexpr int m = decltype(J)::value / NT, n = decltype(J)::value % NT;
      acc[m][n] = mma16<T>(f.a[m], f.b[n], acc[m][n]);
      __builtin_amdgcn_sched_barrier(0);
      then(J);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // Part J of kMma of the reads of step kk.
  auto read_part = [&](Frags& f, int buf, int kk, auto J) {
    constexpr int per = (kReads + kMma - 1) / kMma;
    each<per>([&](auto P) {
      constexpr int r = decltype(J)::value * per + decltype(P)::value;
      if constexpr (r < kReads) read_one(f, buf, kk, std::integral_constant<int, r>{});
    });
  };

  load(s0);
  each<kPieces>([&](auto I) { put(s0, 0, I, std::false_type{}); });
  if (s0 + 1 < s1) load(s0 + 1);
  __syncthreads();
  Frags f0, f1;
  each<kReads>([&](auto R) { read_one(f0, 0, 0, R); });
  // Everything but the products goes out between them: a step's fragments after the products of the step
  // before, stage s + 1's pieces (into the buffer whose last reads the barrier of stage s - 1 ended) after
  // those of the second and third step, stage s + 2's loads after the last's. The barrier falls before the
  // last step, whose fragments are in registers by then. FAR: stages s + 1 and s + 2 are whole and there.
  auto stage = [&](int s, auto FAR) {
    constexpr bool far = decltype(FAR)::value;
    const int buf = (s - s0) & 1;
    const bool more = far || s + 1 < s1;
    constexpr int kPer = (kPieces + 2 * kMma - 1) / (2 * kMma);
    auto pieces = [&](auto J, auto FROM) {
      each<kPer>([&](auto P) {
        constexpr int i = (decltype(FROM)::value + decltype(J)::value) * kPer + decltype(P)::value;
        if constexpr (i < kPieces) put(s + 1, buf ^ 1, std::integral_constant<int, i>{}, FAR);
      });
    };
    mma(f0, [&](auto J) { read_part(f1, buf, 1, J); });
    if constexpr (far) {
      mma(f1, [&](auto J) {
        read_part(f0, buf, 2, J);
        pieces(J, std::integral_constant<int, 0>{});
      });
      mma(f0, [&](auto J) {
        read_part(f1, buf, 3, J);
        pieces(J, std::integral_constant<int, kMma>{});
      });
    } else {
      mma(f1, [&](auto J) { read_part(f0, buf, 2, J); });
      if (more) each<kPieces>([&](auto I) { put(s + 1, buf ^ 1, I, std::false_type{}); });
      mma(f0, [&](auto J) { read_part(f1, buf, 3, J); });
      if (s + 2 < s1) load(s + 2);
    }
    __syncthreads();
    mma(f1, [&](auto J) {
      read_part(f0, buf ^ 1, 0, J);  // (past the last stage: what no product takes)
      if constexpr (far) {
        constexpr int j = decltype(J)::value, per = (AP + 1 + kMma - 1) / kMma;
        each<per>([&](auto P) {
          constexpr int i = j * per + decltype(P)::value;
          if constexpr (i < AP) {
            if (has_a) load_piece(s + 2, i);
          } else if constexpr (i == AP) {
            load_block(s + 2);
          }
        });
      }
    });
  };
  int s = s0;
  for (; s + 2 < s1 && (s + 3) * kGradK <= g.n; ++s) stage(s, std::true_type{});
  for (; s < s1; ++s) stage(s, std::false_type{});

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
template <typename T, int V, bool DEEP>
__global__ __launch_bounds__(256) void mx_grad_sum_kernel(const float* __restrict__ parts, int splits,
                                                          int64_t m, int packs, int k,
                                                          T* __restrict__ dx, int64_t ld_dx) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= m * packs) return;
  const int64_t row = i / packs;
  const int c = static_cast<int>(i - row * packs) * V;
  const float* p = parts + row * k + c;
  float v[V];
  sum_parts<DEEP, V>(p, m * k, splits, v);
  store_from_f32<T, V>(dx + row * ld_dx + c, v);
}

// The tile height and the number of splits for a shape, by what a launch is estimated to take: rounds of
// 256 workgroups, each 3 us (5 of 256 tokens) and its stages (1.7, 1.05, 0.9 or 0.65 us of 256, 128, 64
// or 32 tokens); a split contraction pays for the second launch and 8 bytes a sum, which stay in the
// caches (10 TB/s). Measured with n x k = 17,920 x 1,536 fp4, fp16 dy, the kernel and the sums: 4,096
// tokens in 256-token tiles and 5 splits 216 + 21 us (2: 225 + 10, 1: 370; 128-token tiles unsplit 274, in 4
// splits 268 + 18); 2,048 in 256-token tiles and 5 splits 98 + 11 (4: 105 + 9; 128-token tiles in 3 178 +
// 7); 707 in 128-token tiles and 7 splits 47 + 6 (4: 67 + 5; 256-token tiles in 14 43 + 10); 256 in
// 128-token tiles and 20 splits 22 + 6 (256: 25 + 11, 64: 29 + 4). 16 tokens, 2,048 x 1,536, in 32-token
// tiles and 32 splits 4.8 + 3.6 (16: 4.8 + 2.7, 8: 5.8 + 3.8).
struct GradPlan {
  int tm, splits;
};

GradPlan find_grad_plan(int64_t m, int64_t n, int64_t k) {
  const int64_t stages = (n + kGradK - 1) / kGradK, tk = (k + kGradN - 1) / kGradN;
  GradPlan best{256, 1};
  double least = 1e30;
  for (int tm : {256, 128, 64, 32}) {
    const int64_t tiles = (m + tm - 1) / tm * tk;
    const double stage = tm == 256 ? 1.7 : tm == 128 ? 1.05 : tm == 64 ? 0.9 : 0.65;
    for (int64_t s = 1; s <= 64 && s <= stages; ++s) {
      const double rounds = static_cast<double>((tiles * s + 255) / 256);
      const double us = rounds * (static_cast<double>((stages + s - 1) / s) * stage + (tm == 256 ? 5.0 : 3.0)) +
                        (s > 1 ? 4.0 + 8e-7 * static_cast<double>(s) * static_cast<double>(m * k) : 0.0);
      if (us < least) {
        least = us;
        best = {tm, static_cast<int>(s)};
      }
    }
  }
  return best;
}

GradPlan grad_plan(int64_t m, int64_t n, int64_t k) {
  static thread_local PlanMemo<GradPlan> memo;
  return memo.get({m, n, k, 0}, [&] { return find_grad_plan(m, n, k); });
}

int check_sizes(const char* fn, int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n <= 0 || k <= 0 || m >= (1 << 30) || n >= (1 << 28) || k > (1 << 28))
    return fail(RUS_ERR_INVALID, "%s: bad sizes m=%lld n=%lld k=%lld", fn, (long long)m,
                (long long)n, (long long)k);
  return RUS_OK;
}

}  // namespace
}  // namespace rus

using namespace rus;

extern "C" int rus_mx_gemm_t_workspace(int64_t m, int64_t n, int64_t k, int64_t* floats) {
  const char* fn = "rus_mx_gemm_t_workspace";
  if (!floats) return fail(RUS_ERR_INVALID, "%s: null result", fn);
  if (int e = check_sizes(fn, m, n, k)) return e;
  const GradPlan p = grad_plan(m, n, k);
  *floats = p.splits > 1 ? p.splits * m * k : 0;
  return RUS_OK;
}

extern "C" int rus_mx_gemm_t_plan(int64_t m, int64_t n, int64_t k, int32_t* plan) {
  const char* fn = "rus_mx_gemm_t_plan";
  if (!plan) return fail(RUS_ERR_INVALID, "%s: null result", fn);
  if (int e = check_sizes(fn, m, n, k)) return e;
  const GradPlan p = grad_plan(m, n, k);
  plan[0] = p.tm;
  plan[1] = p.splits;
  return RUS_OK;
}

extern "C" int rus_mx_gemm_t(const void* dy, int64_t stride_dy, int32_t dtype, const void* w_codes,
                             const void* w_scales, int32_t w_fmt, int64_t m, int64_t n, int64_t k,
                             void* dx, int64_t stride_dx, float* workspace, int64_t n_workspace,
                             void* stream) {
  const char* fn = "rus_mx_gemm_t";
  if (int e = check_sizes(fn, m, n, k)) return e;
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
  if (int e = check_items(fn, tiles * plan.splits + 7, kGradThreads)) return e;
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
  auto types = [&](auto t) -> int {
    typedef decltype(t) T;
    if (w_fmt == RUS_MX_FP4)
      tile(t, std::integral_constant<int, kFp4>{});
    else
      tile(t, std::integral_constant<int, kFp8>{});
    if (!split) return RUS_OK;
    if (int e = check_launch(fn)) return e;
    const bool wide = k % 4 == 0 && stride_dx % 4 == 0 && aligned(dx, 8);
    const int packs = static_cast<int>(wide ? k / 4 : k);
    const dim3 sum(static_cast<unsigned>((m * packs + 255) / 256));
    auto add = [&](auto k) {
      hipLaunchKernelGGL(k, sum, dim3(256), 0, st, workspace, plan.splits, m, packs, g.k, static_cast<T*>(dx),
                         stride_dx);
    };
    if (deep_sum(m * packs, plan.splits))
      wide ? add(mx_grad_sum_kernel<T, 4, true>) : add(mx_grad_sum_kernel<T, 1, true>);
    else
      wide ? add(mx_grad_sum_kernel<T, 4, false>) : add(mx_grad_sum_kernel<T, 1, false>);
    return RUS_OK;
  };
  if (int e = dtype == RUS_DTYPE_F16 ? types(f16{}) : types(bf16{})) return e;
  return check_launch(fn);
}
