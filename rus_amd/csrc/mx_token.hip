// Products of microscaled weights with a few tokens (up to four): y = x W^T (+ bias) and the gated
// feed-forward's silu(x Wg^T) (x Wu^T), x in blocks or rounded to blocks here.
//
// A token has one use for each weight, so this is a pass over W, bound by how fast its lines arrive and,
// at one pass of a few us, by their latency. Eight lanes read 128 bytes (fp4) of one row, a lane one
// block of 32; a wave so takes eight rows, whole lines each, and the workgroup's waves are dealt the
// contraction's chunks of eight blocks. All loads of a wave (up to kAhead chunks) go out before anything
// is waited for. Meanwhile the workgroup rounds x to blocks, once, and keeps its elements in LDS as fp16
// (which holds both element types exactly); that costs a few elements a thread and spares the launch that
// would do it. A block's 32 products are summed by v_dot2_f32_f16, exact products and fp32 sums, and join
// the row's sum times both blocks' scales, as one exponent: the product of the scales alone may pass fp32.
//
// One token: 1,536 x 8,960 fp4 (7.3 MB) 6.4 us with W from memory and 5.4 from the last-level cache, 2 x
// 8,960 x 1,536 with the gate (14.6 MB) 7.4 and 6.2; an empty launch takes about 2.
//
// Matrix instructions would not help: their operand wants 32 rows at once, 32 bytes of each, four times
// the line requests; tokens 1 to 32 cost them the same.
#include "mx.h"
#include "swiglu_math.h"

namespace rus {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef u32x4s u32x4u __attribute__((aligned(2)));

// Bytes of a block of x in LDS: 64 and a gap, so that eight blocks' reads miss each other's banks.
constexpr int kPitch = 80;

// A block's 32 elements, two at a time, as fp16.
template <int FMT>
__device__ __forceinline__ void halves(const u32x4s (&c)[kCodeBytes<FMT> / 16], f16x2 (&h)[16]) {
  each<16>([&](auto I) {
    constexpr int i = decltype(I)::value;
    if constexpr (FMT == kFp4)
      h[i] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c[0][i / 4], 1.0f, i % 4));
    else
      h[i] = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[i / 8][i / 2 % 4], 1.0f, i % 2));
  });
}

// x to LDS: the elements of block b of token t at (t nb + b) kPitch, the scale bytes after all blocks.
template <typename T>
__device__ __forceinline__ void stage_x(const TokenArgs& g, char* lds, uint32_t* bytes) {
  const int packs = g.nb * 4, total = g.m * packs;
  for (int p = threadIdx.x; p < total; p += blockDim.x) {
    const int t = p / packs, q = p - t * packs, block = p >> 2;
    float v[8];
    uint32_t b;
    if (g.x) {
      const T* row = static_cast<const T*>(g.x) + t * g.ldx;
      if (q * 8 + 8 <= g.k) {
        const Pack<T, 8> e = __builtin_bit_cast(Pack<T, 8>, u32x4s(*reinterpret_cast<const u32x4u*>(row + q * 8)));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(e.v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = q * 8 + i < g.k ? static_cast<float>(row[q * 8 + i]) : 0.0f;
      }
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, abs_bits(v[i]));
      top = quad_max(top);
      b = g.x_fmt == kFp8 ? scale_byte<kFp8>(top) : scale_byte<kFp4>(top);
      const float inv = inv_scale(b);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= inv;
      if (g.x_fmt == kFp8) {
        uint32_t w[2];
        to_fp8<8>(v, b == 255, w);
        from_fp8(w[0], w[1], 1.0f, v);
      } else {
        uint32_t w[1];
        to_fp4<8>(v, b == 255, w);
        from_fp4(w[0], 1.0f, v);
      }
    } else {
      b = g.xs[block];
      if (g.x_fmt == kFp8) {
        const u32x2s w = reinterpret_cast<const u32x2s*>(g.xc)[p];
        from_fp8(w.x, w.y, 1.0f, v);
      } else {
        from_fp4(reinterpret_cast<const uint32_t*>(g.xc)[p], 1.0f, v);
      }
    }
    store_from_f32<f16, 8>(reinterpret_cast<f16*>(lds + block * kPitch + (p & 3) * 16), v);
    if ((p & 3) == 0) bytes[block] = b;
  }
}

template <int FW, int EPI, typename T, int M>
__global__ __launch_bounds__(512) void mx_token_kernel(TokenArgs g) {
  constexpr int P = EPI == kTokenGlu ? 2 : 1, C = kCodeBytes<FW> / 16, kAhead = P == 1 ? 6 : 3;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ float red[8][P][8][M];
  uint32_t* const bytes = reinterpret_cast<uint32_t*>(lds + g.m * g.nb * kPitch);
  const int lane = threadIdx.x & 63, r = lane >> 3, c = lane & 7;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int f0 = blockIdx.x * 8;
  const int64_t row = min(f0 + r, g.n - 1);  // rows past the last re-read it; what they give is not stored
  const int chunks = (g.nb + 7) >> 3;
  float acc[P][M] = {};
  bool staged = false;
  int j0 = wave;
  do {  // at least once: every wave meets the others below
    u32x4s code[kAhead][P][C];
    uint32_t scale[kAhead][P];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int block = min((j0 + i * waves) * 8 + c, g.nb - 1);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int64_t at = (row + static_cast<int64_t>(p) * g.n) * g.nb + block;
        const u32x4s* src = reinterpret_cast<const u32x4s*>(g.wc + at * kCodeBytes<FW>);
#pragma unroll
        for (int j = 0; j < C; ++j) code[i][p][j] = src[j];
        scale[i][p] = g.ws[at];
      }
    }
    if (!staged) {
      stage_x<T>(g, lds, bytes);
      __syncthreads();
      staged = true;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int block = (j0 + i * waves) * 8 + c;
      if ((j0 + i * waves) * 8 >= g.nb) break;
      const int at = min(block, g.nb - 1);
      f16x2 hw[P][16];
#pragma unroll
      for (int p = 0; p < P; ++p) halves<FW>(code[i][p], hw[p]);
#pragma unroll
      for (int t = 0; t < M; ++t) {
        const int xb = min(t, g.m - 1) * g.nb + at;
        u32x4s v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const u32x4s*>(lds + xb * kPitch + 16 * j);
        const uint32_t b = bytes[xb];
#pragma unroll
        for (int p = 0; p < P; ++p) {
          float d[2] = {};
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const uint32_t pair = v[j / 4][j % 4];
            d[j & 1] = __builtin_amdgcn_fdot2(hw[p][j], __builtin_bit_cast(f16x2, pair), d[j & 1], false);
          }
          float s = __builtin_ldexpf(d[0] + d[1], static_cast<int>(b + scale[i][p]) - 254);
          if (max(b, scale[i][p]) == 255) s = __builtin_nanf("");
          acc[p][t] += block < g.nb ? s : 0.0f;
        }
      }
    }
    j0 += kAhead * waves;
  } while (j0 < chunks);
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int t = 0; t < M; ++t) {
      float s = acc[p][t];
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) s += __shfl_xor(s, off, kWave);
      if (c == 0) red[wave][p][r][t] = s;
    }
  __syncthreads();
  const int t = threadIdx.x >> 3, f = f0 + (threadIdx.x & 7);
  if (t >= g.m || f >= g.n) return;
  float s[P] = {};
  for (int w = 0; w < waves; ++w)
#pragma unroll
    for (int p = 0; p < P; ++p) s[p] += red[w][p][threadIdx.x & 7][t];
  if constexpr (EPI == kTokenGlu) {
    s[0] = s[0] * glu_sigmoid(s[0]) * s[1];
  } else {
    if (g.bias) s[0] += static_cast<float>(static_cast<const T*>(g.bias)[f]);
  }
  static_cast<T*>(g.y)[t * g.ldy + f] = from_f32<T>(s[0]);
}

// Eight waves where the contraction is long or workgroups are few, four else (each workgroup rounds x for
// itself). One token, W from memory: 1,536 x 8,960 fp4 11.6, 8.3 and 6.3 us with 2, 4 and 8 waves, 2 x
// 8,960 x 1,536 with the gate 8.3, 7.0 and 9.8, 17,920 x 1,536 8.3, 8.3 and 12.9; four tokens x 2,048 x
// 1,536 8.0, 6.2 and 5.2.
int token_waves(int64_t n, int64_t nb) { return (nb + 7) / 8 > 16 || n <= 4096 ? 8 : 4; }

template <int FW, int EPI, typename T>
void launch(const TokenArgs& g, hipStream_t st) {
  const int waves = token_waves(g.n, g.nb);
  const size_t lds = static_cast<size_t>(g.m) * g.nb * (kPitch + 4);
  auto go = [&](auto k) {
    hipLaunchKernelGGL(k, dim3((g.n + 7) / 8), dim3(waves * kWave), lds, st, g);
  };
  if (g.m == 1)
    go(mx_token_kernel<FW, EPI, T, 1>);
  else if (g.m == 2)
    go(mx_token_kernel<FW, EPI, T, 2>);
  else
    go(mx_token_kernel<FW, EPI, T, 4>);
}

template <int EPI, typename T>
void by_weight(const TokenArgs& g, int w_fmt, hipStream_t st) {
  if (w_fmt == RUS_MX_FP4)
    launch<kFp4, EPI, T>(g, st);
  else
    launch<kFp8, EPI, T>(g, st);
}

}  // namespace

// One or two tokens, four where there are few features, as far as x fits into LDS. W from memory, this
// kernel against rounding x in a launch of its own and the other kernels, weights in 4 bits (in 8): 1,536 x
// 8,960 one token 6.4 and 13.8 us (7.4 and 13.9), two 8.3 and 13.3 (9.1 and 14.2); 2,048 x 1,536 one 4.1
// and 6.5 (4.5 and 7.1), four 5.2 and 6.9 (5.6 and 7.4); 17,920 x 1,536 one 8.6 and 10.0 (11.3 and 11.9),
// two 10.9 and 10.3 (13.7 and 12.5; one launch less for the host), four 15.4 and 11.9 (18.1 and 15.5); with
// the gate, 2 x 8,960 x 1,536, one 7.4 and 12.1 (9.5 and 15.3), two 10.2 and 12.4 (11.2 and 15.7), four
// 13.6 and 12.3 (15.3 and 15.9).
bool few_tokens(int64_t m, int64_t n, int64_t nb) {
  return m <= (n <= 4096 ? 4 : 2) && m * nb * (kPitch + 4) <= 61440 &&
         (n + 7) / 8 * token_waves(n, nb) * kWave < kMaxItems;  // (else the 32 x 32 kernel)
}

int token_product(const char* fn, const TokenArgs& g, int w_fmt, bool glu, bool bf, hipStream_t st) {
  if (glu) {
    if (bf)
      by_weight<kTokenGlu, bf16>(g, w_fmt, st);
    else
      by_weight<kTokenGlu, f16>(g, w_fmt, st);
  } else {
    if (bf)
      by_weight<kTokenPlain, bf16>(g, w_fmt, st);
    else
      by_weight<kTokenPlain, f16>(g, w_fmt, st);
  }
  return check_launch(fn);
}

}  // namespace rus
