// Rotary positions with several axes (time, height, width; rows and columns of an image) for gfx950.
//
// Pair i of a head's P rotated pairs turns by a = pos[axis[i]][t] * f[i]:
//   (x1, x2) -> (x1 cos a - x2 sin a, x2 cos a + x1 sin a)
// with x1, x2 the elements i and i + P of the head (halves) or 2 i and 2 i + 1 (adjacent); elements from 2 P on are
// copied. The backward turns by -a. Angles are formed here, not read from a table: with several axes a token's
// combination of positions is its own, and positions may be far or fractions.
//
// The angle in turns, pos * (f / 2 pi), is a product in 64 bits of which the nearest quarter turn is taken off, so
// positions up to 2^31 keep an angle good to 2^-21 turns at f = 1 (32 bits would lose it from 2^20 on); the rest, at
// most an eighth of a turn, goes to 32 bits and through the Taylor polynomials of sine and cosine (degree 9 and 10:
// 2e-9 away at pi / 4).
//
// Bound by HBM: q and k are read and written once, the 16 to 24 bytes of positions aside. A block takes up to 4
// tokens: its threads form the tokens' cosines and sines in the LDS (one pair each at P = 64: every head of the token
// uses them), then move the heads in packs of 16 bytes. 16,381 tokens of 12 + 2 heads of 128 in bf16: 19.4 us, 6.1 TB/s;
// 4,097 of 32 heads of 64 in fp32: 12.0 us, 5.6 TB/s; below some 1,000 tokens the launch is all (8 tokens 2.8 us).
#include "common.h"

namespace rus {
namespace {

typedef __bf16 bf16;

constexpr int kRopeThreads = 256, kMaxPairs = 512, kMaxTokens = 4;

struct RopeSide {  // one of q, k
  const void* x;
  void* y;           // [n_tok][heads][d], contiguous
  int64_t st, sh;    // strides of x: token, head
  int heads;
};

struct RopeAxesArgs {
  RopeSide side[2];
  const void* pos;
  const uint8_t* axis;   // [pairs]
  const double* turns;   // [pairs] f / 2 pi
  int64_t n_tok, ld_pos;
  int pos_type, n_axes, d, pairs, tokens;  // tokens per block
  float dir;             // 1 forward, -1 backward
};

__device__ __forceinline__ double position(const RopeAxesArgs& a, int axis, int64_t t) {
  const int64_t o = axis * a.ld_pos + t;
  if (a.pos_type == RUS_POS_I64) return static_cast<double>(static_cast<const int64_t*>(a.pos)[o]);
  if (a.pos_type == RUS_POS_I32) return static_cast<double>(static_cast<const int32_t*>(a.pos)[o]);
  return static_cast<double>(static_cast<const float*>(a.pos)[o]);
}

// cos and sin of 2 pi x. The quarter turn and the rest by exact differences in 64 bits.
__device__ __forceinline__ void cos_sin_turns(double x, float& c, float& s) {
  const double r = x - __builtin_rint(x);
  const double q = __builtin_rint(4.0 * r);  // -2 .. 2
  const float y = static_cast<float>((r - 0.25 * q) * 6.283185307179586476925);
  const float z = y * y;
  float ps = __builtin_fmaf(z, 2.755731922e-6f, -1.984126984e-4f);
  ps = __builtin_fmaf(z, ps, 8.333333333e-3f);
  ps = __builtin_fmaf(z, ps, -1.666666667e-1f);
  const float sn = __builtin_fmaf(z * y, ps, y);
  float pc = __builtin_fmaf(z, -2.755731922e-7f, 2.480158730e-5f);
  pc = __builtin_fmaf(z, pc, -1.388888889e-3f);
  pc = __builtin_fmaf(z, pc, 4.166666667e-2f);
  pc = __builtin_fmaf(z, pc, -0.5f);
  const float cn = __builtin_fmaf(z, pc, 1.0f);
  const int n = static_cast<int>(q) & 3;
  c = n & 1 ? sn : cn;
  s = n & 1 ? cn : sn;
  if (n == 1 || n == 2) c = -c;
  if (n & 2) s = -s;
}

// E: elements per access (the largest that sizes, strides and addresses allow).
template <typename T, int E, bool ADJ>
__global__ __launch_bounds__(kRopeThreads) void rope_axes_kernel(RopeAxesArgs a) {
  __shared__ __attribute__((aligned(16))) float cs[kMaxTokens * kMaxPairs], sn[kMaxTokens * kMaxPairs];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens;
  const int nt = static_cast<int>(min(static_cast<int64_t>(a.tokens), a.n_tok - t0));
  for (int i = threadIdx.x; i < nt * a.pairs; i += kRopeThreads) {
    const int t = i / a.pairs, p = i - t * a.pairs;
    const int axis = min(static_cast<int>(a.axis[p]), a.n_axes - 1);
    float c, s;
    cos_sin_turns(position(a, axis, t0 + t) * a.turns[p], c, s);
    cs[i] = c;
    sn[i] = s * a.dir;
  }
  __syncthreads();
  constexpr int VP = ADJ ? (E >= 2 ? E / 2 : 1) : E;  // pairs per item
  const int rot = a.pairs / VP, items = rot + (a.d - 2 * a.pairs) / E;
  const int heads = a.side[0].heads + a.side[1].heads, per_token = heads * items;
  for (int i = threadIdx.x; i < nt * per_token; i += kRopeThreads) {
    const int t = i / per_token, r = i - t * per_token;
    int head = r / items;
    const int c = r - head * items;
    const int w = head >= a.side[0].heads;
    const RopeSide& sd = a.side[w];
    head -= w ? a.side[0].heads : 0;
    const T* x = static_cast<const T*>(sd.x) + (t0 + t) * sd.st + head * sd.sh;
    T* y = static_cast<T*>(sd.y) + ((t0 + t) * sd.heads + head) * a.d;
    if (c >= rot) {  // behind the rotated elements
      const int e = 2 * a.pairs + (c - rot) * E;
      store_pack<T, E>(y + e, load_pack<T, E>(x + e));
      continue;
    }
    const float* cp = cs + t * a.pairs + c * VP;
    const float* sp = sn + t * a.pairs + c * VP;
    if constexpr (!ADJ) {
      const int e = c * E;
      float u[E], v[E], o1[E], o2[E];
      load_f32<T, E>(x + e, u);
      load_f32<T, E>(x + a.pairs + e, v);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        o1[j] = __builtin_fmaf(u[j], cp[j], -(v[j] * sp[j]));
        o2[j] = __builtin_fmaf(v[j], cp[j], u[j] * sp[j]);
      }
      store_from_f32<T, E>(y + e, o1);
      store_from_f32<T, E>(y + a.pairs + e, o2);
    } else {
      constexpr int N = 2 * VP;
      const int e = c * N;
      float u[N], o[N];
      if constexpr (E >= 2) {
        load_f32<T, N>(x + e, u);
      } else {
        u[0] = static_cast<float>(x[e]);
        u[1] = static_cast<float>(x[e + 1]);
      }
#pragma unroll
      for (int j = 0; j < VP; ++j) {
        o[2 * j] = __builtin_fmaf(u[2 * j], cp[j], -(u[2 * j + 1] * sp[j]));
        o[2 * j + 1] = __builtin_fmaf(u[2 * j + 1], cp[j], u[2 * j] * sp[j]);
      }
      if constexpr (E >= 2) {
        store_from_f32<T, N>(y + e, o);
      } else {
        y[e] = from_f32<T>(o[0]);
        y[e + 1] = from_f32<T>(o[1]);
      }
    }
  }
}

template <typename T, int E>
void launch(const RopeAxesArgs& a, bool adjacent, unsigned blocks, hipStream_t st) {
  if (adjacent)
    hipLaunchKernelGGL((rope_axes_kernel<T, E, true>), dim3(blocks), dim3(kRopeThreads), 0, st, a);
  else
    hipLaunchKernelGGL((rope_axes_kernel<T, E, false>), dim3(blocks), dim3(kRopeThreads), 0, st, a);
}

template <typename T>
void launch_e(const RopeAxesArgs& a, bool adjacent, int e, unsigned blocks, hipStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (e == 8) return launch<T, 8>(a, adjacent, blocks, st);
  if (e >= 4) return launch<T, 4>(a, adjacent, blocks, st);
  if (e == 2) return launch<T, 2>(a, adjacent, blocks, st);
  launch<T, 1>(a, adjacent, blocks, st);
}

}  // namespace
}  // namespace rus

extern "C" int rus_rope_axes(const void* q, int64_t q_stride_t, int64_t q_stride_h, int32_t h_q, void* q_out,
                             const void* k, int64_t k_stride_t, int64_t k_stride_h, int32_t h_k, void* k_out,
                             int64_t n_tokens, int32_t head_dim, int32_t pairs, int32_t adjacent, const void* pos,
                             int32_t pos_type, int64_t ld_pos, int32_t n_axes, const uint8_t* axis,
                             const double* turns, int32_t inverse, int32_t dtype, void* stream) {
  using namespace rus;
  const char* fn = "rus_rope_axes";
  if (n_tokens < 0 || n_tokens >= (int64_t(1) << 31) || h_q < 0 || h_k < 0 || h_q > 65536 || h_k > 65536 ||
      head_dim <= 0 || head_dim > 65536 || n_axes <= 0 || n_axes > 256 || pairs <= 0 || 2 * pairs > head_dim)
    return fail(RUS_ERR_INVALID, "%s: bad sizes: %lld tokens, %d + %d heads of %d, %d pairs, %d axes", fn,
                (long long)n_tokens, h_q, h_k, head_dim, pairs, n_axes);
  if (static_cast<int64_t>(h_q + h_k) * head_dim >= (1 << 28))
    return fail(RUS_ERR_UNSUPPORTED, "%s: %d + %d heads of %d (under 2^28 elements a token)", fn, h_q, h_k, head_dim);
  if (pairs > kMaxPairs)
    return fail(RUS_ERR_UNSUPPORTED, "%s: %d pairs (at most %d)", fn, pairs, kMaxPairs);
  if (dtype != RUS_DTYPE_F16 && dtype != RUS_DTYPE_BF16 && dtype != RUS_DTYPE_F32)
    return fail(RUS_ERR_INVALID, "%s: unknown dtype %d", fn, dtype);
  if (pos_type != RUS_POS_I64 && pos_type != RUS_POS_I32 && pos_type != RUS_POS_F32)
    return fail(RUS_ERR_INVALID, "%s: unknown position type %d", fn, pos_type);
  if (n_tokens == 0 || h_q + h_k == 0) return RUS_OK;
  const int es = dtype == RUS_DTYPE_F32 ? 4 : 2;
  if ((h_q && (!q || !q_out || !aligned(q, es) || !aligned(q_out, es))) ||
      (h_k && (!k || !k_out || !aligned(k, es) || !aligned(k_out, es))) || !pos ||
      !aligned(pos, pos_type == RUS_POS_I64 ? 8 : 4) || !axis || !turns || !aligned(turns, 8))
    return fail(RUS_ERR_INVALID, "%s: null or misaligned pointer", fn);
  if (ld_pos < 0) return fail(RUS_ERR_INVALID, "%s: negative ld_pos", fn);
  RopeAxesArgs a{};
  a.side[0] = RopeSide{q, q_out, q_stride_t, q_stride_h, h_q};
  a.side[1] = RopeSide{k, k_out, k_stride_t, k_stride_h, h_k};
  a.pos = pos;
  a.axis = axis;
  a.turns = turns;
  a.n_tok = n_tokens;
  a.ld_pos = ld_pos;
  a.pos_type = pos_type;
  a.n_axes = n_axes;
  a.d = head_dim;
  a.pairs = pairs;
  a.dir = inverse ? -1.0f : 1.0f;
  // The widest access at which every head's row and both halves of it start.
  int e = 16 / es;
  auto fits = [&](int n) {
    if (head_dim % n || (adjacent ? 2 * pairs : pairs) % n) return false;
    for (const RopeSide& s : a.side)
      if (s.heads && (s.st % n || s.sh % n || !aligned(s.x, n * es) || !aligned(s.y, n * es))) return false;
    return true;
  };
  while (e > 1 && !fits(e)) e /= 2;
  // Four tokens share a block's launch and angles once the blocks outnumber what the chip holds; before that one each
  // ends sooner. 12 + 2 heads of 128, bf16, us with one / four: 8 tokens 2.8 / 3.4, 707 3.3 / 3.8, 2,048 4.6 / 4.7, 3,000
  // 6.2 / 5.4, 16,381 22.7 / 19.4; 32 heads of 64, fp32: 2,048 6.1 / 6.4, 4,097 12.7 / 12.0.
  a.tokens = n_tokens >= 2560 ? kMaxTokens : 1;
  const unsigned blocks = static_cast<unsigned>((n_tokens + a.tokens - 1) / a.tokens);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == RUS_DTYPE_F16)
    launch_e<f16>(a, adjacent, e, blocks, st);
  else if (dtype == RUS_DTYPE_BF16)
    launch_e<bf16>(a, adjacent, e, blocks, st);
  else
    launch_e<float>(a, adjacent, e, blocks, st);
  return check_launch(fn);
}
