// What the lm_head kernels share beside the GEMM mainloop: a tile of logits (or of what replaces them) stored
// token-major, and the references that P is kept against over the chunks of the vocabulary.
#pragma once

#include <math.h>

#include "mfma_gemm.h"

namespace rus {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Writes the block's 256 (vocab) x 256 (token) tile, held in the accumulator layout, as fp16
// out[token][vocab - tile base]: value(mt, nt, r, row) is the element of accumulator (mt, nt, r),
// whose vocab row local to A is row; rows >= g.M are written as 0. Staged through the LDS as
// [token][vocab] with 8-byte quads XOR-swizzled by row (pairs kept adjacent) so every lane stores
// 16 contiguous bytes of one token's row: out[tok][tl.m0 + c] for tok < g.N, c < kpad.
// NW waves in the mainloop's layout (4: 128 x 128 each, 8: 128 x 64).
template <int NW = 4, class F>
__device__ __forceinline__ void store_tile_tv(char* smem, const GemmArgs& g, const Tile& tl,
                                              f16* out, int64_t ld, int kpad, F value) {
  constexpr int NT = 16 / NW, RW = kBN / (NW / 2);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = NW == 8 ? wave8_m(wave) : wave >> 1;
  const int wn = NW == 8 ? wave8_n(g, tl, wave) : wave & 1;
  const int h = lane >> 5;
  const int vrow0 = tl.m0 + wm * kWM;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int trow = wn * RW + nt * 32 + (lane & 31);  // token row within the block tile
    char* srow = smem + trow * 512;
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f16x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = vrow0 + mt * 32 + 8 * q + 4 * h + e;
          v[e] = from_f32<f16>(row < g.M ? value(mt, nt, q * 4 + e, row) : 0.0f);
        }
        const int col = wm * kWM + mt * 32 + 8 * q + 4 * h;  // vocab column within the tile
        const int pq = (col >> 2) ^ ((trow & 31) << 1);
        *reinterpret_cast<f16x4*>(srow + pq * 8) = v;
      }
  }
  __syncthreads();
  const int t = threadIdx.x;
  const int c = t & 31;
#pragma unroll 4
  for (int it = 0; it < kBN / (2 * NW); ++it) {
    const int trow = it * 2 * NW + (t >> 5);
    const int tok = tl.n0 + trow;
    const int col = tl.m0 + c * 8;
    if (tok < g.N && col < kpad) {
      const int pq = (2 * c) ^ ((trow & 31) << 1);
      const uint4 v = *reinterpret_cast<const uint4*>(smem + trow * 512 + pq * 8);
      *reinterpret_cast<uint4*>(out + static_cast<int64_t>(tok) * ld + col) = v;
    }
  }
}

// A token's reference stays the one it came with unless a half tile's largest logit lies more than
// kRefWindow (log2 units) above it; P is at most 2^15 in fp16. A half tile past the window (every
// one of the first chunk) takes its own, a multiple of kRefStep not above its maximum, so that the
// half tiles of a token mostly agree (P < 2^kRefStep) and none needs rescaling. Either way the
// largest P of all is at least 1: fp16 resolves every smaller probability as well as it would
// against the maximum. The largest itself would be exact there and is not here, so its relative
// rounding (part_r) goes to the finishing kernel, which takes it back where that probability counts.
constexpr float kRefWindow = 15.0f, kRefStep = 8.0f;

__device__ __forceinline__ float own_ref(float y) {
  return kRefStep * floorf(y / kRefStep);
}

// fp32 -> uint32 in the same order (NaN aside); 0 is below every value.
__device__ __forceinline__ uint32_t ordered_bits(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t u) {
  return __builtin_bit_cast(float, u ^ ((u >> 31) ? 0x80000000u : 0xffffffffu));
}

}  // namespace
}  // namespace rus
