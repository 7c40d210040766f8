// Operand tiles of the attn_masked kernels: 32 tokens x HD head dims of one head, copied straight from global memory
// into LDS (global_load_lds_dwordx4, no register holds a tile in flight) and read from there as 16-byte row fragments
// or, by ds_read_b64_tr_b16, as transposed ones. The layouts of the matrix instruction's operands and accumulator are
// those of attention.hip's comment: an accumulator tile used as an operand carries its reduction index in the order
// k(h, i) = 16 s + 8 (i / 4) + 4 h + i % 4, which the transposed reads produce.
#pragma once

#include "attn_masked.h"

namespace rus {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_void_ptr;
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Eight 16-bit elements, one operand fragment of a lane.
typedef u32x4 Frag;

template <typename T>
__device__ __forceinline__ f32x16 mfma(Frag a, Frag b, f32x16 c) {
  if constexpr (sizeof(T) == 2 && __is_same(T, f16))
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}

// acc + the fragment's eight values, in 32 bits.
template <typename T>
__device__ __forceinline__ float sum8(Frag x, float acc) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = x[i];  // (bit_cast of the vector's element itself takes its first)
    if constexpr (__is_same(T, f16))
      acc = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, u), f16x2{1, 1}, acc, false);
    else
      acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, u), bf16x2{1, 1}, acc, false);
  }
  return acc;
}

// acc + the products of two fragments' values, in 32 bits, in order.
template <typename T>
__device__ __forceinline__ float dot8(Frag x, Frag y, float acc) {
  const Pack<T, 8> a = __builtin_bit_cast(Pack<T, 8>, x), b = __builtin_bit_cast(Pack<T, 8>, y);
#pragma unroll
  for (int i = 0; i < 8; ++i) acc = __builtin_fmaf(static_cast<float>(a.v[i]), static_cast<float>(b.v[i]), acc);
  return acc;
}

// Fragment of k-step s (registers 8 s .. 8 s + 7) of an accumulator tile, each value rounded once.
template <typename T>
__device__ __forceinline__ Frag frag_acc(const f32x16& c, int s) {
  Pack<T, 8> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = from_f32<T>(c[8 * s + i]);
  return __builtin_bit_cast(Frag, r);
}

// The same, with what the roundings left behind in the registers.
template <typename T>
__device__ __forceinline__ Frag split_acc(f32x16& c, int s) {
  const Frag f = frag_acc<T>(c, s);
  const Pack<T, 8> r = __builtin_bit_cast(Pack<T, 8>, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) c[8 * s + i] -= static_cast<float>(r.v[i]);
  return f;
}

// Accumulator row of register r for lane half h.
__device__ __forceinline__ int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// The values of lanes l and l ^ 32 (in some order).
__device__ __forceinline__ float2 half_pair(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return float2{__builtin_bit_cast(float, static_cast<uint32_t>(p[0])),
                __builtin_bit_cast(float, static_cast<uint32_t>(p[1]))};
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float,
                            __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, false));
}

// Sum over groups of 16 (or 8) neighbouring lanes, in every lane, by VALU moves: lanes c ^ 1, c ^ 2, then, each group of 4
// holding its sum, 7 - c within 8 and 15 - c within 16.
template <int N>
__device__ __forceinline__ float group_sum(float x) {
  static_assert(N == 8 || N == 16, "groups of 8 or 16 lanes");
  x += dpp<0xB1>(x);   // quad_perm 1 0 3 2
  x += dpp<0x4E>(x);   // quad_perm 2 3 0 1
  x += dpp<0x141>(x);  // row_half_mirror
  if constexpr (N == 16) x += dpp<0x140>(x);  // row_mirror
  return x;
}

template <int HD>
struct Tiles {
  static constexpr int kRow = 2 * HD;          // bytes of a tile row
  static constexpr int kBytes = 32 * kRow;     // of a tile
  static constexpr int kChunks = kRow / 16;    // 16-byte chunks of a row
  static constexpr int kCopies = kBytes / 1024;  // wave instructions that fill a tile
  static constexpr int kSteps = HD / 16, kDims = HD / 32;

  // The 16-byte chunk c of row r is stored at chunk c ^ swz(r): a quarter wave's fragment reads (16 rows, one chunk) and
  // a half wave's transposing reads (4 rows x 64 bytes) each cover the 64 banks once.
  static __device__ __forceinline__ int swz(int r) {
    if constexpr (HD == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
    const int u = (r >> 1) & 7;  // two rows of 128 bytes span the banks
    return ((u & 1) << 2) | (u >> 1);
  }
};

// A wave's share, C copies from copy c0 (a multiple of C) on, of the kCopies that fill a tile: copy i fills kStep whole
// rows, lane l the position l % kChunks of row kStep i + l / kChunks, i.e. it loads that position's chunk. From copy to
// copy the swizzle changes in a bit or two that do not depend on the lane. The tile's first row is a uniform pointer;
// rows past the last repeat it (finite or not: hidden either way).
template <int HD, int C>
struct TileLane {
  using L = Tiles<HD>;
  static constexpr int kStep = 64 / L::kChunks;
  int c0, row0;       // first copy, the lane's row in it
  uint32_t ch0, off0;  // byte offset of the lane's chunk within that row, of that row
  uint32_t stride;    // bytes per token

  __device__ __forceinline__ TileLane(int first, int lane, int64_t stride_el)
      : c0(first), row0(kStep * first + lane / L::kChunks), stride(static_cast<uint32_t>(stride_el) * 2) {
    ch0 = ((lane % L::kChunks) ^ L::swz(row0)) << 4;
    off0 = row0 * stride;
  }
  __device__ __forceinline__ int row(int i) const { return row0 + kStep * i; }
  // A copy whose offsets the compiler forms again rather than keep each copy's in a register across the loop.
  __device__ __forceinline__ TileLane fresh() const {
    TileLane t = *this;
    asm("" : "+v"(t.ch0), "+v"(t.off0));
    return t;
  }
  __device__ __forceinline__ uint32_t chunk(int i) const {
    return ch0 ^ (HD == 128 ? (i & 3) << 4 : (i & 1) << 5);
  }
  // Byte offset from the tile's first row of what copy i reads; rows: tokens left in the row of the batch.
  __device__ __forceinline__ uint32_t at(int i, int rows) const {
    return (rows >= 32 ? off0 + static_cast<uint32_t>(i * kStep) * stride : min(row(i), rows - 1) * stride) + chunk(i);
  }
  // The builtin's LDS target must be a __shared__ array of its own, so that the compiler knows which LDS reads have to
  // wait for it.
  __device__ __forceinline__ void copy(char* tile, const void* x, int rows) const {
#pragma unroll
    for (int i = 0; i < C; ++i)
      __builtin_amdgcn_global_load_lds(static_cast<const char*>(x) + at(i, rows),
                                       (lds_void_ptr)(tile + (c0 + i) * 1024), 16, 0, 0);
  }
};

// A lane's LDS offsets for the fragments of a tile: one base per kind, changed by step and head-dim tile in a few bits
// only. The empty asm keeps the compiler from holding all combinations in registers across the loop.
template <int HD>
struct FragLane {
  using L = Tiles<HD>;
  uint32_t row, tr;

  __device__ __forceinline__ explicit FragLane(int lane) {
    const int c = lane & 31, h = lane >> 5, j = lane & 15, r0 = 4 * h + (j >> 2);
    row = c * L::kRow + ((h ^ L::swz(c)) << 4);
    tr = r0 * L::kRow + (((((lane >> 4) & 1) * 2 + ((j & 3) >> 1)) ^ L::swz(r0)) << 4) + (j & 1) * 8;
  }
  __device__ __forceinline__ FragLane fresh() const {
    FragLane f = *this;
    asm("" : "+v"(f.row), "+v"(f.tr));
    return f;
  }
  // Head dims 16 s + 8 h .. + 8 of tile row lane % 32.
  __device__ __forceinline__ Frag frag(const char* tile, int s) const {
    return *reinterpret_cast<const Frag*>(tile + (row ^ (s << 5)));
  }
  // x[k(h, i)][32 d + lane % 32], i = 0 .. 7, of k-step s: row r0 + 8 differs from r0 in one bit of the swizzle.
  __device__ __forceinline__ Frag frag_t(const char* tile, int s, int d) const {
    const v4i16 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(tile + (tr ^ (d << 6)) + s * 16 * L::kRow));
    const v4i16 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_v4i16*)(tile + (tr ^ (d << 6) ^ 32) + s * 16 * L::kRow + 8 * L::kRow));
    const u32x2 a = __builtin_bit_cast(u32x2, x0), b = __builtin_bit_cast(u32x2, x1);
    return Frag{a.x, a.y, b.x, b.y};
  }
};

// Every copy of this wave has landed and every LDS read of it has returned.
__device__ __forceinline__ void stage_wait() { __builtin_amdgcn_s_waitcnt(0x0070); }  // vmcnt(0) lgkmcnt(0)

// All but the last N copies of this wave have landed.
template <int N>
__device__ __forceinline__ void wait_copies() {
  __builtin_amdgcn_s_waitcnt(N | (7 << 4) | (15 << 8));
  asm volatile("" ::: "memory");
}

// This wave's LDS reads have returned: a copy may now overwrite the tile they read.
__device__ __forceinline__ void wait_reads() {
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0), vmcnt / expcnt not waited on
  asm volatile("" ::: "memory");
}

// stage_wait and the block's barrier: the buffer just filled may be read, the buffer just read may be filled.
__device__ __forceinline__ void stage_barrier() {
  stage_wait();
  __syncthreads();
}

// Row of one token, head dims 32 d + 8 r4 + 4 h + i from x[d][4 r4 + i] * f: the lane pair (l, l ^ 32) exchanges halves
// so that each stores 16 contiguous bytes.
template <typename T, int ND>
__device__ __forceinline__ void store_row(T* row, const f32x16 (&x)[ND], float f, int h, bool valid) {
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      Pack<T, 4> w0, w1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w0.v[i] = from_f32<T>(x[d][8 * b + i] * f);
        w1.v[i] = from_f32<T>(x[d][8 * b + 4 + i] * f);
      }
      const u32x2 a = __builtin_bit_cast(u32x2, w0), c = __builtin_bit_cast(u32x2, w1);
      const auto p0 = __builtin_amdgcn_permlane32_swap(a.x, c.x, false, false);
      const auto p1 = __builtin_amdgcn_permlane32_swap(a.y, c.y, false, false);
      const u32x4 o = {static_cast<uint32_t>(p0[0]), static_cast<uint32_t>(p1[0]), static_cast<uint32_t>(p0[1]),
                       static_cast<uint32_t>(p1[1])};
      if (valid) *reinterpret_cast<u32x4*>(row + 32 * d + 16 * b + 8 * h) = o;
    }
}

// Whether a sum that only finite operands can leave finite has stayed so: 0 x anything finite.
template <int ND>
__device__ __forceinline__ bool all_finite(const f32x16 (&x)[ND], float f) {
  float z = 0.0f;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) z = fmaxf(z, fabsf(x[d][r] * f) <= 3.402823466e38f ? 0.0f : 1.0f);
  return z == 0.0f;
}

// What the products of NT tiles start from: 0, or, where only a bias by distance is added, the bias in the products' own
// unit (slope / scale), so that it costs no instruction behind the products. d0: distance of the lane's first element;
// tile n's register r is d0 - step * (32 n + acc_row(r, 0)) away. ahead: none of these distances is negative.
template <bool CAP, bool BIAS, int NT>
__device__ __forceinline__ void start_scores(f32x16 (&st)[NT], float slope, float d0, float step, bool ahead) {
  if constexpr (BIAS && !CAP) {
    const float at0 = -slope * d0, per = slope * step;
    if (ahead) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          st[n][r] = __builtin_fmaf(per, static_cast<float>(32 * n + acc_row(r, 0)), at0);
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          st[n][r] = -slope * fabsf(d0 - step * static_cast<float>(32 * n + acc_row(r, 0)));
    }
  } else {
#pragma unroll
    for (int n = 0; n < NT; ++n) st[n] = f32x16{};
  }
}

// With a cap: scores of NT tiles of products, log2 units, and 1 - t^2 in factor. The choice of tanh is made for a whole
// wave (its largest |x|: where that is above 1/4 the fast form's error is 2^-20 of the largest score, as that of its
// product is). slope2, d0, step: the bias, as above.
template <bool BIAS, int NT, bool FACTOR>
__device__ __forceinline__ void capped_scores(const MaskedArgs& a, float slope2, f32x16 (&st)[NT], f32x16 (&factor)[NT],
                                              float d0, float step) {
  float top = 0.0f;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(st[n][r]));
  if (__ballot(!(top * a.kc <= kSmallTanh))) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float u = __builtin_amdgcn_rcpf(1.0f + exp2_raw(st[n][r] * a.k2));
        if constexpr (FACTOR) factor[n][r] = 4.0f * __builtin_fmaf(-u, u, u);
        st[n][r] = __builtin_fmaf(-2.0f * a.cap2, u, a.cap2);
      }
  } else {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float t = tanh_small(st[n][r] * a.kc);
        if constexpr (FACTOR) factor[n][r] = __builtin_fmaf(-t, t, 1.0f);
        st[n][r] = t * a.cap2;
      }
  }
  if constexpr (BIAS) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float d = d0 - step * static_cast<float>(32 * n + acc_row(r, 0));
        st[n][r] = __builtin_fmaf(-slope2, fabsf(d), st[n][r]);
      }
  }
}

}  // namespace
}  // namespace rus
