// Products of microscaled rows: y = x W^T (+ bias), and the gated feed-forward's first half
// silu(x Wg^T) (x Wu^T) with its backward, on v_mfma_scale_f32_32x32x64_f8f6f4.
//
// The instruction takes 64 of the contraction at a time: two blocks of 32, whose scales it applies
// itself. A lane (row l % 32, half g = l / 32) of an fp4 operand holds block g's 32 codes; of an fp8
// operand bytes 16 g .. +16 of block 0 and of block 1; its scale byte is block g's. W is the first
// operand (the rows of the result), x the second (its columns): register r of lane l holds row
// 8 (r / 4) + 4 (l / 32) + r % 4 and token l % 32. Row i of a tile is feature 16 ((i / 4) % 2) +
// 4 (i / 8) + i % 4, so that a lane's 16 registers are 16 neighbouring features.
// The instruction's sums are fp32; within the 16 products of an fp8 operand that it adds first it
// keeps about 13 bits below the largest (fp4 by fp4 loses nothing), so results are 16-bit types.
#include "mx.h"
#include "swiglu_math.h"

namespace rus {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

enum { kPlain = 0, kGluFwd = 1, kGluBwd = 2, kParts = 3 };  // kParts: fp32 sums of a part of the contraction
constexpr int outs_of(int epi) { return epi == kGluFwd || epi == kGluBwd ? 2 : 1; }  // rows of W per feature

typedef u32x4s u32x4u __attribute__((aligned(2)));  // a 16-byte access at any alignment of elements

struct MxArgs {
  const uint8_t *xc, *xs;  // x: codes and scales, [m] rows
  const uint8_t *wc, *ws;  // W: [n] rows, or [2 n] (gate rows, then up rows)
  int m, n, nb;            // tokens, output features, blocks of the contraction (multiple of 4)
  int splits;              // kParts: parts the contraction's groups of four blocks are dealt to
  const void* bias;        // kPlain: [n] or null
  const void* dh;          // kGluBwd: [m, n]
  int64_t ld_dh;
  void* y;                 // [m, n], [m, 2 n] for kGluBwd, fp32 [splits, m, n] for kParts
  int64_t ldy;
  bool vec;                // rows of y (and dh, bias) allow aligned packs
};

template <int FMT>
constexpr int kMfmaFmt = FMT == kFp4 ? 4 : 0;

__device__ __forceinline__ int feature_of(int i) {
  return 16 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3);
}

// One operand row of one group of four blocks: the two MFMA steps' fragments and their scales.
template <int FMT>
struct Frag {
  u32x4s v[FMT == kFp4 ? 2 : 4];
  uint32_t s;
  __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* scales, int g) {
    if constexpr (FMT == kFp4) {
      const u32x4s* p = reinterpret_cast<const u32x4s*>(codes + g * 32);
      v[0] = p[0];
      v[1] = p[1];
    } else {
      const u32x4s* p = reinterpret_cast<const u32x4s*>(codes + g * 16);
      v[0] = p[0];
      v[1] = p[4];
      v[2] = p[2];
      v[3] = p[6];
    }
    s = *reinterpret_cast<const uint32_t*>(scales) >> (16 * g);
  }
  template <int S>
  __device__ __forceinline__ i32x8 get() const {
    if constexpr (FMT == kFp4)
      return i32x8{(int)v[S].x, (int)v[S].y, (int)v[S].z, (int)v[S].w, 0, 0, 0, 0};
    else
      return i32x8{(int)v[2 * S].x,     (int)v[2 * S].y,     (int)v[2 * S].z,     (int)v[2 * S].w,
                   (int)v[2 * S + 1].x, (int)v[2 * S + 1].y, (int)v[2 * S + 1].z, (int)v[2 * S + 1].w};
  }
};

template <int FW, int FX>
__device__ __forceinline__ void mma(const Frag<FW>& w, const Frag<FX>& x, f32x16& acc) {
  acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w.template get<0>(), x.template get<0>(), acc,
                                                        kMfmaFmt<FW>, kMfmaFmt<FX>, 0, (int)w.s, 0,
                                                        (int)x.s);
  acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w.template get<1>(), x.template get<1>(), acc,
                                                        kMfmaFmt<FW>, kMfmaFmt<FX>, 1, (int)w.s, 1,
                                                        (int)x.s);
}

// N neighbouring values from / to a row, from feature f on of `n`.
template <typename T, int N>
__device__ __forceinline__ void load_n(const T* row, int f, int n, bool vec, float (&v)[N]) {
  if (vec && f + N <= n) {
    load_f32<T, N>(row + f, v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = f + i < n ? static_cast<float>(row[f + i]) : 0.0f;
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T* row, int f, int n, bool vec, const float (&v)[N]) {
  if (vec && f + N <= n) {
    store_from_f32<T, N>(row + f, v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (f + i < n) row[f + i] = from_f32<T>(v[i]);
  }
}

// Part `split`'s groups of four blocks.
struct Range {
  int first, count;
};
__device__ __forceinline__ Range groups_of(const MxArgs& g, int split) {
  const int groups = g.nb / 4;
  const int a = static_cast<int>(static_cast<int64_t>(groups) * split / g.splits);
  return {a, static_cast<int>(static_cast<int64_t>(groups) * (split + 1) / g.splits) - a};
}

// What becomes of N neighbouring features f.. of token t: a = x W^T (or the gate's), u the up's.
template <int EPI, typename T, int N>
__device__ __forceinline__ void finish(const MxArgs& g, int t, int f, const float (&a)[N],
                                       const float (&u)[N]) {
  if constexpr (EPI == kParts) {
    float* p = static_cast<float*>(g.y) + (static_cast<int64_t>(blockIdx.z) * g.m + t) * g.n;
    store_n<float, N>(p, f, g.n, g.vec, a);
    return;
  }
  T* y = static_cast<T*>(g.y) + t * g.ldy;
  float o[N];
  if constexpr (EPI == kPlain) {
    float b[N] = {};
    if (g.bias) load_n<T, N>(static_cast<const T*>(g.bias), f, g.n, g.vec, b);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = a[i] + b[i];
    store_n<T, N>(y, f, g.n, g.vec, o);
  } else if constexpr (EPI == kGluFwd) {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = a[i] * glu_sigmoid(a[i]) * u[i];
    store_n<T, N>(y, f, g.n, g.vec, o);
  } else {
    float d[N], du[N];
    load_n<T, N>(static_cast<const T*>(g.dh) + t * g.ld_dh, f, g.n, g.vec, d);
#pragma unroll
    for (int i = 0; i < N; ++i) glu_bwd(d[i], a[i], u[i], o[i], du[i]);
    store_n<T, N>(y, f, g.n, g.vec, o);
    store_n<T, N>(y + g.n, f, g.n, g.vec, du);
  }
}

// ---- tens of tokens --------------------------------------------------------------------------------
//
// 32 features x 32 tokens per workgroup of four waves, the contraction's groups of four blocks dealt to
// the waves, operands straight from memory to registers, two groups' loads in flight at a time; the
// waves' sums meet in LDS. Bound by the lines that a CU's address unit takes in (about 2.3 cycles each: a
// load touches 32 rows for 32 bytes of each), so eight waves bring nothing where workgroups are many (32
// tokens fp8 by fp4: 17,920 x 1,536 10.0 us with four and 10.2 with eight, 2,048 x 1,536 5.1 and 5.3). Few
// of them over a long contraction (1,536 x 8,960, 32 tokens: 16.5 and 15.5) leave CUs idle, which parts of
// the contraction fill (five parts: 6.2 and 6.1).
constexpr int kAhead = 2, kRowsWaves = 4;

template <int FX, int FW, int EPI, typename T>
__global__ __launch_bounds__(kRowsWaves* kWave) void mx_rows_kernel(MxArgs g) {
  constexpr int WAVES = kRowsWaves;
  constexpr int NA = outs_of(EPI);
  __shared__ float red[WAVES][NA][16][kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int f0 = blockIdx.x * 32, t0 = blockIdx.y * 32;
  // rows past the edge re-read the last one; what they give is not stored
  const int64_t tok = min(t0 + (lane & 31), g.m - 1);
  const int64_t feat = min(f0 + feature_of(lane & 31), g.n - 1);
  const uint8_t* xc = g.xc + tok * g.nb * kCodeBytes<FX>;
  const uint8_t* xs = g.xs + tok * g.nb;
  const uint8_t *wc[NA], *ws[NA];
#pragma unroll
  for (int a = 0; a < NA; ++a) {
    wc[a] = g.wc + (feat + static_cast<int64_t>(a) * g.n) * g.nb * kCodeBytes<FW>;
    ws[a] = g.ws + (feat + static_cast<int64_t>(a) * g.n) * g.nb;
  }
  f32x16 acc[NA] = {};
  const Range mine = EPI == kParts ? groups_of(g, blockIdx.z) : Range{0, g.nb / 4};
  const int end = mine.first + mine.count;
  for (int b = mine.first + wave; b < end; b += kAhead * WAVES) {
    Frag<FX> x[kAhead];
    Frag<FW> w[kAhead][NA];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = 4 * min(b + u * WAVES, end - 1);
#pragma unroll
      for (int a = 0; a < NA; ++a) w[u][a].load(wc[a] + at * kCodeBytes<FW>, ws[a] + at, half);
      x[u].load(xc + at * kCodeBytes<FX>, xs + at, half);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (b + u * WAVES >= end) break;
#pragma unroll
      for (int a = 0; a < NA; ++a) mma(w[u][a], x[u], acc[a]);
    }
  }
#pragma unroll
  for (int a = 0; a < NA; ++a)
#pragma unroll
    for (int r = 0; r < 16; ++r) red[wave][a][r][lane] = acc[a][r];
  __syncthreads();
  const int t = t0 + (lane & 31), f = f0 + 16 * half + 4 * wave;
  if (t >= g.m || f >= g.n) return;
  float v[2][4] = {};
#pragma unroll
  for (int a = 0; a < NA; ++a)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 0; w < WAVES; ++w) v[a][i] += red[w][a][4 * wave + i][lane];
  finish<EPI, T, 4>(g, t, f, v[0], v[1]);
}

// ---- tiles -----------------------------------------------------------------------------------------
//
// BF rows of W x BT tokens per workgroup of four waves (2 x 2 of BF/2 x BT/2; eight, 2 x 4, for 256
// tokens), the contraction staged GROUPS x 128 at a time (a group of four blocks is two MFMA steps)
// through two LDS buffers that memory is copied into directly (global_load_lds: 64 lanes' 16 bytes land
// one after the other), a stage ahead of its products. Two workgroups of four waves share a CU: one's
// waits and epilogue run under the other's products. One of eight has it to itself.
//
// What bounds it is the copies: a CU takes a line from its L2 in about 2.3 cycles whether it needs 128
// bytes of it or 64 (55 or 28 bytes per cycle, measured with nothing else running). Where both operands
// are fp4, a stage is therefore two groups, so that rows are whole lines, and where there are tiles
// enough a tile is 256 x 256, which copies half as much a product (8,161 x 17,920 x 1,536: 164 us, 2.7
// PFLOP/s, against 180 with 128 x 128; 8,161 x 8,960 x 8,960: 353, 3.7 PFLOP/s, and 426); with an fp8
// operand the products take twice as long and a taller tile of one group covers the copies (8,161 x 17,920
// x 1,536 with fp4 weights: 208 us, 2.2 PFLOP/s, with 256 x 128, 254 with 128 x 128; fp8 weights, 128 x
// 128 only: 275). (Averages of 20 calls on the same operands; on three sets of them in turn 169, 407, 234
// and 327.) They go out between the products, since a wave that issues them in a row waits for each.
//
// LDS rows of W are in MFMA order (row 32 q + i holds feature 32 q + feature_of(i)); with a gate, the
// lower half is gate, the upper half up rows of the same features, and a wave takes the same part of
// both, so that a lane holds both. The 16-byte chunk c of row r lies at c ^ ((r / 4) % 4) of a 64-byte
// row, c ^ ((r / 2) % 8) of a 128-byte one, by each lane fetching the chunk that belongs at its place: 16
// neighbouring rows read at one chunk cover all banks once. Scales come four groups at a time, 16 bytes
// of a row in one request. LDS is read by explicit instructions and waits: the compiler would wait for
// the copies in flight before any LDS read. A register read this way is tied to the wait before its first
// use.

// Four waves, 2 x 2; eight, 2 x 4, for 256 tokens.
template <int BT>
constexpr int kTileThreads = BT == 256 ? 512 : 256;
typedef u32x4s u32x4w __attribute__((aligned(4)));  // a 16-byte access at any word
typedef __attribute__((address_space(3))) void* lds_void;

template <int FMT, int GROUPS>
constexpr int kStageRow = (FMT == kFp4 ? 64 : 128) * GROUPS;

template <int ROWB>
__device__ __forceinline__ int swizzle(int r) {
  static_assert(ROWB == 64 || ROWB == 128, "rows of one line or half of one");
  return ROWB == 64 ? (r >> 2) & 3 : (r >> 1) & 7;
}

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void)p));
}
template <int OFF>
__device__ __forceinline__ u32x4s lds_read16(uint32_t addr) {
  u32x4s v;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFF));
  return v;
}
template <int OFF>
__device__ __forceinline__ uint32_t lds_read2(uint32_t addr) {
  uint32_t v;
  asm volatile("ds_read_u16 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFF));
  return v;
}
template <int N>
__device__ __forceinline__ void wait_lds() {
  static_assert(N <= 15, "lgkmcnt counts to 15");
  asm volatile("s_waitcnt lgkmcnt(%0)" ::"i"(N));
}
__device__ __forceinline__ void tie(u32x4s& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void tie(uint32_t& v) { asm volatile("" : "+v"(v)); }

// The codes of ROWS rows of one operand on their way into LDS. Copy i of wave w fills bytes
// 1024 (waves i + w) .. +1024 of the operand's stage.
template <int FMT, int ROWS, int GROUPS, int PARTS, int THREADS>
struct Copier {
  static constexpr int kRow = kStageRow<FMT, GROUPS>, kPer = kRow / 16;  // bytes and chunks per row
  static constexpr int kCopies = ROWS * kPer / THREADS;             // copies per wave
  static constexpr int kBytes = ROWS * kRow;
  static_assert(kCopies % PARTS == 0, "whole copies per part");
  // LDS row r holds the operand's row part(r * PARTS / ROWS) + in(r), in below 256: the gate's rows, then
  // the up's, or one part.
  const uint8_t* base[PARTS];
  uint32_t off[kCopies];
  template <typename P, typename R>
  __device__ __forceinline__ void init(const uint8_t* codes, int nb, P part, R in) {
    const int bytes = nb * kCodeBytes<FMT>;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) base[i] = codes + part(i) * bytes;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int q = i * THREADS + threadIdx.x, r = q / kPer;
      off[i] = static_cast<uint32_t>(in(r) * bytes + ((q % kPer) ^ swizzle<kRow>(r)) * 16);
    }
  }
  // Of stage s. `last`: it has one group only; lanes of the second fetch the first again.
  template <int I>
  __device__ __forceinline__ void copy(int s, bool last, char* stage, int wave) const {
    uint32_t o = off[I];
    if constexpr (GROUPS == 2) {
      const int q = I * THREADS + threadIdx.x;
      if (last && ((q % kPer) ^ swizzle<kRow>(q / kPer)) >= kPer / 2) o -= kRow / 2;
    }
    const uint8_t* p = base[I * PARTS / kCopies] + static_cast<int64_t>(s) * kRow;
    __builtin_amdgcn_global_load_lds(p + o, (lds_void)(stage + (THREADS / kWave * I + wave) * 1024), 16, 0, 0);
  }
};

// The scales of four groups (a quad) of one row per thread.
struct ScaleRow {
  const uint8_t* src;
  u32x4s v;
  // Of the four groups from `first` on, none past the row's end (rows of at least four).
  __device__ __forceinline__ void load(int first) { v = *reinterpret_cast<const u32x4w*>(src + 4 * first); }
  __device__ __forceinline__ void load_short(int groups) {  // a row of fewer
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint32_t*>(src + 4 * min(j, groups - 1));
  }
};

// NT tiles' fragments of one MFMA step from LDS.
template <int FMT, int NT, int GROUPS, int UP>
struct StepFrags {
  static constexpr int kReads = (FMT == kFp4 ? 1 : 2) * NT;
  static constexpr int kRow = kStageRow<FMT, GROUPS>;
  u32x4s v[kReads];
  // Tile t's first row, from this lane's row of the first: 32 apart, the second half from UP on.
  static constexpr int row_of(int t) { return UP && t >= NT / 2 ? UP + (t - NT / 2) * 32 : t * 32; }
  // Read R of step S. row0: address of this lane's row of the first tile, sw: its swizzle.
  template <int S, int R>
  __device__ __forceinline__ void read(uint32_t row0, int sw, int half) {
    if constexpr (FMT == kFp4) {
      constexpr int c = 4 * (S >> 1) + (S & 1);
      v[R] = lds_read16<row_of(R) * kRow>(row0 + (((c + 2 * half) ^ sw) << 4));
    } else {
      static_assert(GROUPS == 1, "fp8 rows of one group");
      v[R] = lds_read16<row_of(R >> 1) * kRow>(row0 + (((4 * (R & 1) + 2 * S + half) ^ sw) << 4));
    }
  }
  __device__ __forceinline__ void tied() {
#pragma unroll
    for (int i = 0; i < kReads; ++i) tie(v[i]);
  }
  __device__ __forceinline__ i32x8 get(int t) const {
    if constexpr (FMT == kFp4)
      return i32x8{(int)v[t].x, (int)v[t].y, (int)v[t].z, (int)v[t].w, 0, 0, 0, 0};
    else
      return i32x8{(int)v[2 * t].x,     (int)v[2 * t].y,     (int)v[2 * t].z,     (int)v[2 * t].w,
                   (int)v[2 * t + 1].x, (int)v[2 * t + 1].y, (int)v[2 * t + 1].z, (int)v[2 * t + 1].w};
  }
};

// The tile a workgroup takes. Each XCD takes a run of tiles; within it eight token tiles at a time
// cross all features, so the tiles in flight share operand rows in its L2.
struct TilePlace {
  int f0, t0;
};
__device__ __forceinline__ bool tile_place(int tiles_f, int tiles_t, int nf, int bt, TilePlace& p) {
  const int total = tiles_f * tiles_t, per = (total + 7) >> 3;
  const int local = blockIdx.x >> 3, work = (blockIdx.x & 7) * per + local;
  if (local >= per || work >= total) return false;
  const int band = work / (8 * tiles_f), in = work - band * 8 * tiles_f;
  const int width = min(8, tiles_t - 8 * band);
  p.t0 = (8 * band + in % width) * bt;
  p.f0 = in / width * nf;
  return true;
}

// Results leave through LDS: a wave's 32 tokens x COLS features at a time, each token's row then written
// in whole lines (a lane's own 16 features are 32 bytes of a line: four times the requests). EDGE: the
// tile reaches past the matrix.
template <int EPI, typename T, int COLS, bool EDGE, int FT, int TT>
__device__ __forceinline__ void write_tile(const MxArgs& g, int fw, int tw0, char* mine, int lane,
                                           const f32x16 (&acc)[FT][TT]) {
  constexpr int kPitch = COLS * 2 + 16, kLanes = COLS / 8;  // bytes of an LDS row; lanes along one
  constexpr int NA = FT / outs_of(EPI), kOuts = EPI == kGluBwd ? 2 : 1;
  const int half = lane >> 5;
  if constexpr (EPI == kParts) {  // 64 bytes a lane, whole lines a pair of them
#pragma unroll
    for (int b = 0; b < TT; ++b)
#pragma unroll
      for (int a = 0; a < FT; ++a)
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const int t = tw0 + 32 * b + (lane & 31), f = fw + 32 * a + 16 * half + 4 * p;
          if (EDGE && (t >= g.m || f >= g.n)) continue;
          const float v[4] = {acc[a][b][4 * p], acc[a][b][4 * p + 1], acc[a][b][4 * p + 2], acc[a][b][4 * p + 3]};
          finish<EPI, T, 4>(g, t, f, v, v);
        }
    return;
  }
  auto settle = [] {  // the wave's own LDS accesses so far are done
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  };
  const int c = 8 * (lane % kLanes), f = fw + c;
  Pack<T, 8> dh[EPI == kGluBwd ? TT : 1][kLanes / 2];  // all of it at once: one latency
  if constexpr (EPI == kGluBwd) {
#pragma unroll
    for (int b = 0; b < TT; ++b)
#pragma unroll
      for (int i = 0; i < kLanes / 2; ++i) {
        const int t = tw0 + 32 * b + (i * 64 + lane) / kLanes;
        const T* src = static_cast<const T*>(g.dh) + static_cast<int64_t>(EDGE ? min(t, g.m - 1) : t) * g.ld_dh + f;
        if (!EDGE || f + 8 <= g.n) {
          dh[b][i] = __builtin_bit_cast(Pack<T, 8>, u32x4s(*reinterpret_cast<const u32x4u*>(src)));
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) dh[b][i].v[j] = f + j < g.n ? src[j] : static_cast<T>(0.0f);
        }
      }
  }
#pragma unroll
  for (int b = 0; b < TT; ++b) {
    const int tw = tw0 + 32 * b;
    if (EDGE && tw >= g.m) return;
    if constexpr (EPI == kGluBwd) {
#pragma unroll
      for (int i = 0; i < kLanes / 2; ++i)
        store_pack<T, 8>(reinterpret_cast<T*>(mine + (i * 64 + lane) / kLanes * kPitch + c * 2), dh[b][i]);
      settle();
    }
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        T* at = reinterpret_cast<T*>(mine + (lane & 31) * kPitch + (32 * a + 16 * half + 8 * p) * 2);
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = acc[a][b][8 * p + i];
        if constexpr (outs_of(EPI) == 2) {
          float u[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i] = acc[a + NA][b][8 * p + i];
          if constexpr (EPI == kGluFwd) {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = o[i] * glu_sigmoid(o[i]) * u[i];
          } else {
            float d[8], du[8];
            load_f32<T, 8>(at, d);
#pragma unroll
            for (int i = 0; i < 8; ++i) glu_bwd(d[i], o[i], u[i], o[i], du[i]);
            store_from_f32<T, 8>(at + 16 * kPitch, du);
          }
        }
        store_from_f32<T, 8>(at, o);
      }
    settle();
    T* y = static_cast<T*>(g.y) + f;
#pragma unroll
    for (int i = 0; i < kLanes / 2; ++i) {
      const int r = (i * 64 + lane) / kLanes;
      if (EDGE && (tw + r >= g.m || f >= g.n)) continue;
#pragma unroll
      for (int k = 0; k < kOuts; ++k) {
        const Pack<T, 8> v = load_pack<T, 8>(reinterpret_cast<const T*>(mine + (k * 32 + r) * kPitch + c * 2));
        T* dst = y + (tw + r) * g.ldy + k * g.n;
        if (!EDGE || f + 8 <= g.n) {
          *reinterpret_cast<u32x4u*>(dst) = __builtin_bit_cast(u32x4s, v);
        } else {
          for (int j = 0; j < 8; ++j)
            if (f + j < g.n) dst[j] = v.v[j];
        }
      }
    }
    settle();
  }
}

template <int FX, int FW, int EPI, typename T, int BF, int BT, int GROUPS>
__device__ __forceinline__ void mx_tile(const MxArgs& g, const TilePlace& tp, char* smem) {
  constexpr int THREADS = kTileThreads<BT>, WT = THREADS / kWave / 2;  // waves along the tokens
  constexpr int FT = BF / 64, TT = BT / 32 / WT;   // 32 x 32 results of a wave
  constexpr int NF = BF / outs_of(EPI);            // output features of a tile
  constexpr int PARTS = outs_of(EPI), kWaveRows = BF / 2 / PARTS;  // rows of W per wave and part
  typedef Copier<FW, BF, GROUPS, PARTS, THREADS> CW;
  typedef Copier<FX, BT, GROUPS, 1, THREADS> CX;
  typedef StepFrags<FW, FT, GROUPS, PARTS == 1 ? 0 : BF / 2> WF;
  typedef StepFrags<FX, TT, GROUPS, 0> XF;
  constexpr int kStage = CW::kBytes + CX::kBytes, kScales = (BF + BT) * 16;
  char* const scales = smem + 2 * kStage;
  const int f0 = tp.f0, t0 = tp.t0;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wf = wave / WT, wt = wave % WT;
  const bool edge = t0 + BT > g.m || f0 + NF > g.n;

  // rows past the edge re-read the last one; what they give is not stored
  auto w_part = [&](int i) -> int64_t { return f0 + static_cast<int64_t>(i) * g.n; };
  auto w_in = [&](int r) -> int { return min((r % NF & ~31) + feature_of(r & 31), g.n - 1 - f0); };
  auto x_part = [&](int) -> int64_t { return t0; };
  auto x_in = [&](int r) -> int { return min(r, g.m - 1 - t0); };
  CW cw;
  CX cx;
  const Range mine = EPI == kParts ? groups_of(g, blockIdx.z) : Range{0, g.nb / 4};
  cw.init(g.wc + 4 * mine.first * kCodeBytes<FW>, g.nb, w_part, w_in);
  cx.init(g.xc + 4 * mine.first * kCodeBytes<FX>, g.nb, x_part, x_in);
  ScaleRow sw, sx;
  const int sr = threadIdx.x;
  sw.src = g.ws + (w_part(sr % BF / NF) + w_in(sr % BF)) * g.nb + 4 * mine.first;
  sx.src = g.xs + (t0 + static_cast<int64_t>(x_in(sr % BT))) * g.nb + 4 * mine.first;

  const int groups = mine.count, stages = (groups + GROUPS - 1) / GROUPS;
  // The quad from group `first` on; where it is cut short the four groups that end the row. Group g's
  // word lies at g % 4 of its quad's place.
  auto quad_start = [&](int first) { return groups < 4 ? 0 : min(first, groups - 4); };
  auto load_scales = [&](int first) {
    sw.load(quad_start(first));
    sx.load(quad_start(first));
  };
  auto put_scales = [&](int first) {
    uint32_t* p = reinterpret_cast<uint32_t*>(scales + ((first >> 2) & 1) * kScales);
    const int start = quad_start(first);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t* word = p + ((start + j) & 3) * (BF + BT);
      if (BF >= THREADS || sr < BF) word[sr] = sw.v[j];
      if (BT >= THREADS || sr < BT) word[BF + sr] = sx.v[j];
    }
  };
  constexpr int kCopies = CW::kCopies + CX::kCopies;
  auto copy = [&](int s, auto I) {
    constexpr int i = decltype(I)::value;
    char* st = smem + (s & 1) * kStage;
    const bool last = GROUPS == 2 && (s + 1) * GROUPS > groups;
    if constexpr (i < CW::kCopies)
      cw.template copy<i>(s, last, st, wave);
    else if constexpr (i < kCopies)
      cx.template copy<i - CW::kCopies>(s, last, st + CW::kBytes, wave);
  };
  const int wr = wf * kWaveRows + (lane & 31), xr = wt * (BT / WT) + (lane & 31);
  const uint32_t wat = lds_addr(smem) + wr * CW::kRow, xat = lds_addr(smem) + CW::kBytes + xr * CX::kRow;
  const int wsw = swizzle<CW::kRow>(wr), xsw = swizzle<CX::kRow>(xr);
  const uint32_t wsat = lds_addr(scales) + wr * 4 + 2 * half, xsat = lds_addr(scales) + (BF + xr) * 4 + 2 * half;

  if (groups < 4) {
    sw.load_short(groups);
    sx.load_short(groups);
  } else {
    load_scales(0);
  }
  each<kCopies>([&](auto I) { copy(0, I); });

  // The sums start from the bias, or from a zero that the compiler does not see: a known one makes it run
  // the first stage in a copy of the loop of its own, with more registers than there are.
  float zero = 0.0f;
  asm volatile("" : "+v"(zero));
  f32x16 acc[FT][TT];
#pragma unroll
  for (int a = 0; a < FT; ++a) {
    f32x16 first;
#pragma unroll
    for (int i = 0; i < 16; ++i) first[i] = zero;
    if (EPI == kPlain && g.bias) {
      const int f = f0 + wf * (BF / 2) + 32 * a + 16 * half;
      const T* bias = static_cast<const T*>(g.bias);
      if (!edge) {
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const Pack<T, 8> v =
              __builtin_bit_cast(Pack<T, 8>, u32x4s(*reinterpret_cast<const u32x4u*>(bias + f + 8 * p)));
#pragma unroll
          for (int i = 0; i < 8; ++i) first[8 * p + i] = static_cast<float>(v.v[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) first[i] = static_cast<float>(bias[min(f + i, g.n - 1)]);
      }
    }
#pragma unroll
    for (int b = 0; b < TT; ++b) acc[a][b] = first;
  }
  put_scales(0);
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();

  // Everything but the products goes out between them, since a wave that issues reads or copies in a row
  // waits while the LDS or the address unit takes them: after each product of a step a part of the next
  // step's fragment reads and of the copies. The stage's one barrier falls before its last step, whose
  // fragments are in registers by then; that step then reads the next stage's first fragments and scales
  // and begins the copies of the stage after it, into the buffer just read.
  constexpr int kSteps = 2 * GROUPS, kMma = FT * TT;       // steps of a stage, products of a step
  constexpr int kStepReads = WF::kReads + XF::kReads, kScaleReads = GROUPS * (FT + TT);
  constexpr int kCopySlots = kSteps * kMma * 2 / 3;  // the rest of the stage is theirs to land
  uint32_t ws[GROUPS][FT], xs[GROUPS][TT], wn[GROUPS][FT], xn[GROUPS][TT];
  WF w[2];
  XF x[2];
  auto read_one = [&](int s, auto S, auto R) {  // fragment read R of step S of stage s
    constexpr int k = decltype(S)::value, r = decltype(R)::value;
    const uint32_t buf = (s & 1) * kStage;
    if constexpr (r < WF::kReads)
      w[k & 1].template read<k, r>(wat + buf, wsw, half);
    else
      x[k & 1].template read<k, r - WF::kReads>(xat + buf, xsw, half);
  };
  auto read_scale = [&](int s, auto R) {  // scale read R of stage s
    constexpr int r = decltype(R)::value, u = r / (FT + TT), i = r % (FT + TT);
    const int gi = GROUPS * s + u;
    const uint32_t sc = (gi & 3) * (BF + BT) * 4 + ((gi >> 2) & 1) * kScales;
    if constexpr (i < FT)
      wn[u][i] = lds_read2<WF::row_of(i) * 4>(wsat + sc);
    else
      xn[u][i - FT] = lds_read2<(i - FT) * 128>(xsat + sc);
  };
  auto send = [&](int s, auto SLOT) {  // the copies of stage s that go out in this slot
    each<kCopies>([&](auto I) {
      if constexpr (decltype(I)::value * kCopySlots / kCopies == decltype(SLOT)::value) copy(s, I);
    });
  };
  auto take_scales = [&] {
#pragma unroll
    for (int u = 0; u < GROUPS; ++u) {
#pragma unroll
      for (int a = 0; a < FT; ++a) {
        tie(wn[u][a]);
        ws[u][a] = wn[u][a];
      }
#pragma unroll
      for (int b = 0; b < TT; ++b) {
        tie(xn[u][b]);
        xs[u][b] = xn[u][b];
      }
    }
  };
  // Step S of stage s. NEXT: a step follows, in the next stage after the stage's last; SEND: a stage of
  // which copies go out here. Both known at compile time: a branch between products would let the
  // compiler gather them behind it.
  auto step = [&](int s, auto S, auto NEXT, auto SEND) {
    constexpr int k = decltype(S)::value, last = k == kSteps - 1;
    constexpr int reads = !decltype(NEXT)::value ? 0 : kStepReads + (last ? kScaleReads : 0);
    constexpr int early = kMma > 3 ? kMma * 3 / 4 : 1, per = (reads + early - 1) / early;
    each<kMma>([&](auto J) {
      constexpr int j = decltype(J)::value, a = j / TT, b = j % TT;
      acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
          w[k & 1].get(a), x[k & 1].get(b), acc[a][b], kMfmaFmt<FW>, kMfmaFmt<FX>, k & 1,
          (int)ws[k >> 1][a], k & 1, (int)xs[k >> 1][b]);
      __builtin_amdgcn_sched_barrier(0);
      each<per>([&](auto P) {
        constexpr int r = j * per + decltype(P)::value;
        if constexpr (r < kStepReads && r < reads)
          read_one(last ? s + 1 : s, std::integral_constant<int, (k + 1) % kSteps>{},
                   std::integral_constant<int, r>{});
        else if constexpr (r < reads)
          read_scale(s + 1, std::integral_constant<int, r - kStepReads>{});
      });
      if constexpr (decltype(SEND)::value)
        send(last ? s + 2 : s + 1, std::integral_constant<int, (last ? 0 : (k + 1) * kMma) + j>{});
      __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (decltype(NEXT)::value) {
      wait_lds<0>();
      w[(k + 1) & 1].tied();
      x[(k + 1) & 1].tied();
      if constexpr (last) take_scales();
    }
  };
  // Stage s with LEFT stages after it (2: or more).
  auto stage = [&](int s, auto LEFT) {
    constexpr int left = decltype(LEFT)::value;
    using More = std::integral_constant<bool, (left > 0)>;
    using More2 = std::integral_constant<bool, (left > 1)>;
    using Yes = std::true_type;
    if constexpr (left > 0) {  // scales of the next quad: fetched with the first stage of one, put down with its last
      const int g0 = GROUPS * s & 3, next = (GROUPS * s & ~3) + 4;
      if (next < groups) {
        if (g0 == 0) load_scales(next);
        if (g0 == 4 - GROUPS) put_scales(next);
      }
    }
    step(s, std::integral_constant<int, 0>{}, Yes{}, More{});
    if constexpr (GROUPS == 2) {
      step(s, std::integral_constant<int, 1>{}, Yes{}, More{});
      if constexpr (left == 0)
        if (2 * s + 1 == groups) return;  // the last stage has one group
      step(s, std::integral_constant<int, 2>{}, Yes{}, More{});
    }
    if constexpr (left > 0) {
      __builtin_amdgcn_s_waitcnt(0);  // stage s + 1 has landed (this wave's copies and scales) ...
      __syncthreads();                // ... and every wave's, and every wave has read stage s
    }
    step(s, std::integral_constant<int, kSteps - 1>{}, More{}, More2{});
  };

  if (stages > 1) each<kMma>([&](auto J) { send(1, J); });
  each<kStepReads>([&](auto R) { read_one(0, std::integral_constant<int, 0>{}, R); });
  each<kScaleReads>([&](auto R) { read_scale(0, R); });
  wait_lds<0>();
  w[0].tied();
  x[0].tied();
  take_scales();
  int s = 0;
  for (; s + 2 < stages; ++s) stage(s, std::integral_constant<int, 2>{});
  if (s + 1 < stages) stage(s++, std::integral_constant<int, 1>{});
  stage(s, std::integral_constant<int, 0>{});
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();  // every wave has read the last stage: results go over it

  constexpr int kCols = NF / 2, kMine = (EPI == kGluBwd ? 2 : 1) * 32 * (kCols * 2 + 16);
  static_assert(EPI == kParts || THREADS / kWave * kMine <= 2 * kStage + 2 * kScales, "the results fit");
  if (edge)
    write_tile<EPI, T, kCols, true>(g, f0 + wf * kCols, t0 + wt * (BT / WT), smem + wave * kMine, lane, acc);
  else
    write_tile<EPI, T, kCols, false>(g, f0 + wf * kCols, t0 + wt * (BT / WT), smem + wave * kMine, lane, acc);
}

template <int FX, int FW, int EPI, typename T, int BF, int BT, int GROUPS>
__global__ __launch_bounds__(kTileThreads<BT>) __attribute__((amdgpu_waves_per_eu(2))) void
mx_tile_kernel(MxArgs g, int tiles_f, int tiles_t) {
  constexpr int kBytes =
      2 * (BF * kStageRow<FW, GROUPS> + BT * kStageRow<FX, GROUPS> + (BF + BT) * 16);
  __shared__ __attribute__((aligned(16))) char smem[kBytes];
  TilePlace tp;
  if (!tile_place(tiles_f, tiles_t, BF / outs_of(EPI), BT, tp)) return;
  mx_tile<FX, FW, EPI, T, BF, BT, GROUPS>(g, tp, smem);
}

// y = T(the parts' sums, added in order, + bias), V features per thread.
template <typename T, int V, bool DEEP>
__global__ __launch_bounds__(256) void mx_sum_kernel(const float* __restrict__ parts, int splits,
                                                     int64_t m, int packs, int n,
                                                     const T* __restrict__ bias, T* __restrict__ y,
                                                     int64_t ldy) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= m * packs) return;
  const int64_t row = i / packs;
  const int f = static_cast<int>(i - row * packs) * V;
  const float* p = parts + row * n + f;
  float v[V];
  sum_parts<DEEP, V>(p, m * n, splits, v);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] += bias ? static_cast<float>(bias[f + j]) : 0.0f;
  store_from_f32<T, V>(y + row * ldy + f, v);
}

// ---- which kernel --------------------------------------------------------------------------------
//
// The one whose launch is estimated shortest. A launch takes a + groups (b + r (rounds - 1)) us, groups
// of four blocks of the contraction per workgroup, rounds of 256 workgroups (and c for each after the
// first); a contraction cut into parts pays for a second launch and 8 bytes a value and part.
//
// Measured (us a kernel, average of 20 on the same operands) at k = 1,536 / 8,960 with 16, 256, 512 and
// 1,024 workgroups:
//   fp8 by fp4  128 x 64   7.2, 8.4, 11.5, 19.3 / 29, 42, 50, 96      fp4 by fp4  6.6, 7.4, 9.8, 16.5 / 24, 32, 41, 78
//               128 x 128  7.8, 10.7, 16.8, 28.5 / 32, 52, 72, 146                6.8, 9.0, 13.1, 21.1 / 22, 35, 49, 97
//               256 x 128  11.0, 16.2, 25.6, 45.2 / 49, 68, 116, 238   256 x 256  11.8, 20.5, 37.6, 70.0 / 48, 76, 151, 306
//   fp8 by fp8  128 x 64   8.0, 9.5, 13.1, 23.3 / 32, 47, 57, 114     fp4 by fp8  8.1, 8.8, 12.2, 21.9 / 31, 44, 52, 106
//               128 x 128  8.7, 11.2, 17.3, 30.1 / 38, 56, 76, 166                7.9, 10.7, 15.9, 27.7 / 32, 50, 69, 147
// and the 32 x 32 kernel (fp8 by fp4) on 2,048 features 4.4 at one token, 5.1 at 32, 7.9 at 256; on 1,536
// features with k = 8,960 11.5 and 16.5 whole, 5.0 and 6.2 in five parts (and 2.5 to 3 for their sum).
// The estimates fit few workgroups and fall up to a third short where a round is full; the choice needs
// their order. It took the shortest kind measured in 41 of 44 products and gates of 33 to 8,161 tokens
// (1,536 to 17,920 features, all formats): 707 tokens x 2,048 128 x 64 (8.4; 128 x 128 9.0, 256 x 128
// 12.1), x 17,920 256 x 128 (23.4; 25.6, 28.4), 4,096 x 1,536 x 8,960 256 x 128 (63.2; 64.0, 73.6). Not
// at 192 tokens x 17,920 (256 x 128 13.5, 128 x 64 10.9) nor the 4-bit gate at 4,096 (78 and 76).
struct GemmPlan {
  int bf, bt, splits;  // bt 32: the 32 x 32 kernel
};

GemmPlan find_gemm_plan(int64_t m, int64_t n, int64_t nb, int x_fmt, int w_fmt, bool glu) {
  const bool both4 = x_fmt == RUS_MX_FP4 && w_fmt == RUS_MX_FP4;
  const double few = (0.1 + 0.0027 * static_cast<double>(m < 32 ? m : 32)) * (glu ? 1.6 : 1.0);
  const struct {
    int bf, bt;
    double a, b, r, c;
  } kinds[] = {{32, 32, 2.5, few, few, 0.0},
               {128, 64, both4 ? 2.75 : 2.5, both4 ? 0.25 : 0.32, both4 ? 0.35 : 0.375, 0.0},
               {128, 128, 3.0, both4 ? 0.25 : 0.364, both4 ? 0.4 : 0.6, 0.0},
               {256, 128, 4.0, 0.54, 0.875, 0.0},
               {256, 256, 4.0, 0.75, 0.83, 6.0}};
  const int64_t groups = nb / 4;
  GemmPlan best{32, 32, 1};
  double least = 1e300;
  for (const auto& k : kinds) {
    if (k.bf == 256 && (k.bt == 256 ? !both4 : x_fmt != RUS_MX_FP8 || w_fmt != RUS_MX_FP4)) continue;
    if (k.bt == 32 && m > 256) continue;
    const int64_t nf = k.bt == 32 || !glu ? k.bf : k.bf / 2;
    const int64_t tiles = ((n + nf - 1) / nf) * ((m + k.bt - 1) / k.bt);
    for (int64_t s = 1; s <= (glu ? 1 : 32) && 2 * s <= groups + 1; ++s) {
      const double rounds = static_cast<double>((tiles * s + 255) / 256 - 1);
      const double us = k.a + static_cast<double>((groups + s - 1) / s) * (k.b + k.r * rounds) + k.c * rounds +
                        (s > 1 ? 3.0 + 2e-6 * static_cast<double>(s) * static_cast<double>(m * n) : 0.0);
      if (us < least) {
        least = us;
        best = {k.bf, k.bt, static_cast<int>(s)};
      }
    }
  }
  return best;
}

GemmPlan gemm_plan(int64_t m, int64_t n, int64_t nb, int x_fmt, int w_fmt, bool glu) {
  static thread_local PlanMemo<GemmPlan> memo;
  return memo.get({m, n, nb, x_fmt * 4 + w_fmt * 2 + glu},
                  [&] { return find_gemm_plan(m, n, nb, x_fmt, w_fmt, glu); });
}

// (The 32 x 32 kernel always fits: below 2^23 workgroups of 256 along the features.)
int check_tiles(const char* fn, const GemmPlan& plan, int64_t m, int64_t n, bool glu) {
  if (plan.bt == 32) return RUS_OK;
  const int64_t nf = glu ? plan.bf / 2 : plan.bf;
  return check_items(fn, ((n + nf - 1) / nf) * ((m + plan.bt - 1) / plan.bt) + 7, plan.bt == 256 ? 512 : 256);
}

template <int EPI, typename T, int FX, int FW>
void launch(const MxArgs& g, const GemmPlan& plan, hipStream_t st) {
  constexpr int G = FX == kFp4 && FW == kFp4 ? 2 : 1;
  const unsigned parts = EPI == kParts ? g.splits : 1;
  auto tile = [&](auto kern, int bf, int bt) {
    const int nf = bf / outs_of(EPI);
    const int tiles_f = (g.n + nf - 1) / nf, tiles_t = (g.m + bt - 1) / bt;
    const int64_t total = static_cast<int64_t>(tiles_f) * tiles_t;
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(8 * ((total + 7) / 8)), 1, parts),
                       dim3(bt == 256 ? 512 : 256), 0, st, g, tiles_f, tiles_t);
  };
  if (plan.bt == 32)
    hipLaunchKernelGGL((mx_rows_kernel<FX, FW, EPI, T>), dim3((g.n + 31) / 32, (g.m + 31) / 32, parts),
                       dim3(kRowsWaves * kWave), 0, st, g);
  else if (plan.bt == 64)
    tile(mx_tile_kernel<FX, FW, EPI, T, 128, 64, G>, 128, 64);
  else if (plan.bf == 128)
    tile(mx_tile_kernel<FX, FW, EPI, T, 128, 128, G>, 128, 128);
  else if constexpr (FX == kFp4 && FW == kFp4)
    tile(mx_tile_kernel<FX, FW, EPI, T, 256, 256, G>, 256, 256);
  else if constexpr (FX == kFp8 && FW == kFp4)
    tile(mx_tile_kernel<FX, FW, EPI, T, 256, 128, G>, 256, 128);
}

template <int EPI, typename T>
void by_format(const MxArgs& g, const GemmPlan& plan, int32_t x_fmt, int32_t w_fmt, hipStream_t st) {
  if (x_fmt == RUS_MX_FP8)
    return w_fmt == RUS_MX_FP4 ? launch<EPI, T, kFp8, kFp4>(g, plan, st) : launch<EPI, T, kFp8, kFp8>(g, plan, st);
  return w_fmt == RUS_MX_FP4 ? launch<EPI, T, kFp4, kFp4>(g, plan, st) : launch<EPI, T, kFp4, kFp8>(g, plan, st);
}

// The gated products; `first` runs once nothing is left to refuse.
template <int EPI, typename F>
int dispatch(const char* fn, const MxArgs& g, int32_t x_fmt, int32_t w_fmt, int32_t dtype, hipStream_t st, F first) {
  const GemmPlan plan = gemm_plan(g.m, g.n, g.nb, x_fmt, w_fmt, true);
  if (int e = check_tiles(fn, plan, g.m, g.n, true)) return e;
  if (int e = first()) return e;
  if (dtype == RUS_DTYPE_BF16)
    by_format<EPI, bf16>(g, plan, x_fmt, w_fmt, st);
  else
    by_format<EPI, f16>(g, plan, x_fmt, w_fmt, st);
  return check_launch(fn);
}

// The plain product: one launch, or the parts and their sum.
template <typename T>
int product(const char* fn, MxArgs g, const GemmPlan& plan, int32_t x_fmt, int32_t w_fmt, float* parts,
            hipStream_t st) {
  if (plan.splits == 1) {
    by_format<kPlain, T>(g, plan, x_fmt, w_fmt, st);
    return check_launch(fn);
  }
  T* y = static_cast<T*>(g.y);
  const T* bias = static_cast<const T*>(g.bias);
  const bool wide = g.n % 4 == 0 && g.ldy % 4 == 0 && aligned(y, 8);
  const int packs = wide ? g.n / 4 : g.n;
  g.splits = plan.splits;
  g.bias = nullptr;
  g.vec = g.n % 4 == 0;
  g.y = parts;
  by_format<kParts, f16>(g, plan, x_fmt, w_fmt, st);
  if (int e = check_launch(fn)) return e;
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(g.m) * packs + 255) / 256));
  auto add = [&](auto k) {
    hipLaunchKernelGGL(k, grid, dim3(256), 0, st, parts, plan.splits, static_cast<int64_t>(g.m), packs, g.n, bias, y,
                       g.ldy);
  };
  if (deep_sum(static_cast<int64_t>(g.m) * packs, plan.splits))
    wide ? add(mx_sum_kernel<T, 4, true>) : add(mx_sum_kernel<T, 1, true>);
  else
    wide ? add(mx_sum_kernel<T, 4, false>) : add(mx_sum_kernel<T, 1, false>);
  return check_launch(fn);
}

int check_sizes(const char* fn, int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n <= 0 || k <= 0 || m >= (1 << 30) || n >= (1 << 28) || k > (1 << 22))
    return fail(RUS_ERR_INVALID, "%s: bad sizes m=%lld n=%lld k=%lld", fn, (long long)m, (long long)n,
                (long long)k);
  return RUS_OK;
}

// What a plan depends on: nothing is planned, or remembered, for formats that do not exist.
int check_plan(const char* fn, int64_t m, int64_t n, int64_t k, int32_t x_fmt, int32_t w_fmt) {
  if (int e = check_sizes(fn, m, n, k)) return e;
  if (int e = check_format(fn, x_fmt, "x")) return e;
  return check_format(fn, w_fmt, "w");
}

// Checks shared by the three entry points; fills what they share.
int prepare(const char* fn, MxArgs& g, const void* xc, const void* xs, int32_t x_fmt, const void* wc,
            const void* ws, int32_t w_fmt, int64_t m, int64_t n, int64_t k, void* y,
            int64_t ldy, int64_t y_cols, int32_t dtype, bool raw = false) {
  if (int e = check_sizes(fn, m, n, k)) return e;
  if (dtype != RUS_DTYPE_F16 && dtype != RUS_DTYPE_BF16)
    return fail(RUS_ERR_UNSUPPORTED, "%s: results are fp16 or bf16, not dtype %d", fn, (int)dtype);
  if (ldy < y_cols && m > 1)
    return fail(RUS_ERR_INVALID, "%s: output row stride %lld smaller than %lld columns", fn,
                (long long)ldy, (long long)y_cols);
  if (m == 0) return RUS_OK;
  if (!raw)
    if (int e = check_mx(fn, xc, xs, x_fmt, "x")) return e;
  if (int e = check_mx(fn, wc, ws, w_fmt, "w")) return e;
  if (!y || !aligned(y, 2)) return fail(RUS_ERR_INVALID, "%s: output is null or misaligned", fn);
  g = MxArgs{};
  g.xc = static_cast<const uint8_t*>(xc);
  g.xs = static_cast<const uint8_t*>(xs);
  g.wc = static_cast<const uint8_t*>(wc);
  g.ws = static_cast<const uint8_t*>(ws);
  g.m = static_cast<int>(m);
  g.n = static_cast<int>(n);
  g.nb = static_cast<int>(mx_blocks(k));
  g.y = y;
  g.ldy = ldy;
  g.splits = 1;
  g.vec = aligned(y, 16) && ldy % 8 == 0 && n % 8 == 0;
  return RUS_OK;
}

}  // namespace
}  // namespace rus

using namespace rus;

extern "C" int rus_mx_gemm_workspace(int64_t m, int64_t n, int64_t k, int32_t x_fmt, int32_t w_fmt,
                                     int64_t* floats) {
  const char* fn = "rus_mx_gemm_workspace";
  if (!floats) return fail(RUS_ERR_INVALID, "%s: null result", fn);
  if (int e = check_plan(fn, m, n, k, x_fmt, w_fmt)) return e;
  const GemmPlan p = gemm_plan(m, n, mx_blocks(k), x_fmt, w_fmt, false);
  *floats = m > 0 && !few_tokens(m, n, mx_blocks(k)) && p.splits > 1 ? p.splits * m * n : 0;
  return RUS_OK;
}

extern "C" int rus_mx_gemm_plan(int64_t m, int64_t n, int64_t k, int32_t x_fmt, int32_t w_fmt, int32_t glu,
                                int32_t* plan) {
  const char* fn = "rus_mx_gemm_plan";
  if (!plan) return fail(RUS_ERR_INVALID, "%s: null result", fn);
  if (int e = check_plan(fn, m, n, k, x_fmt, w_fmt)) return e;
  const int64_t nb = mx_blocks(k);
  const bool few = glu != 2 && few_tokens(m, n, nb);
  const GemmPlan p = gemm_plan(m, n, nb, x_fmt, w_fmt, glu != 0);
  plan[0] = few ? 8 : p.bf;
  plan[1] = few ? static_cast<int32_t>(m) : p.bt;
  plan[2] = few ? 1 : p.splits;
  return RUS_OK;
}

// Scratch of a call that quantises its activations: codes, scales, sums, each 16-byte aligned.
namespace rus {
namespace {
struct RowsScratch {
  int64_t codes, scales, sums;
  int64_t bytes() const { return codes + scales + 4 * sums; }
};
RowsScratch rows_scratch(int64_t m, int64_t n, int64_t k, int32_t act, int32_t w_fmt, bool glu) {
  const int64_t nb = mx_blocks(k);
  if (few_tokens(m, n, nb)) return {0, 0, 0};
  const GemmPlan p = gemm_plan(m, n, nb, act, w_fmt, glu);
  return {m * nb * (act == RUS_MX_FP4 ? 16 : 32), (m * nb + 15) / 16 * 16, p.splits > 1 ? p.splits * m * n : 0};
}
// The scratch's parts, or a refusal.
int place(const char* fn, const RowsScratch& need, void* scratch, int64_t n_scratch, char*& codes, char*& scales,
          float*& sums) {
  if (!scratch || !aligned(scratch, 16) || n_scratch < need.bytes())
    return fail(RUS_ERR_INVALID, "%s: scratch holds %lld bytes (16-byte aligned), needs %lld", fn,
                (long long)n_scratch, (long long)need.bytes());
  codes = static_cast<char*>(scratch);
  scales = codes + need.codes;
  sums = need.sums ? reinterpret_cast<float*>(scales + need.scales) : nullptr;
  return RUS_OK;
}

TokenArgs token_args(const MxArgs& g, int x_fmt, int64_t k, const void* bias) {
  return {nullptr, 0, g.xc, g.xs, g.wc, g.ws, x_fmt, g.m, g.n, static_cast<int>(k), g.nb, bias, g.y, g.ldy};
}

// rus_mx_gemm and rus_mx_glu_fwd.
template <typename F>
int run_gemm(const char* fn, const void* xc, const void* xs, int32_t x_fmt, const void* wc, const void* ws,
             int32_t w_fmt, int64_t m, int64_t n, int64_t k, const void* bias, void* y, int64_t ldy,
             int32_t dtype, float* workspace, int64_t n_workspace, void* stream, F first) {
  MxArgs g;
  if (int e = prepare(fn, g, xc, xs, x_fmt, wc, ws, w_fmt, m, n, k, y, ldy, n, dtype)) return e;
  if (m == 0) return RUS_OK;
  if (bias && !aligned(bias, 2)) return fail(RUS_ERR_INVALID, "%s: misaligned bias", fn);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (few_tokens(m, n, g.nb))
    return token_product(fn, token_args(g, x_fmt, k, bias), w_fmt, false, dtype == RUS_DTYPE_BF16, st);
  const GemmPlan plan = gemm_plan(m, n, g.nb, x_fmt, w_fmt, false);
  if (int e = check_tiles(fn, plan, m, n, false)) return e;
  if (plan.splits > 1 && (n_workspace < plan.splits * m * n || !workspace || !aligned(workspace, 16)))
    return fail(RUS_ERR_INVALID, "%s: workspace holds %lld floats (16-byte aligned), needs %lld", fn,
                (long long)n_workspace, (long long)(plan.splits * m * n));
  g.bias = bias;
  g.vec = g.vec && (!bias || aligned(bias, 16));
  if (int e = first()) return e;
  return dtype == RUS_DTYPE_BF16 ? product<bf16>(fn, g, plan, x_fmt, w_fmt, workspace, st)
                                 : product<f16>(fn, g, plan, x_fmt, w_fmt, workspace, st);
}

template <typename F>
int run_glu(const char* fn, const void* xc, const void* xs, int32_t x_fmt, const void* wc, const void* ws,
            int32_t w_fmt, int64_t m, int64_t n, int64_t k, void* h, int64_t ldh, int32_t dtype, void* stream,
            F first) {
  MxArgs g;
  if (int e = prepare(fn, g, xc, xs, x_fmt, wc, ws, w_fmt, m, n, k, h, ldh, n, dtype)) return e;
  if (m == 0) return RUS_OK;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (few_tokens(m, n, g.nb))
    return token_product(fn, token_args(g, x_fmt, k, nullptr), w_fmt, true, dtype == RUS_DTYPE_BF16, st);
  return dispatch<kGluFwd>(fn, g, x_fmt, w_fmt, dtype, st, first);
}

// A few tokens that are rounded to blocks inside the product.
int run_tokens(const char* fn, const void* x, int64_t ldx, int32_t act, const void* wc, const void* ws,
               int32_t w_fmt, int64_t m, int64_t n, int64_t k, const void* bias, void* y, int64_t ldy,
               int32_t dtype, bool glu, void* stream) {
  MxArgs g;
  if (int e = prepare(fn, g, nullptr, nullptr, act, wc, ws, w_fmt, m, n, k, y, ldy, n, dtype, true)) return e;
  if (ldx < k && m > 1) return fail(RUS_ERR_INVALID, "%s: stride_x=%lld smaller than a row", fn, (long long)ldx);
  if (!x || !aligned(x, 2)) return fail(RUS_ERR_INVALID, "%s: x is null or misaligned", fn);
  if (bias && !aligned(bias, 2)) return fail(RUS_ERR_INVALID, "%s: misaligned bias", fn);
  TokenArgs t = token_args(g, act, k, bias);
  t.x = x;
  t.ldx = ldx;
  return token_product(fn, t, w_fmt, glu, dtype == RUS_DTYPE_BF16, static_cast<hipStream_t>(stream));
}

}  // namespace
}  // namespace rus

extern "C" int rus_mx_gemm(const void* x_codes, const void* x_scales, int32_t x_fmt,
                           const void* w_codes, const void* w_scales, int32_t w_fmt, int64_t m,
                           int64_t n, int64_t k, const void* bias, void* y, int64_t stride_y,
                           int32_t dtype, float* workspace, int64_t n_workspace, void* stream) {
  return run_gemm("rus_mx_gemm", x_codes, x_scales, x_fmt, w_codes, w_scales, w_fmt, m, n, k, bias, y,
                  stride_y, dtype, workspace, n_workspace, stream, [] { return RUS_OK; });
}

extern "C" int rus_mx_rows_scratch(int64_t m, int64_t n, int64_t k, int32_t act, int32_t w_fmt, int32_t glu,
                                   int64_t* bytes) {
  const char* fn = "rus_mx_rows_scratch";
  if (!bytes) return fail(RUS_ERR_INVALID, "%s: null result", fn);
  if (int e = check_plan(fn, m, n, k, act, w_fmt)) return e;
  *bytes = m > 0 ? rows_scratch(m, n, k, act, w_fmt, glu != 0).bytes() : 0;
  return RUS_OK;
}

extern "C" int rus_mx_gemm_rows(const void* x, int64_t stride_x, int32_t act, const void* w_codes,
                                const void* w_scales, int32_t w_fmt, int64_t m, int64_t n, int64_t k,
                                const void* bias, void* y, int64_t stride_y, int32_t dtype,
                                void* scratch, int64_t n_scratch, void* stream) {
  const char* fn = "rus_mx_gemm_rows";
  if (int e = check_sizes(fn, m, n, k)) return e;
  if (m == 0) return RUS_OK;
  if (int e = check_plan(fn, m, n, k, act, w_fmt)) return e;
  if (few_tokens(m, n, mx_blocks(k)))
    return run_tokens(fn, x, stride_x, act, w_codes, w_scales, w_fmt, m, n, k, bias, y, stride_y, dtype, false,
                      stream);
  const RowsScratch need = rows_scratch(m, n, k, act, w_fmt, false);
  char *codes, *scales;
  float* sums;
  if (int e = place(fn, need, scratch, n_scratch, codes, scales, sums)) return e;
  return run_gemm(fn, codes, scales, act, w_codes, w_scales, w_fmt, m, n, k, bias, y, stride_y, dtype, sums,
                  need.sums, stream, [&] {
                    return quantize_rows(fn, x, dtype, m, k, stride_x, act, codes, scales,
                                         static_cast<hipStream_t>(stream));
                  });
}

extern "C" int rus_mx_glu_fwd_rows(const void* x, int64_t stride_x, int32_t act, const void* w_codes,
                                   const void* w_scales, int32_t w_fmt, int64_t m, int64_t n, int64_t k,
                                   void* h, int64_t stride_h, int32_t dtype, void* scratch,
                                   int64_t n_scratch, void* stream) {
  const char* fn = "rus_mx_glu_fwd_rows";
  if (int e = check_sizes(fn, m, n, k)) return e;
  if (m == 0) return RUS_OK;
  if (int e = check_plan(fn, m, n, k, act, w_fmt)) return e;
  if (few_tokens(m, n, mx_blocks(k)))
    return run_tokens(fn, x, stride_x, act, w_codes, w_scales, w_fmt, m, n, k, nullptr, h, stride_h, dtype, true,
                      stream);
  char *codes, *scales;
  float* sums;
  if (int e = place(fn, rows_scratch(m, n, k, act, w_fmt, true), scratch, n_scratch, codes, scales, sums))
    return e;
  return run_glu(fn, codes, scales, act, w_codes, w_scales, w_fmt, m, n, k, h, stride_h, dtype, stream, [&] {
    return quantize_rows(fn, x, dtype, m, k, stride_x, act, codes, scales, static_cast<hipStream_t>(stream));
  });
}

extern "C" int rus_mx_glu_fwd(const void* x_codes, const void* x_scales, int32_t x_fmt,
                              const void* w_codes, const void* w_scales, int32_t w_fmt, int64_t m,
                              int64_t n, int64_t k, void* h, int64_t stride_h, int32_t dtype,
                              void* stream) {
  return run_glu("rus_mx_glu_fwd", x_codes, x_scales, x_fmt, w_codes, w_scales, w_fmt, m, n, k, h, stride_h,
                 dtype, stream, [] { return RUS_OK; });
}

extern "C" int rus_mx_glu_bwd(const void* dh, int64_t stride_dh, const void* x_codes,
                              const void* x_scales, int32_t x_fmt, const void* w_codes,
                              const void* w_scales, int32_t w_fmt, int64_t m, int64_t n, int64_t k,
                              void* d_gu, int64_t stride_d_gu, int32_t dtype, void* stream) {
  const char* fn = "rus_mx_glu_bwd";
  MxArgs g;
  if (int e = prepare(fn, g, x_codes, x_scales, x_fmt, w_codes, w_scales, w_fmt, m, n, k, d_gu,
                      stride_d_gu, 2 * n, dtype))
    return e;
  if (m == 0) return RUS_OK;
  if (stride_dh < n && m > 1)
    return fail(RUS_ERR_INVALID, "%s: stride_dh=%lld smaller than a row", fn, (long long)stride_dh);
  if (!dh || !aligned(dh, 2)) return fail(RUS_ERR_INVALID, "%s: dh is null or misaligned", fn);
  g.dh = dh;
  g.ld_dh = stride_dh;
  g.vec = g.vec && aligned(dh, 16) && stride_dh % 8 == 0;
  return dispatch<kGluBwd>(fn, g, x_fmt, w_fmt, dtype, static_cast<hipStream_t>(stream), [] { return RUS_OK; });
}
