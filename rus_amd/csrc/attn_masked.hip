// Attention over packed rows with a tanh cap on the scores, a bias by distance, a prefix that every query sees, and
// fewer queries than keys where a cache is read: forward and backward, fp16 / bf16, head dims 64 and 128. The
// definition is in attn_masked.h.
#include <algorithm>
#include <type_traits>

#include "attn_masked.h"
#include "attn_masked_tiles.h"

namespace rus {
namespace {

constexpr int kWaves = 4, kRows = 128;  // waves of a block, tokens of a block
constexpr int kFwdTiles = 2;             // key tiles per stage of the forward

// Blocks a CU that the registers are divided for. 16 heads of 64, us with two / three: eight rows of 700 forward 35 / 31,
// backward 112 / 89, two of 2,048 59 / 50, 146 / 145; 1,025 + 577 + 257 + 64 with a cap 30 / 27, 77 / 73. The backward's
// dQ blocks of 32 tokens keep two: their sums would go to scratch memory (the same tokens 73 / 79).
template <int HD>
constexpr int kCuBlocks = HD == 64 ? 3 : 2;

// Block id -> (item, head): the query heads of a KV group that work on one item take ids 8 apart, i.e. one XCD (ids go
// round robin over the 8), so that they read their shared keys from one L2. False past the last item.
__device__ __forceinline__ bool head_item(const MaskedArgs& a, int n_items, int& item, int& head) {
  const int grp = a.h_q / a.h_kv, chunk = 8 * grp;
  const int t = blockIdx.x / chunk, r = blockIdx.x % chunk;
  const int64_t i = static_cast<int64_t>(t) * chunk + (r & 7) * grp + (r >> 3);
  item = static_cast<int>(i / a.h_q);
  head = static_cast<int>(i % a.h_q);
  return i / a.h_q < n_items;
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ MaskedRow uniform(MaskedRow r) {
  return MaskedRow{uniform(r.qa), uniform(r.lq), uniform(r.ka), uniform(r.lk), uniform(r.pre)};
}

// ---------------------------------------------------------------------------------------------
// Forward. S^T = K Q^T on 32 NT keys: a lane owns one query (column) and half of the keys; the running maximum and sum
// are per-lane scalars, and P^T feeds O^T += V^T P^T from the accumulator. m is the running maximum itself at every
// step, and O is divided by lr, the sum of the rounded P, in which their common rounding cancels (l, of the unrounded,
// gives the lse). P is rounded to T because the matrix instruction takes nothing wider at its rate; everything else
// stays in 32 bits.
// ---------------------------------------------------------------------------------------------
template <int ND>
struct FwdState {
  f32x16 o[ND];
  float m, l, lr;
  __device__ __forceinline__ FwdState() : m(-INFINITY), l(0.0f), lr(0.0f) {
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f32x16{};
  }
};

// left: keys of the lane's query from the first of these on that it sees; whole: every query of the wave sees all.
// d0: distance of the lane's first element (key 4 h). keys_read() is called when the K tiles have been read,
// values_ready() before the V tiles are.
template <typename T, int HD, bool CAP, bool BIAS, int NT, typename F, typename G>
__device__ __forceinline__ void fwd_keys(const MaskedArgs& a, const FragLane<HD>& fl, const char* kt, const char* vt,
                                         const Frag (&qf)[HD / 16], FwdState<HD / 32>& w,
                                         const Scorer<CAP, BIAS>& sc, bool whole, int left, float d0, bool ahead, int h,
                                         F keys_read, G values_ready) {
  using L = Tiles<HD>;
  f32x16 st[NT];
  start_scores<CAP, BIAS, NT>(st, sc.slope, d0, 1.0f, ahead);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int s = 0; s < L::kSteps; ++s) st[n] = mfma<T>(fl.frag(kt + n * L::kBytes, s), qf[s], st[n]);
  }
  keys_read();
  // (without a cap scaled inside the exponential)
  if constexpr (CAP) capped_scores<BIAS, NT, false>(a, sc.slope2, st, st, d0, 1.0f);
  if (!whole) {
    const int most = left - 4 * h;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) st[n][r] = 32 * n + acc_row(r, 0) < most ? st[n][r] : -INFINITY;
  }
  float mx = -INFINITY;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[n][r]);
  const float2 mp = half_pair(mx);
  mx = fmaxf(mp.x, mp.y);
  if constexpr (!CAP) mx *= a.sl2;  // scale > 0
  const float mn = fmaxf(w.m, mx);
  const float ref = mn == -INFINITY ? 0.0f : mn;  // nothing seen yet: every P is 2^-inf
  if (__ballot(mx > w.m)) {
    const float alpha = exp2_raw(w.m - ref);
    w.l *= alpha;
    w.lr *= alpha;
    w.m = mn;
#pragma unroll
    for (int d = 0; d < L::kDims; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) w.o[d][r] *= alpha;
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float rs = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float p = exp2_raw(CAP ? st[n][r] - ref : __builtin_fmaf(st[n][r], a.sl2, -ref));
      st[n][r] = p;
      rs += p;
    }
    w.l += rs;  // this lane's 16 keys; the other half's join at the end
  }
  values_ready();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const Frag p0 = frag_acc<T>(st[n], 0), p1 = frag_acc<T>(st[n], 1);
    w.lr = sum8<T>(p1, sum8<T>(p0, w.lr));
#pragma unroll
    for (int d = 0; d < L::kDims; ++d) {
      w.o[d] = mfma<T>(fl.frag_t(vt + n * L::kBytes, 0, d), p0, w.o[d]);  // O^T += V^T P^T
      w.o[d] = mfma<T>(fl.frag_t(vt + n * L::kBytes, 1, d), p1, w.o[d]);
    }
  }
}

template <typename T, int HD>
__device__ __forceinline__ void load_row_frags(Frag (&f)[HD / 16], const T* row, int h) {
#pragma unroll
  for (int s = 0; s < HD / 16; ++s) f[s] = *reinterpret_cast<const Frag*>(row + 16 * s + 8 * h);
}

// 128 queries of one head, 32 to a wave; tiles of 32 keys stream through double-buffered LDS, two to a stage, each
// copied once for all four waves while the previous stage is used. Hidden keys reach the product as 0 x V: where V is
// not finite the sums are not either, and such a query is formed again by itself (plain_fwd_row). Bound by the products
// and the exponentials beside them, which two blocks a CU overlap: 4,096 + 2,048 + 1,024 + 993 tokens, 12 / 2 heads of
// 128, bf16 with a bias 117 us (600 TFLOP/s of what is visible), one row of 4,096 104 us (490): the longest row's last
// blocks run by themselves.
template <typename T, int HD, bool CAP, bool BIAS>
__device__ __forceinline__ void fwd_block(const MaskedArgs& a, char* buf0, char* buf1) {
  using L = Tiles<HD>;
  constexpr int NT = kFwdTiles;
  int item, head, s, b, nb;
  if (!head_item(a, a.n_blocks, item, head)) return;
  if (!find_span_block(a.cu_q, a.n_seq, static_cast<int>(a.n_q), item, kRows, s, b, nb)) return;
  const MaskedRow r = uniform(as_queries(masked_row(a, s), s, a.n_seq));
  b = uniform(nb - 1 - b);  // the last queries see the most keys: first
  const int g = head / (a.h_q / a.h_kv);
  const int wave = uniform(static_cast<int>(threadIdx.x) >> 6);
  const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
  const int i0 = b * kRows, iw = i0 + 32 * wave, i = min(iw + col, r.lq - 1);
  const bool valid = iw + col < r.lq;
  const int vis = r.vis(i, a.causal);
  const int tiles = (r.vis(min(i0 + kRows, r.lq) - 1, a.causal) + 31) / 32;
  const int stages = (tiles + NT - 1) / NT;
  // Keys that all of the wave's queries see, and that any does.
  const int vis_all = iw < r.lq ? r.vis(iw, a.causal) : 0;
  const int mine = iw < r.lq ? (r.vis(min(iw + 31, r.lq - 1), a.causal) + 31) / 32 : 0;
  const T* kh = token<T>(a.k, r.ka, a.k_st, g, a.k_sh);
  const T* vh = token<T>(a.v, r.ka, a.v_st, g, a.v_sh);
  constexpr int C = L::kCopies / kWaves;
  const TileLane<HD, C> tk(C * wave, lane, a.k_st), tv(C * wave, lane, a.v_st);
  const FragLane<HD> fl0(lane);
  const Scorer<CAP, BIAS> sc(a, head);
  auto copy = [&](char* dst, int j) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int t = min(NT * j + n, tiles - 1);  // (behind the last tile: the last again, hidden)
      const int rows = r.lk - 32 * t;
      tk.copy(dst + n * L::kBytes, kh + 32 * t * a.k_st, rows);
      tv.copy(dst + (NT + n) * L::kBytes, vh + 32 * t * a.v_st, rows);
    }
  };
  if (stages) copy(buf0, 0);
  Frag qf[L::kSteps];
  load_row_frags<T, HD>(qf, token<T>(a.q, r.qa + i, a.q_st, head, a.q_sh), h);
  FwdState<L::kDims> w;
  stage_barrier();
  auto stage = [&](const char* cur, char* next, int j) {
    if (j + 1 < stages) copy(next, j + 1);
    const char* vt = cur + NT * L::kBytes;
    const FragLane<HD> fl = fl0.fresh();
    const int mt = mine - NT * j, k0 = 32 * NT * j;  // this wave's tiles from here on, first key
    const float d0 = static_cast<float>(r.off() + i - k0 - 4 * h);
    if (mt > 0)
      fwd_keys<T, HD, CAP, BIAS, NT>(a, fl, cur, vt, qf, w, sc, k0 + 32 * NT <= vis_all, vis - k0, d0,
                                     k0 + 32 * NT - 1 <= r.off() + iw, h, [] {}, [] {});
    stage_barrier();
  };
  for (int j = 0; j < stages; j += 2) {
    stage(buf0, buf1, j);
    if (j + 1 < stages) stage(buf1, buf0, j + 1);
  }
  if (iw >= r.lq) return;
  const float2 lp = half_pair(w.l), rp = half_pair(w.lr);
  const float f = vis > 0 ? 1.0f / (rp.x + rp.y) : 0.0f;
  if (vis <= 0) {
#pragma unroll
    for (int d = 0; d < L::kDims; ++d) w.o[d] = f32x16{};
  }
  uint64_t again = __ballot(valid && !all_finite(w.o, f));
  uint32_t cols = static_cast<uint32_t>(again) | static_cast<uint32_t>(again >> 32);
  const bool keep = valid && !((cols >> col) & 1);
  const int64_t t = r.qa + i;
  store_row<T, L::kDims>(static_cast<T*>(a.out) + (t * a.h_q + head) * HD, w.o, f, h, keep);
  if (h == 0 && keep) a.lse[head * a.n_q + t] = vis > 0 ? (w.m + log2f(lp.x + lp.y)) * kLn2 : -INFINITY;
  for (; cols; cols &= cols - 1) plain_fwd_row<T, HD, CAP, BIAS>(a, r, iw + __builtin_ctz(cols), head);
}

template <typename T, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * kWaves)
__attribute__((amdgpu_waves_per_eu(kCuBlocks<HD>, kCuBlocks<HD>))) void masked_fwd_kernel(
    MaskedArgs a) {
  __shared__ __attribute__((aligned(16))) char buf0[2 * kFwdTiles * Tiles<HD>::kBytes];
  __shared__ __attribute__((aligned(16))) char buf1[2 * kFwdTiles * Tiles<HD>::kBytes];
  fwd_block<T, HD, CAP, BIAS>(a, buf0, buf1);
}

// ---------------------------------------------------------------------------------------------
// Few queries over many keys: a block holds up to 32 (query, head) pairs of one KV head as the columns of S^T, so that
// K and V are read once for all of the group's heads, its waves take key tiles in turn (each with LDS of its own, no
// barrier in the loop), and the keys are split over blocks whose parts another launch joins. Part: per column the sum
// of P V on the part's own maximum, then that maximum, the sum of P and the sum of the rounded P. Bound by reading K and
// V once few queries are left: one token over 131,071 keys, 2 KV heads of 128, 26 us (5.1 TB/s), eight over 15,253 keys
// in all 12 us; rows of some hundred tokens by a row's tiles in turn (707 tokens 12 us).
// ---------------------------------------------------------------------------------------------
constexpr int kMaxSplitGroup = 32;

__host__ __device__ inline int split_tokens(int grp) { return 32 / grp; }  // queries of a block

template <typename T, int HD, bool CAP, bool BIAS>
__device__ __forceinline__ void split_block(const MaskedArgs& a, char* kbuf, char* vbuf) {
  using L = Tiles<HD>;
  const int grp = a.h_q / a.h_kv, tpb = split_tokens(grp);
  const int z = blockIdx.x % a.splits, rest = blockIdx.x / a.splits;
  const int g = rest % a.h_kv, item = rest / a.h_kv;
  int s, b, nb;
  if (!find_span_block(a.cu_q, a.n_seq, static_cast<int>(a.n_q), item, tpb, s, b, nb)) return;
  const MaskedRow r = uniform(as_queries(masked_row(a, s), s, a.n_seq));
  b = uniform(b);
  const int wave = uniform(static_cast<int>(threadIdx.x) >> 6);
  const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
  const int i0 = b * tpb, nq = min(tpb, r.lq - i0);  // the block's first query, its queries
  const bool valid = col < nq * grp;
  const int i = i0 + (valid ? col / grp : 0), head = g * grp + (valid ? col % grp : 0);
  const int vis = r.vis(i, a.causal), vis_all = r.vis(i0, a.causal);
  const int tiles = (r.vis(i0 + nq - 1, a.causal) + 31) / 32;
  const int first = z * a.split_tiles;
  if (first >= tiles && z > 0) return;  // the join knows
  const int last = z == a.splits - 1 ? tiles : min(tiles, first + a.split_tiles);
  const T* kh = token<T>(a.k, r.ka, a.k_st, g, a.k_sh);
  const T* vh = token<T>(a.v, r.ka, a.v_st, g, a.v_sh);
  const TileLane<HD, L::kCopies> tk(0, lane, a.k_st), tv(0, lane, a.v_st);
  const FragLane<HD> fl0(lane);
  const Scorer<CAP, BIAS> sc(a, head);
  char* kt = kbuf + wave * L::kBytes;
  char* vt = vbuf + wave * L::kBytes;
  // One K and one V tile a wave: the next K tile is on its way once this one's products are formed, the next V tile once
  // this one's are, so that either has the other's work to arrive under (and two blocks fit a CU).
  auto copy_k = [&](int t) { tk.copy(kt, kh + 32 * t * a.k_st, r.lk - 32 * t); };
  auto copy_v = [&](int t) { tv.copy(vt, vh + 32 * t * a.v_st, r.lk - 32 * t); };
  if (first + wave < last) {
    copy_k(first + wave);
    copy_v(first + wave);
  }
  Frag qf[L::kSteps];
  load_row_frags<T, HD>(qf, token<T>(a.q, r.qa + i, a.q_st, head, a.q_sh), h);
  FwdState<L::kDims> w;
  stage_wait();
  for (int t = first + wave; t < last; t += kWaves) {
    const FragLane<HD> fl = fl0.fresh();
    const int k0 = 32 * t;
    const bool more = t + kWaves < last;
    if (t > first + wave) wait_copies<L::kCopies>();  // this K tile; the V tile behind it may be on its way
    fwd_keys<T, HD, CAP, BIAS, 1>(
        a, fl, kt, vt, qf, w, sc, k0 + 32 <= vis_all, vis - k0, static_cast<float>(r.off() + i - k0 - 4 * h),
        k0 + 31 <= r.off() + i0, h,
        [&] {
          wait_reads();
          if (more) copy_k(t + kWaves);
        },
        [&] {
          if (more)
            wait_copies<L::kCopies>();  // this V tile; the next K tile may be on its way
          else
            wait_copies<0>();
        });
    wait_reads();
    if (more) copy_v(t + kWaves);
  }
  // The waves' sums meet in the LDS, [HD][32 columns] each: two in the place of the K tiles, two in that of the V tiles.
  auto sums = [&](int v) { return reinterpret_cast<float*>(v < 2 ? kbuf : vbuf) + (v & 1) * HD * 32; };
  __shared__ float ml[kWaves][3][32];
  __shared__ uint32_t again;
  const float2 lp = half_pair(w.l), rp = half_pair(w.lr);
  if (threadIdx.x == 0) again = 0;
  if (h == 0) {
    ml[wave][0][col] = w.m;
    ml[wave][1][col] = lp.x + lp.y;
    ml[wave][2][col] = rp.x + rp.y;
  }
  __syncthreads();  // every wave is done with its tiles
  float M = -INFINITY;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) M = fmaxf(M, ml[v][0][col]);
  const float ref = M == -INFINITY ? 0.0f : M;
  float l = 0.0f, lr = 0.0f;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    const float f = exp2_raw(ml[v][0][col] - ref);
    l += ml[v][1][col] * f;
    lr += ml[v][2][col] * f;
  }
  const float mine = exp2_raw(w.m - ref);
  float* own = sums(wave);
#pragma unroll
  for (int d = 0; d < L::kDims; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) own[(32 * d + acc_row(e, h)) * 32 + col] = w.o[d][e] * mine;
  __syncthreads();
  // Thread: 8 head dims of a column; the waves' sums in wave order.
  constexpr int N = 8;
  const bool direct = a.splits == 1;
  for (int x = threadIdx.x; x < 32 * (HD / N); x += 64 * kWaves) {
    const int c = x & 31, d0 = (x >> 5) * N;
    if (c >= nq * grp) continue;
    const int64_t t = r.qa + i0 + c / grp, hd = g * grp + c % grp;
    float o[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      o[e] = 0.0f;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) o[e] += sums(v)[(d0 + e) * 32 + c];
    }
    if (direct) {
      // sums of the column: every thread of it forms them again
      float mc = -INFINITY, rc = 0.0f;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) mc = fmaxf(mc, ml[v][0][c]);
      mc = mc == -INFINITY ? 0.0f : mc;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) rc += ml[v][2][c] * exp2_raw(ml[v][0][c] - mc);
      const bool any = r.vis(i0 + c / grp, a.causal) > 0;
      const float f = any ? 1.0f / rc : 0.0f;
      bool fine = true;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        o[e] = any ? o[e] * f : 0.0f;
        fine = fine && fabsf(o[e]) <= 3.402823466e38f;
      }
      if (!fine) atomicOr(&again, 1u << c);
      store_from_f32<T, N>(static_cast<T*>(a.out) + (t * a.h_q + hd) * HD + d0, o);
    } else {
      store_pack<float, N>(a.part + ((static_cast<int64_t>(z) * a.n_q + t) * a.h_q + hd) * (HD + 4) + d0,
                           __builtin_bit_cast(Pack<float, N>, o));
    }
  }
  if (wave == 0 && h == 0 && valid) {
    const int64_t t = r.qa + i;
    if (direct) {
      a.lse[head * a.n_q + t] = vis > 0 ? (M + log2f(l)) * kLn2 : -INFINITY;
    } else {
      float* p = a.part + ((static_cast<int64_t>(z) * a.n_q + t) * a.h_q + head) * (HD + 4) + HD;
      p[0] = M;
      p[1] = l;
      p[2] = lr;
    }
  }
  if (!direct) return;
  stage_wait();  // the stores above come before those below
  __syncthreads();
  uint32_t cols = again;
  for (; cols; cols &= cols - 1) {  // (uniform over the block; the waves take columns in turn)
    const int c = __builtin_ctz(cols);
    if (c % kWaves == wave) plain_fwd_row<T, HD, CAP, BIAS>(a, r, i0 + c / grp, g * grp + c % grp);
  }
}

template <typename T, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * kWaves)
__attribute__((amdgpu_waves_per_eu(kCuBlocks<HD>, kCuBlocks<HD>))) void masked_split_kernel(
    MaskedArgs a) {
  __shared__ __attribute__((aligned(16))) char kbuf[kWaves * Tiles<HD>::kBytes];
  __shared__ __attribute__((aligned(16))) char vbuf[kWaves * Tiles<HD>::kBytes];
  split_block<T, HD, CAP, BIAS>(a, kbuf, vbuf);
}

// Joins the parts of one (query, head), a block each: its waves take the parts in turn, eight loads at a time, and add
// their sums in wave order. What it costs is the loads' latency: 8 tokens of 12 heads, up to 32 parts 4.2 us, one token,
// 256 parts 7.6 us.
template <typename T, int HD, bool CAP, bool BIAS, int kJoinWaves>
__global__ __launch_bounds__(64 * kJoinWaves) void masked_join_kernel(MaskedArgs a) {
  constexpr int N = HD / 64, kDepth = 8;
  __shared__ float acc[kJoinWaves][HD], ms[kJoinWaves], ls[kJoinWaves], rs[kJoinWaves];
  const int64_t x = blockIdx.x;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, head = static_cast<int>(x % a.h_q);
  const int64_t t = x / a.h_q;
  const int tpb = split_tokens(a.h_q / a.h_kv);
  const int s = row_of(a, static_cast<int>(t));
  const MaskedRow r = as_queries(masked_row(a, s), s, a.n_seq);
  const int i = static_cast<int>(t) - r.qa, i0 = i / tpb * tpb;
  const int vis = r.vis(i, a.causal);
  // The parts that the query's block wrote.
  const int tiles = (r.vis(min(i0 + tpb, r.lq) - 1, a.causal) + 31) / 32;
  const int n = max(1, min(a.splits, (tiles + a.split_tiles - 1) / a.split_tiles));
  const int64_t step = a.n_q * a.h_q * (HD + 4);
  const float* p = a.part + x * (HD + 4);
  float m = -INFINITY, l = 0.0f, lr = 0.0f, o[N] = {};
  for (int z0 = wave; z0 < n; z0 += kJoinWaves * kDepth) {
    float pm[kDepth], pl[kDepth], pr[kDepth], y[kDepth][N];
#pragma unroll
    for (int e = 0; e < kDepth; ++e) {
      const float* pz = p + min(z0 + kJoinWaves * e, n - 1) * step;
      pm[e] = pz[HD];
      pl[e] = pz[HD + 1];
      pr[e] = pz[HD + 2];
      load_f32<float, N>(pz + lane * N, y[e]);
    }
    float mn = m;
#pragma unroll
    for (int e = 0; e < kDepth; ++e) {
      if (z0 + kJoinWaves * e >= n) pm[e] = -INFINITY;
      mn = fmaxf(mn, pm[e]);
    }
    const float ref = mn == -INFINITY ? 0.0f : mn, alpha = exp2_raw(m - ref);
    m = mn;
    l *= alpha;
    lr *= alpha;
#pragma unroll
    for (int d = 0; d < N; ++d) o[d] *= alpha;
#pragma unroll
    for (int e = 0; e < kDepth; ++e) {
      if (z0 + kJoinWaves * e >= n) continue;
      const float f = exp2_raw(pm[e] - ref);
      l = __builtin_fmaf(pl[e], f, l);
      lr = __builtin_fmaf(pr[e], f, lr);
#pragma unroll
      for (int d = 0; d < N; ++d) o[d] = __builtin_fmaf(y[e][d], f, o[d]);
    }
  }
#pragma unroll
  for (int d = 0; d < N; ++d) acc[wave][lane * N + d] = o[d];
  if (lane == 0) ms[wave] = m, ls[wave] = l, rs[wave] = lr;
  __syncthreads();
  if (wave > 0) return;
  m = ms[0];
#pragma unroll
  for (int v = 1; v < kJoinWaves; ++v) m = fmaxf(m, ms[v]);
  const float ref = m == -INFINITY ? 0.0f : m;
  l = lr = 0.0f;
#pragma unroll
  for (int d = 0; d < N; ++d) o[d] = 0.0f;
#pragma unroll
  for (int v = 0; v < kJoinWaves; ++v) {
    const float f = exp2_raw(ms[v] - ref);
    l = __builtin_fmaf(ls[v], f, l);
    lr = __builtin_fmaf(rs[v], f, lr);
#pragma unroll
    for (int d = 0; d < N; ++d) o[d] = __builtin_fmaf(acc[v][lane * N + d], f, o[d]);
  }
  const float f = 1.0f / lr;
  bool fine = true;
#pragma unroll
  for (int d = 0; d < N; ++d) {
    o[d] = vis > 0 ? o[d] * f : 0.0f;
    fine = fine && fabsf(o[d]) <= 3.402823466e38f;
  }
  if (__ballot(!fine)) {
    plain_fwd_row<T, HD, CAP, BIAS>(a, r, i, head);
    return;
  }
  store_from_f32<T, N>(static_cast<T*>(a.out) + x * HD + lane * N, o);
  if (lane == 0) a.lse[head * a.n_q + t] = vis > 0 ? (m + log2f(l)) * kLn2 : -INFINITY;
}

// ---------------------------------------------------------------------------------------------
// Backward. P and dS are rounded to T for the products that take them; their sums, D and lse are not. In blocks of 128
// gradients are off the definition by 1.4 times what their own rounding is (bf16 0.24% against 0.17%, fp16 0.030% against
// 0.021%), which the products at twice the instructions would not be worth; blocks of 32, with instructions to spare, give
// what these roundings left to the products too, and their gradients are off by their own rounding alone. fp16 loses bits
// of P and dS below 2^-14: gradients far below 1 want a scaled loss there.
// ---------------------------------------------------------------------------------------------

// LDS of the backward: the streamed tiles' two buffers, and for the dK / dV blocks the block's V rows and the streamed
// queries' lse and D.
struct BwdLds {
  char* buf0;
  char* buf1;
  char* v;
  float* ld0;  // lse (log2 units) of 32 queries, then D
  float* ld1;
};

// A 32 x 32 tile, a lane owning a query: st holds the products, dp dP^T; then st P (1 - t^2) and dp dS'^T, whose sum
// before the factor joins r. left: keys of the lane's query from the tile's first on that it sees, edge: whether any query
// of the wave misses one.
template <typename T, bool CAP, bool BIAS>
__device__ __forceinline__ void query_scores(const MaskedArgs& a, float slope2, f32x16 (&st)[1], f32x16& dp, float dsum,
                                             float lse2, float d0, bool edge, int left, int h, float& r) {
  f32x16 f[1];
  if constexpr (CAP) capped_scores<BIAS, 1, true>(a, slope2, st, f, d0, 1.0f);
#pragma unroll
  for (int e = 0; e < 16; ++e)
    st[0][e] = exp2_raw(CAP ? st[0][e] - lse2 : __builtin_fmaf(st[0][e], a.sl2, -lse2));
#pragma unroll
  for (int e = 0; e < 16; ++e) dp[e] = st[0][e] * (dp[e] - dsum);
  if (edge) {
    const int most = left - 4 * h;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const bool in = acc_row(e, 0) < most;
      st[0][e] = in ? st[0][e] : 0.0f;
      dp[e] = in ? dp[e] : 0.0f;
      if constexpr (CAP) f[0][e] = in ? f[0][e] : 0.0f;
    }
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) r += dp[e];
  if constexpr (CAP) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      dp[e] *= f[0][e];
      st[0][e] *= f[0][e];
    }
  }
}

// P in st and dS in dp of a 32 x 32 tile, a lane owning a key; stats(q, lse, D): those of the queries 8 q + 4 h .. + 4
// (lse in log2 units). edge: whether a query of the tile (below `first`: those that miss the lane's key; from `rows` on:
// none) stays out.
template <typename T, bool CAP, bool BIAS, typename F>
__device__ __forceinline__ void key_scores(const MaskedArgs& a, float slope2, f32x16 (&st)[1], f32x16 (&f)[1], f32x16& dp,
                                           F stats, float d0, bool edge, int first, int rows, int h) {
  if constexpr (CAP) capped_scores<BIAS, 1, true>(a, slope2, st, f, d0, -1.0f);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    f32x4 lv, dd;
    stats(q, lv, dd);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = 4 * q + i;
      const float p = exp2_raw(CAP ? st[0][e] - lv[i] : __builtin_fmaf(st[0][e], a.sl2, -lv[i]));
      st[0][e] = p;
      dp[e] = p * (dp[e] - dd[i]);
      if constexpr (CAP) dp[e] *= f[0][e];
    }
  }
  if (edge) {
    const int least = first - 4 * h, most = rows - 4 * h;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const bool in = acc_row(e, 0) >= least && acc_row(e, 0) < most;
      st[0][e] = in ? st[0][e] : 0.0f;
      dp[e] = in ? dp[e] : 0.0f;
    }
  }
}

// dQ and D of 128 queries: key tiles stream through LDS, each wave owns 32 queries (Q fragments in registers, its dO
// tile in LDS: the two sums leave no registers for it, and with it they went to scratch memory). Bound by the four
// products and the exponentials between them: 4,096 + 2,048 + 1,024 + 993 tokens, 12 / 2 heads of 128, bf16 with a bias
// 196 us (720 TFLOP/s of what is visible).
template <typename T, int HD, bool CAP, bool BIAS>
__device__ __forceinline__ void bwd_dq(const MaskedArgs& a, int blk, int head, char* buf0, char* buf1, char* dot) {
  using L = Tiles<HD>;
  int s, b, nb;
  if (!find_span_block(a.cu_q, a.n_seq, static_cast<int>(a.n_q), blk, kRows, s, b, nb)) return;
  const MaskedRow r = uniform(as_queries(masked_row(a, s), s, a.n_seq));
  b = uniform(nb - 1 - b);
  const int g = head / (a.h_q / a.h_kv);
  const int wave = uniform(static_cast<int>(threadIdx.x) >> 6);
  const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
  const int i0 = b * kRows, iw = i0 + 32 * wave, i = min(iw + col, r.lq - 1);
  const bool valid = iw + col < r.lq;
  const int vis = r.vis(i, a.causal);
  const int tiles = (r.vis(min(i0 + kRows, r.lq) - 1, a.causal) + 31) / 32;
  const int vis_all = iw < r.lq ? r.vis(iw, a.causal) : 0;
  const int mine = iw < r.lq ? (r.vis(min(iw + 31, r.lq - 1), a.causal) + 31) / 32 : 0;
  const T* kh = token<T>(a.k, r.ka, a.k_st, g, a.k_sh);
  const T* vh = token<T>(a.v, r.ka, a.v_st, g, a.v_sh);
  constexpr int C = L::kCopies / kWaves;
  const TileLane<HD, C> tk(C * wave, lane, a.k_st), tv(C * wave, lane, a.v_st);
  const FragLane<HD> fl0(lane);
  const Scorer<CAP, BIAS> sc(a, head);
  auto copy = [&](char* dst, int j) {
    const int rows = r.lk - 32 * j;
    tk.copy(dst, kh + 32 * j * a.k_st, rows);
    tv.copy(dst + L::kBytes, vh + 32 * j * a.v_st, rows);
  };
  if (tiles) copy(buf0, 0);
  const int64_t t = r.qa + i;
  char* dt = dot + wave * L::kBytes;
  if (iw < r.lq)
    TileLane<HD, L::kCopies>(0, lane, a.do_st)
        .copy(dt, token<T>(a.dout, static_cast<int64_t>(r.qa) + iw, a.do_st, head, a.do_sh), r.lq - iw);
  Frag qf[L::kSteps];
  load_row_frags<T, HD>(qf, token<T>(a.q, t, a.q_st, head, a.q_sh), h);
  float ds = 0.0f;
  {
    Frag df[L::kSteps], of[L::kSteps];
    load_row_frags<T, HD>(df, token<T>(a.dout, t, a.do_st, head, a.do_sh), h);
    load_row_frags<T, HD>(of, static_cast<const T*>(a.o) + (t * a.h_q + head) * HD, h);
#pragma unroll
    for (int k = 0; k < L::kSteps; ++k) ds = dot8<T>(of[k], df[k], ds);
  }
  const float2 dp2 = half_pair(ds);
  const float dsum = dp2.x + dp2.y;
  const float lse2 = a.lse[head * a.n_q + t] * kLog2e;
  f32x16 dq[L::kDims], pk[L::kDims];  // sum dS' K, sum P (1 - t^2) K
  float rest = 0.0f;
#pragma unroll
  for (int d = 0; d < L::kDims; ++d) {
    dq[d] = f32x16{};
    pk[d] = f32x16{};
  }
  stage_barrier();
  auto stage = [&](const char* kt, char* next, int j) {
    if (j + 1 < tiles) copy(next, j + 1);
    const char* vt = kt + L::kBytes;
    const FragLane<HD> fl = fl0.fresh();
    if (j < mine) {
      f32x16 st[1], dp = f32x16{};
      start_scores<CAP, BIAS, 1>(st, sc.slope, static_cast<float>(r.off() + i - 32 * j - 4 * h), 1.0f,
                                 32 * j + 31 <= r.off() + iw);
#pragma unroll
      for (int k = 0; k < L::kSteps; ++k) {
        st[0] = mfma<T>(fl.frag(kt, k), qf[k], st[0]);  // S^T = K Q^T
        dp = mfma<T>(fl.frag(vt, k), fl.frag(dt, k), dp);  // dP^T = V dO^T
      }
      query_scores<T, CAP, BIAS>(a, sc.slope2, st, dp, dsum, lse2, static_cast<float>(r.off() + i - 32 * j - 4 * h),
                                 32 * j + 32 > vis_all, vis - 32 * j, h, rest);
      const Frag p0 = frag_acc<T>(st[0], 0), p1 = frag_acc<T>(st[0], 1);
      const Frag s0 = frag_acc<T>(dp, 0), s1 = frag_acc<T>(dp, 1);
#pragma unroll
      for (int d = 0; d < L::kDims; ++d) {
        const Frag k0 = fl.frag_t(kt, 0, d), k1 = fl.frag_t(kt, 1, d);
        dq[d] = mfma<T>(k0, s0, dq[d]);  // dQ^T += K^T dS'^T
        pk[d] = mfma<T>(k0, p0, pk[d]);
        dq[d] = mfma<T>(k1, s1, dq[d]);
        pk[d] = mfma<T>(k1, p1, pk[d]);
      }
    }
    stage_barrier();
  };
  for (int j = 0; j < tiles; j += 2) {
    stage(buf0, buf1, j);
    if (j + 1 < tiles) stage(buf1, buf0, j + 1);
  }
  if (iw >= r.lq) return;
  const float2 rp = half_pair(rest);
  rest = rp.x + rp.y;
#pragma unroll
  for (int d = 0; d < L::kDims; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) dq[d][e] = __builtin_fmaf(-rest, pk[d][e], dq[d][e]);
  const uint64_t again = __ballot(valid && !(all_finite(dq, a.scale) && fabsf(rest) <= 3.402823466e38f));
  uint32_t cols = static_cast<uint32_t>(again) | static_cast<uint32_t>(again >> 32);
  const bool keep = valid && !((cols >> col) & 1);
  // (a single key's P is 1 whatever its score: its dQ is 0, not what the roundings leave)
  store_row<T, L::kDims>(static_cast<T*>(a.out) + (t * a.h_q + head) * HD, dq, vis > 1 ? a.scale : 0.0f, h, keep);
  if (h == 0 && keep) a.dsum[head * a.n_q + t] = vis > 0 ? dsum + rest : 0.0f;
  for (; cols; cols &= cols - 1) plain_dq_row<T, HD, CAP, BIAS>(a, r, iw + __builtin_ctz(cols), head);
}

// dK and dV of 128 keys for one query head: Q and dO tiles stream through LDS with their lse and D, each wave owns 32
// keys (K fragments in registers, V fragments from LDS). A lane owns one key (column of S = Q K^T) and half of the
// queries. Bound as dQ, with two products' operands read from LDS by columns: the same tokens 249 us (570 TFLOP/s).
template <typename T, int HD, bool CAP, bool BIAS>
__device__ __forceinline__ void bwd_dkdv(const MaskedArgs& a, int blk, int head, const BwdLds& lds) {
  using L = Tiles<HD>;
  int s, b, nb;
  if (!find_span_block(a.cu_k, a.n_seq, static_cast<int>(a.n_k), blk, kRows, s, b, nb)) return;
  const MaskedRow r = uniform(as_keys(masked_row(a, s), s, a.n_seq));
  b = uniform(b);
  const int grp = a.h_q / a.h_kv, g = head / grp;
  const int tid = threadIdx.x, wave = uniform(tid >> 6);
  const int lane = tid & 63, h = lane >> 5, col = lane & 31;
  const int k0 = b * kRows, kw = k0 + 32 * wave, kj = kw + col, kc = min(kj, r.lk - 1);
  // The block's query tiles run from the first query that sees its first key; a wave's from its own first.
  const int t0 = r.first(k0, a.causal) / 32, tiles = (r.lq + 31) / 32;
  const int q_lane = r.first(kc, a.causal);                         // the lane's first query
  const int q_wave = kw < r.lk ? r.first(kw, a.causal) / 32 : tiles;  // the wave's first tile
  const int q_all = r.first(min(kw + 31, r.lk - 1), a.causal);      // from here on every key of the wave is seen
  const T* qh = token<T>(a.q, r.qa, a.q_st, head, a.q_sh);
  const T* doh = token<T>(a.dout, r.qa, a.do_st, head, a.do_sh);
  const float* lse = a.lse + head * a.n_q + r.qa;
  const float* dsum = a.dsum + head * a.n_q + r.qa;
  constexpr int C = L::kCopies / kWaves;
  const TileLane<HD, C> tq(C * wave, lane, a.q_st), td(C * wave, lane, a.do_st);
  const FragLane<HD> fl0(lane);
  const Scorer<CAP, BIAS> sc(a, head);
  float stat = 0.0f;  // of threads 0 to 31 a query's lse (log2 units), of 32 to 63 its D
  auto copy = [&](char* dst, int j) {
    const int rows = r.lq - 32 * j;
    tq.copy(dst, qh + 32 * j * a.q_st, rows);
    td.copy(dst + L::kBytes, doh + 32 * j * a.do_st, rows);
    if (wave == 0) stat = h == 0 ? lse[32 * j + min(col, rows - 1)] * kLog2e : dsum[32 * j + min(col, rows - 1)];
  };
  auto finish = [&](float* ld) {
    if (wave == 0) ld[lane] = stat;
  };
  if (t0 < tiles) copy(lds.buf0, t0);
  {
    const TileLane<HD, C> tv(C * wave, lane, a.v_st);
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (k0 + 32 * n < r.lk)
        tv.copy(lds.v + n * L::kBytes, token<T>(a.v, static_cast<int64_t>(r.ka) + k0 + 32 * n, a.v_st, g, a.v_sh),
                r.lk - k0 - 32 * n);
  }
  Frag kf[L::kSteps];
  load_row_frags<T, HD>(kf, token<T>(a.k, static_cast<int64_t>(r.ka) + kc, a.k_st, g, a.k_sh), h);
  f32x16 dk[L::kDims], dv[L::kDims];
#pragma unroll
  for (int d = 0; d < L::kDims; ++d) {
    dk[d] = f32x16{};
    dv[d] = f32x16{};
  }
  if (t0 < tiles) finish(lds.ld0);
  stage_barrier();
  const char* vt = lds.v + wave * L::kBytes;
  auto stage = [&](const char* qt, const float* ld, char* next, float* ldn, int j) {
    if (j + 1 < tiles) copy(next, j + 1);
    const char* dt = qt + L::kBytes;
    const FragLane<HD> fl = fl0.fresh();
    if (j >= q_wave) {
      f32x16 st[1], dp = f32x16{}, f[1];
      start_scores<CAP, BIAS, 1>(st, sc.slope, static_cast<float>(r.off() + 32 * j + 4 * h - kc), -1.0f,
                                 r.off() + 32 * j >= kw + 31);
#pragma unroll
      for (int k = 0; k < L::kSteps; ++k) {
        st[0] = mfma<T>(fl.frag(qt, k), kf[k], st[0]);      // S = Q K^T
        dp = mfma<T>(fl.frag(dt, k), fl.frag(vt, k), dp);   // dP = dO V^T
      }
      key_scores<T, CAP, BIAS>(
          a, sc.slope2, st, f, dp,
          [&](int q, f32x4& lv, f32x4& dd) {
            lv = *reinterpret_cast<const f32x4*>(ld + 8 * q + 4 * h);
            dd = *reinterpret_cast<const f32x4*>(ld + 32 + 8 * q + 4 * h);
          },
          static_cast<float>(r.off() + 32 * j + 4 * h - kc), 32 * j < q_all || 32 * j + 32 > r.lq, q_lane - 32 * j,
          r.lq - 32 * j, h);
      const Frag p0 = frag_acc<T>(st[0], 0), p1 = frag_acc<T>(st[0], 1);
      const Frag s0 = frag_acc<T>(dp, 0), s1 = frag_acc<T>(dp, 1);
#pragma unroll
      for (int d = 0; d < L::kDims; ++d) {
        dv[d] = mfma<T>(p0, fl.frag_t(dt, 0, d), dv[d]);  // dV += P^T dO
        dv[d] = mfma<T>(p1, fl.frag_t(dt, 1, d), dv[d]);
        dk[d] = mfma<T>(s0, fl.frag_t(qt, 0, d), dk[d]);  // dK += dS^T Q
        dk[d] = mfma<T>(s1, fl.frag_t(qt, 1, d), dk[d]);
      }
    }
    if (j + 1 < tiles) finish(ldn);
    stage_barrier();
  };
  for (int j = t0; j < tiles; j += 2) {
    stage(lds.buf0, lds.ld0, lds.buf1, lds.ld1, j);
    if (j + 1 < tiles) stage(lds.buf1, lds.ld1, lds.buf0, lds.ld0, j + 1);
  }
  if (kw >= r.lk) return;
  // Keys are accumulator rows, head dims lanes. A key with a sum that is not finite is formed again by itself.
  uint32_t bad = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    bool fine = true;
#pragma unroll
    for (int d = 0; d < L::kDims; ++d)
      fine = fine && fabsf(dk[d][e] * a.scale) <= 3.402823466e38f && fabsf(dv[d][e]) <= 3.402823466e38f;
    const uint64_t no = __ballot(!fine);
    if (no & 0xffffffffu) bad |= 1u << acc_row(e, 0);
    if (no >> 32) bad |= 1u << acc_row(e, 1);
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int row = acc_row(e, h), key = kw + row;
    if (key >= r.lk || ((bad >> row) & 1)) continue;
#pragma unroll
    for (int d = 0; d < L::kDims; ++d) {
      const int64_t t = r.ka + key;
      if (grp > 1) {  // this head's part, past the L2: other blocks' parts join it in the next launch
        const int64_t o = (head * a.n_k + t) * HD + 32 * d + col;
        store_partial(a.dk_part + o, dk[d][e] * a.scale);
        store_partial(a.dv_part + o, dv[d][e]);
      } else {
        const int64_t o = (t * a.h_kv + g) * HD + 32 * d + col;
        static_cast<T*>(a.dk)[o] = from_f32<T>(dk[d][e] * a.scale);
        static_cast<T*>(a.dv)[o] = from_f32<T>(dv[d][e]);
      }
    }
  }
  for (; bad; bad &= bad - 1) {
    const int key = kw + __builtin_ctz(bad);
    if (key >= r.lk) break;
    const int64_t o = (head * a.n_k + r.ka + key) * HD;
    plain_dkv_row<T, HD, CAP, BIAS>(a, r, key, head, head + 1, grp > 1 ? a.dk_part + o : nullptr,
                                    grp > 1 ? a.dv_part + o : nullptr);
  }
}

template <typename T, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * kWaves)
__attribute__((amdgpu_waves_per_eu(kCuBlocks<HD>, kCuBlocks<HD>))) void masked_dq_kernel(MaskedArgs a) {
  __shared__ __attribute__((aligned(16))) char buf0[2 * Tiles<HD>::kBytes];
  __shared__ __attribute__((aligned(16))) char buf1[2 * Tiles<HD>::kBytes];
  __shared__ __attribute__((aligned(16))) char dot[kWaves * Tiles<HD>::kBytes];
  int item, head;
  if (!head_item(a, a.n_blocks, item, head)) return;
  bwd_dq<T, HD, CAP, BIAS>(a, item, head, buf0, buf1, dot);
}

template <typename T, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * kWaves)
__attribute__((amdgpu_waves_per_eu(kCuBlocks<HD>, kCuBlocks<HD>))) void masked_dkdv_kernel(
    MaskedArgs a) {
  using L = Tiles<HD>;
  __shared__ __attribute__((aligned(16))) char buf0[2 * L::kBytes];
  __shared__ __attribute__((aligned(16))) char buf1[2 * L::kBytes];
  __shared__ __attribute__((aligned(16))) char v[4 * L::kBytes];
  __shared__ __attribute__((aligned(16))) float ld0[64];
  __shared__ __attribute__((aligned(16))) float ld1[64];
  int item, head;
  if (!head_item(a, a.n_kblocks, item, head)) return;
  bwd_dkdv<T, HD, CAP, BIAS>(a, item, head, BwdLds{buf0, buf1, v, ld0, ld1});
}

// ---------------------------------------------------------------------------------------------
// The backward of batches that leave the chip idle in blocks of 128: a block owns 32 tokens of one side, its four waves
// take the other side's tiles in turn (each with LDS of its own) and their sums meet in the LDS in wave order. Bound by
// the latency of a wave's few tiles (the remainders' products cost 707 tokens 4%, 4,096 16%): 707 tokens in six rows,
// 12 / 2 heads of 128 with a cap 21 us dQ, 20 us dK and dV; 1,923 tokens in four, 16 heads of 64 with a cap 46 and 50 us
// (the cap's arithmetic: 24,560 tiles of some 2,000 cycles over 1,024 SIMDs are 20 us each).
// ---------------------------------------------------------------------------------------------
// Of the dQ blocks: two tiles a wave (then the sums), a word and the waves' parts of r, the dO tile.
template <int HD>
constexpr int kNarrowDo = 2 * kWaves * Tiles<HD>::kBytes + 16 + 32 * kWaves * 4;
template <int HD>
constexpr int kNarrowLds = (2 + 2 * kWaves) * Tiles<HD>::kBytes;  // two shared tiles, two a wave; then the sums

// The waves' sums of one set of accumulators: every wave's tiles into LDS (lane-contiguous), then each wave adds 4 ND of
// the 16 ND registers over the waves, in wave order: register wave * 4 ND + x.
template <int ND>
__device__ __forceinline__ void merge_waves(float* buf, const f32x16 (&acc)[ND], int wave, int lane, float (&x)[4 * ND]) {
  __syncthreads();
  if (threadIdx.x == 0) reinterpret_cast<uint32_t*>(buf)[kWaves * 64 * 16 * ND] = 0;  // the rows to form again
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) buf[(wave * 16 * ND + 16 * d + e) * 64 + lane] = acc[d][e];
  __syncthreads();
#pragma unroll
  for (int y = 0; y < 4 * ND; ++y) {
    x[y] = 0.0f;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) x[y] += buf[(v * 16 * ND + wave * 4 * ND + y) * 64 + lane];
  }
}

template <typename T, int HD, bool CAP, bool BIAS>
__device__ __forceinline__ void narrow_dq(const MaskedArgs& a, int blk, int head, char* smem) {
  uint32_t* again = reinterpret_cast<uint32_t*>(smem + kWaves * 64 * 16 * (HD / 32) * 4);  // behind the waves' sums
  using L = Tiles<HD>;
  constexpr int ND = L::kDims;
  int s, b, nb;
  if (!find_span_block(a.cu_q, a.n_seq, static_cast<int>(a.n_q), blk, 32, s, b, nb)) return;
  const MaskedRow r = uniform(as_queries(masked_row(a, s), s, a.n_seq));
  b = uniform(nb - 1 - b);
  const int g = head / (a.h_q / a.h_kv);
  const int wave = uniform(static_cast<int>(threadIdx.x) >> 6);
  const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
  const int i0 = 32 * b, i = min(i0 + col, r.lq - 1);
  const bool valid = i0 + col < r.lq;
  const int vis = r.vis(i, a.causal), vis_all = r.vis(i0, a.causal);
  const int tiles = (r.vis(min(i0 + 31, r.lq - 1), a.causal) + 31) / 32;
  const T* kh = token<T>(a.k, r.ka, a.k_st, g, a.k_sh);
  const T* vh = token<T>(a.v, r.ka, a.v_st, g, a.v_sh);
  const TileLane<HD, L::kCopies> tk(0, lane, a.k_st), tv(0, lane, a.v_st);
  const FragLane<HD> fl(lane);
  const Scorer<CAP, BIAS> sc(a, head);
  char* kt = smem + 2 * wave * L::kBytes;
  char* vt = kt + L::kBytes;
  auto copy = [&](int j) {
    tk.fresh().copy(kt, kh + 32 * j * a.k_st, r.lk - 32 * j);
    tv.fresh().copy(vt, vh + 32 * j * a.v_st, r.lk - 32 * j);
  };
  if (wave < tiles) copy(wave);
  const int64_t t = r.qa + i;
  char* dt = smem + kNarrowDo<HD>;  // the block's dO tile
  constexpr int C = L::kCopies / kWaves;
  TileLane<HD, C>(C * wave, lane, a.do_st)
      .copy(dt, token<T>(a.dout, static_cast<int64_t>(r.qa) + i0, a.do_st, head, a.do_sh), r.lq - i0);
  Frag qf[L::kSteps];
  load_row_frags<T, HD>(qf, token<T>(a.q, t, a.q_st, head, a.q_sh), h);
  float ds = 0.0f;
  {
    Frag df[L::kSteps], of[L::kSteps];
    load_row_frags<T, HD>(df, token<T>(a.dout, t, a.do_st, head, a.do_sh), h);
    load_row_frags<T, HD>(of, static_cast<const T*>(a.o) + (t * a.h_q + head) * HD, h);
#pragma unroll
    for (int k = 0; k < L::kSteps; ++k) ds = dot8<T>(of[k], df[k], ds);
  }
  const float2 dp2 = half_pair(ds);
  const float dsum = dp2.x + dp2.y;
  const float lse2 = a.lse[head * a.n_q + t] * kLog2e;
  f32x16 dq[ND], pk[ND];  // sum dS' K, sum P (1 - t^2) K
  float rest = 0.0f;
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    dq[d] = f32x16{};
    pk[d] = f32x16{};
  }
  stage_barrier();  // every wave's share of the dO tile has landed
  for (int j = wave; j < tiles; j += kWaves) {
    f32x16 st[1], dp = f32x16{};
    start_scores<CAP, BIAS, 1>(st, sc.slope, static_cast<float>(r.off() + i - 32 * j - 4 * h), 1.0f, 32 * j + 31 <= r.off() + i0);
#pragma unroll
    for (int k = 0; k < L::kSteps; ++k) {
      st[0] = mfma<T>(fl.frag(kt, k), qf[k], st[0]);  // S^T = K Q^T
      dp = mfma<T>(fl.frag(vt, k), fl.frag(dt, k), dp);  // dP^T = V dO^T
    }
    query_scores<T, CAP, BIAS>(a, sc.slope2, st, dp, dsum, lse2, static_cast<float>(r.off() + i - 32 * j - 4 * h),
                               32 * j + 32 > vis_all, vis - 32 * j, h, rest);
    const Frag p0 = frag_acc<T>(st[0], 0), p1 = frag_acc<T>(st[0], 1);
    const Frag s0 = split_acc<T>(dp, 0), s1 = split_acc<T>(dp, 1);
    const Frag e0 = frag_acc<T>(dp, 0), e1 = frag_acc<T>(dp, 1);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const Frag k0 = fl.frag_t(kt, 0, d), k1 = fl.frag_t(kt, 1, d);
      dq[d] = mfma<T>(k0, s0, dq[d]);  // dQ^T += K^T dS'^T
      pk[d] = mfma<T>(k0, p0, pk[d]);
      dq[d] = mfma<T>(k0, e0, dq[d]);
      pk[d] = mfma<T>(k1, p1, pk[d]);
      dq[d] = mfma<T>(k1, s1, dq[d]);
      dq[d] = mfma<T>(k1, e1, dq[d]);
    }
    if (j + kWaves < tiles) {
      wait_reads();
      copy(j + kWaves);
      wait_copies<0>();
    }
  }
  float* parts = reinterpret_cast<float*>(again + 4);  // the waves' parts of r
  const float2 rp = half_pair(rest);
  if (h == 0) parts[32 * wave + col] = rp.x + rp.y;
  __syncthreads();
  rest = 0.0f;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) rest += parts[32 * v + col];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) dq[d][e] = __builtin_fmaf(-rest, pk[d][e], dq[d][e]);
  float x[4 * ND];
  merge_waves<ND>(reinterpret_cast<float*>(smem), dq, wave, lane, x);
  bool fine = fabsf(rest) <= 3.402823466e38f;
#pragma unroll
  for (int e = 0; e < 4 * ND; ++e) {
    x[e] *= a.scale;
    fine = fine && fabsf(x[e]) <= 3.402823466e38f;
  }
  if (valid && !fine) atomicOr(again, 1u << col);
  __syncthreads();
  uint32_t cols = *again;
  if (valid && !((cols >> col) & 1)) {
    if (wave == 0 && h == 0) a.dsum[head * a.n_q + t] = vis > 0 ? dsum + rest : 0.0f;
    T* row = static_cast<T*>(a.out) + (t * a.h_q + head) * HD;
#pragma unroll
    for (int q = 0; q < ND; ++q) {  // four registers: head dims 32 d + 8 (e / 4) + 4 h .. + 4
      const int e = wave * 4 * ND + 4 * q;
      float o[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) o[y] = vis > 1 ? x[4 * q + y] : 0.0f;  // (a single key's P is 1: its dQ is 0)
      store_from_f32<T, 4>(row + 32 * (e >> 4) + acc_row(e & 15, h), o);
    }
  }
  for (; cols; cols &= cols - 1)
    if (__builtin_ctz(cols) % kWaves == wave) plain_dq_row<T, HD, CAP, BIAS>(a, r, i0 + __builtin_ctz(cols), head);
}

template <typename T, int HD, bool CAP, bool BIAS>
__device__ __forceinline__ void narrow_dkdv(const MaskedArgs& a, int blk, int head, char* smem) {
  // (the word behind the waves' sums: the tiles leave no other room for two blocks a CU)
  uint32_t* again = reinterpret_cast<uint32_t*>(smem + kWaves * 64 * 16 * (HD / 32) * 4);
  using L = Tiles<HD>;
  constexpr int ND = L::kDims;
  int s, b, nb;
  if (!find_span_block(a.cu_k, a.n_seq, static_cast<int>(a.n_k), blk, 32, s, b, nb)) return;
  const MaskedRow r = uniform(as_keys(masked_row(a, s), s, a.n_seq));
  const int grp = a.h_q / a.h_kv, g = head / grp;
  const int wave = uniform(static_cast<int>(threadIdx.x) >> 6);
  const int lane = threadIdx.x & 63, h = lane >> 5, col = lane & 31;
  const int k0 = 32 * uniform(b), kc = min(k0 + col, r.lk - 1);
  const int t0 = r.first(k0, a.causal) / 32, tiles = (r.lq + 31) / 32;
  const int q_lane = r.first(kc, a.causal);                     // the lane's first query
  const int q_all = r.first(min(k0 + 31, r.lk - 1), a.causal);  // from here on every key is seen
  const T* qh = token<T>(a.q, r.qa, a.q_st, head, a.q_sh);
  const T* doh = token<T>(a.dout, r.qa, a.do_st, head, a.do_sh);
  const float* lse = a.lse + head * a.n_q + r.qa;
  const float* ds = a.dsum + head * a.n_q + r.qa;
  const TileLane<HD, L::kCopies> tq(0, lane, a.q_st), td(0, lane, a.do_st);
  const FragLane<HD> fl(lane);
  const Scorer<CAP, BIAS> sc(a, head);
  char* kt = smem;
  char* vt = smem + L::kBytes;
  char* qt = smem + (2 + 2 * wave) * L::kBytes;
  char* dt = qt + L::kBytes;
  // lse (log2 units) of tile row c in lane c, D in lane c + 32. Heads of 64 leave LDS to spread them from; with 128 the
  // tiles fill what two blocks a CU have, and lanes ask each other.
  float* ld = reinterpret_cast<float*>(smem + kNarrowLds<HD>) + 64 * wave;
  const float* stat_row = h ? ds : lse;
  float stat = 0.0f;
  auto copy = [&](int j) {
    const int rows = r.lq - 32 * j;
    tq.fresh().copy(qt, qh + 32 * j * a.q_st, rows);
    td.fresh().copy(dt, doh + 32 * j * a.do_st, rows);
    stat = stat_row[32 * j + min(col, rows - 1)];
  };
  auto landed = [&] {
    stat = h ? stat : stat * kLog2e;
    if constexpr (HD == 64) ld[lane] = stat;
  };
  constexpr int C = L::kCopies / kWaves;
  TileLane<HD, C>(C * wave, lane, a.k_st)
      .copy(kt, token<T>(a.k, static_cast<int64_t>(r.ka) + k0, a.k_st, g, a.k_sh), r.lk - k0);
  TileLane<HD, C>(C * wave, lane, a.v_st)
      .copy(vt, token<T>(a.v, static_cast<int64_t>(r.ka) + k0, a.v_st, g, a.v_sh), r.lk - k0);
  if (t0 + wave < tiles) copy(t0 + wave);
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    dk[d] = f32x16{};
    dv[d] = f32x16{};
  }
  stage_barrier();
  landed();
  for (int j = t0 + wave; j < tiles; j += kWaves) {
    f32x16 st[1], dp = f32x16{}, f[1];
    start_scores<CAP, BIAS, 1>(st, sc.slope, static_cast<float>(r.off() + 32 * j + 4 * h - kc), -1.0f,
                               r.off() + 32 * j >= k0 + 31);
#pragma unroll
    for (int k = 0; k < L::kSteps; ++k) {
      st[0] = mfma<T>(fl.frag(qt, k), fl.frag(kt, k), st[0]);  // S = Q K^T
      dp = mfma<T>(fl.frag(dt, k), fl.frag(vt, k), dp);        // dP = dO V^T
    }
    key_scores<T, CAP, BIAS>(
        a, sc.slope2, st, f, dp,
        [&](int q, f32x4& lv, f32x4& dd) {
          if constexpr (HD == 64) {
            lv = *reinterpret_cast<const f32x4*>(ld + 8 * q + 4 * h);
            dd = *reinterpret_cast<const f32x4*>(ld + 32 + 8 * q + 4 * h);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              lv[i] = __shfl(stat, 8 * q + 4 * h + i, 64);
              dd[i] = __shfl(stat, 32 + 8 * q + 4 * h + i, 64);
            }
          }
        },
        static_cast<float>(r.off() + 32 * j + 4 * h - kc), 32 * j < q_all || 32 * j + 32 > r.lq, q_lane - 32 * j,
        r.lq - 32 * j, h);
    const Frag p0 = split_acc<T>(st[0], 0), p1 = split_acc<T>(st[0], 1);
    const Frag s0 = split_acc<T>(dp, 0), s1 = split_acc<T>(dp, 1);
    const Frag c0 = frag_acc<T>(st[0], 0), c1 = frag_acc<T>(st[0], 1);
    const Frag e0 = frag_acc<T>(dp, 0), e1 = frag_acc<T>(dp, 1);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const Frag o0 = fl.frag_t(dt, 0, d), o1 = fl.frag_t(dt, 1, d);
      dv[d] = mfma<T>(p0, o0, dv[d]);  // dV += P^T dO
      dv[d] = mfma<T>(c0, o0, dv[d]);
      dv[d] = mfma<T>(p1, o1, dv[d]);
      dv[d] = mfma<T>(c1, o1, dv[d]);
      const Frag q0 = fl.frag_t(qt, 0, d), q1 = fl.frag_t(qt, 1, d);
      dk[d] = mfma<T>(s0, q0, dk[d]);  // dK += dS^T Q
      dk[d] = mfma<T>(e0, q0, dk[d]);
      dk[d] = mfma<T>(s1, q1, dk[d]);
      dk[d] = mfma<T>(e1, q1, dk[d]);
    }
    if (j + kWaves < tiles) {
      wait_reads();
      copy(j + kWaves);
      wait_copies<0>();
      landed();
    }
  }
  // Keys are accumulator rows, head dims lanes.
  float x[4 * ND], y[4 * ND];
  merge_waves<ND>(reinterpret_cast<float*>(smem), dk, wave, lane, x);
  merge_waves<ND>(reinterpret_cast<float*>(smem), dv, wave, lane, y);
#pragma unroll
  for (int e = 0; e < 4 * ND; ++e) {
    x[e] *= a.scale;
    if (!(fabsf(x[e]) <= 3.402823466e38f && fabsf(y[e]) <= 3.402823466e38f))
      atomicOr(again, 1u << acc_row((wave * 4 * ND + e) & 15, h));
  }
  __syncthreads();
  uint32_t bad = *again;
#pragma unroll
  for (int e = 0; e < 4 * ND; ++e) {
    const int reg = wave * 4 * ND + e, row = acc_row(reg & 15, h), key = k0 + row;
    if (key >= r.lk || ((bad >> row) & 1)) continue;
    const int64_t t = r.ka + key;
    const int dim = 32 * (reg >> 4) + col;
    if (grp > 1) {
      const int64_t o = (head * a.n_k + t) * HD + dim;
      store_partial(a.dk_part + o, x[e]);
      store_partial(a.dv_part + o, y[e]);
    } else {
      const int64_t o = (t * a.h_kv + g) * HD + dim;
      static_cast<T*>(a.dk)[o] = from_f32<T>(x[e]);
      static_cast<T*>(a.dv)[o] = from_f32<T>(y[e]);
    }
  }
  for (; bad; bad &= bad - 1) {
    const int key = k0 + __builtin_ctz(bad);
    if (key >= r.lk) break;
    if (__builtin_ctz(bad) % kWaves != wave) continue;
    const int64_t o = (head * a.n_k + r.ka + key) * HD;
    plain_dkv_row<T, HD, CAP, BIAS>(a, r, key, head, head + 1, grp > 1 ? a.dk_part + o : nullptr,
                                    grp > 1 ? a.dv_part + o : nullptr);
  }
}

template <typename T, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void masked_narrow_dq_kernel(
    MaskedArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[kNarrowDo<HD> + Tiles<HD>::kBytes];
  int item, head;
  if (!head_item(a, a.n_blocks, item, head)) return;
  narrow_dq<T, HD, CAP, BIAS>(a, item, head, smem);
}

template <typename T, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * kWaves)
__attribute__((amdgpu_waves_per_eu(kCuBlocks<HD>, kCuBlocks<HD>))) void masked_narrow_dkdv_kernel(
    MaskedArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[kNarrowLds<HD> + (HD == 64 ? kWaves * 64 * 4 : 0)];
  int item, head;
  if (!head_item(a, a.n_kblocks, item, head)) return;
  narrow_dkdv<T, HD, CAP, BIAS>(a, item, head, smem);
}

// dk / dv [key, g, :] = T(sum over the KV group's heads, in head order, of the parts). Thread = 4 head dims of a
// key. Bound by reading the parts: 8,161 keys of 12 heads 19 us (5.4 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void masked_group_sum_kernel(MaskedArgs a, int hd4) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int c = 4 * static_cast<int>(t % hd4), grp = a.h_q / a.h_kv, hd = 4 * hd4;
  const int g = static_cast<int>((t / hd4) % a.h_kv);
  const int64_t key = t / hd4 / a.h_kv;
  if (key >= a.n_k) return;
  const int64_t step = a.n_k * hd;
  const float* src = (blockIdx.y == 0 ? a.dk_part : a.dv_part) + g * grp * step + key * hd + c;
  f32x4 sum = *reinterpret_cast<const f32x4*>(src);
  int j = 1;
  for (; j + 4 < grp; j += 4) {  // four heads' loads in flight
    f32x4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const f32x4*>(src + (j + i) * step);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += x[i];
  }
  f32x4 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (j + i < grp) x[i] = *reinterpret_cast<const f32x4*>(src + (j + i) * step);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (j + i < grp) sum += x[i];
  float o[4] = {sum[0], sum[1], sum[2], sum[3]};
  store_from_f32<T, 4>(static_cast<T*>(blockIdx.y == 0 ? a.dk : a.dv) + (key * a.h_kv + g) * hd + c, o);
}

// Calls f<T, HD, CAP, BIAS>() for the call's types.
template <typename F>
void dispatch(int dtype, int hd, bool cap, bool bias, F f) {
  auto by_bias = [&](auto t, auto d, auto c) {
    if (bias)
      f(t, d, c, std::true_type{});
    else
      f(t, d, c, std::false_type{});
  };
  auto by_cap = [&](auto t, auto d) {
    if (cap)
      by_bias(t, d, std::true_type{});
    else
      by_bias(t, d, std::false_type{});
  };
  auto by_dim = [&](auto t) {
    if (hd == 64)
      by_cap(t, std::integral_constant<int, 64>{});
    else
      by_cap(t, std::integral_constant<int, 128>{});
  };
  if (dtype == RUS_DTYPE_F16)
    by_dim(f16{});
  else
    by_dim(bf16{});
}

// Blocks of `rows` tokens over all rows, bound: each holds a token at least.
int64_t blocks_bound(int64_t n, int32_t n_seq, int rows) { return std::min<int64_t>((n + rows - 1) / rows + n_seq + 2, n); }

// How a forward runs: splits = 0: blocks of 128 queries; otherwise blocks of few queries, the keys in `splits` parts of
// `tiles` tiles each. The former walk a row's keys alone (1.6 us per 64 of them, whatever else runs), so they win where
// rows are short or blocks many; the latter share them among four waves and the parts, but read K and V again for every
// 32 / group queries (2.2 us per 128 keys and round of two blocks a CU, 4 us a round aside; heads of 64 half as long).
// How long the rows are beyond the longest is known on the device only: on average tokens over rows. Measured, 12 / 2
// heads of 128, us in blocks of 128 / of few: 100 tokens 9.7 / 8.2, 707 23.3 / 15.6, 2,048 53 / 45, 3,000 75 / 75, 4,096
// 104 / 120, ten rows of 256 13.9 / 23.0, four of 1,024 52 / 57, 4,096 + 2,048 + 1,024 + 993 117 / 165, 1,500 and 27 rows
// of 64 44 / 37; 4 / 1 heads, 4,096 98 / 51; 16 heads of 64 without a causal mask, eight rows of 700 35 / 59, 1,025 +
// 577 + 257 + 64 31 / 29.
struct SplitPlan {
  int splits, tiles;
  int64_t items;  // blocks of few queries, bound over all rows
};

SplitPlan split_plan(int32_t n_seq, int64_t n_q, int64_t n_k, int32_t max_q, int32_t max_k, int32_t h_q, int32_t h_kv,
                     int32_t head_dim) {
  SplitPlan p{0, 0, 0};
  const int grp = h_q / h_kv;
  if (grp > kMaxSplitGroup) return p;
  const int tpb = split_tokens(grp);
  const int64_t base = std::max<int64_t>((n_q + tpb - 1) / tpb, n_seq) * h_kv;
  const int64_t tiles = std::max<int64_t>((static_cast<int64_t>(max_k) + 31) / 32, 1);
  // (a part is worth its share of the join from two tiles a wave on, parts at all from some 1,000 keys)
  const int64_t splits = tiles < 32 ? 1 : std::max<int64_t>(std::min<int64_t>(512 / base, (tiles + 7) / 8), 1);
  const int64_t part = (tiles + splits - 1) / splits;
  const double row = std::min<double>(static_cast<double>(max_k), static_cast<double>(n_k) / n_seq);
  const double wide_load = std::max(1.0, std::max<int64_t>((n_q + kRows - 1) / kRows, n_seq) * h_q / 512.0);
  const double wide_us = 7.0 + 0.8 * std::max(static_cast<double>(tiles), wide_load * row / 32);
  // (queries of a causal row see half of it on average, a few at the end of a cache nearly all)
  const double step_us = head_dim == 64 ? 1.1 : 2.2, steps = max_q < max_k ? row / 128 : row / 256;
  const double few_us =
      4.0 + std::max(0.4 * part, std::max(1.0, base * splits / 512.0) * (4.0 + step_us * steps / splits)) +
      (splits > 1 ? 4.0 : 0.0);
  if (wide_us <= few_us) return p;
  p.items = std::min<int64_t>((n_q + tpb - 1) / tpb + n_seq + 2, n_q);  // a block has a query at least
  p.splits = static_cast<int>(splits);
  p.tiles = static_cast<int>(part);
  return p;
}

// Whether a backward runs in blocks of 32 tokens rather than of 128. The latter walk the longest row's tiles alone (2.8 us
// a tile for dQ, then dK and dV), the former share them among four waves but read the other side again for every 32
// tokens. Measured, 12 / 2 heads of 128, us in blocks of 128 / of 32: 100 tokens 32 / 23, 707 79 / 49, 2,048 194 / 119,
// 3,000 277 / 232, 4,096 378 / 380, two rows of 256 43 / 30, 1,500 and 27 rows of 64 150 / 111; sixteen rows of 32 22 / 25,
// ten of 256 52 / 71, four of 512 71 / 76, of 1,024 167 / 174, eight of 1,024 254 / 282, 4,096 + 2,048 + 1,024 + 993 429 /
// 540; 16 heads of 64, no causal mask, 1,025 + 577 + 257 + 64 89 / 84, eight rows of 700 92 / 156.
bool narrow_bwd(int32_t n_seq, int64_t n_q, int64_t n_k, int32_t max_q, int32_t max_k, int32_t h_q) {
  const double n = static_cast<double>(std::max(n_q, n_k)), seqs = std::max(n_seq, 1);
  const double blocks = std::max(n / 32, seqs) * h_q, row = n / seqs / 32;
  const double narrow_us = 18.0 + blocks * (0.042 + 0.0014 * row);
  return narrow_us < 18.0 + 2.8 * std::max(max_q, max_k) / 32;
}

// The backward's workspace: the heads' parts of dK and dV where heads share keys, and D.
int64_t bwd_floats(int64_t n_q, int64_t n_k, int32_t h_q, int32_t h_kv, int32_t head_dim) {
  return (h_q > h_kv ? 2 * static_cast<int64_t>(h_q) * n_k * head_dim : 0) + static_cast<int64_t>(h_q) * n_q;
}

// Launch size of n_items for every head (whole chunks of head_item's).
int item_grid(const char* fn, int64_t n_items, const MaskedArgs& a, int64_t& grid) {
  const int64_t chunk = 8 * (a.h_q / a.h_kv), items = n_items * a.h_q;
  grid = (items + chunk - 1) / chunk * chunk;
  if (grid * 64 * kWaves >= (int64_t(1) << 32) || a.n_k * a.h_kv * 32 >= (int64_t(1) << 32))
    return fail(RUS_ERR_UNSUPPORTED, "%s: %lld blocks beyond one dispatch", fn, (long long)grid);
  return RUS_OK;
}

// Sizes that every entry point takes.
int check_sizes(const char* fn, int32_t n_seq, int64_t n_q, int64_t n_k, int32_t max_q, int32_t max_k, int32_t h_q,
                int32_t h_kv, int32_t head_dim) {
  if (head_dim != 64 && head_dim != 128)
    return fail(RUS_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", fn, head_dim);
  if (h_q <= 0 || h_kv <= 0 || h_q % h_kv || h_q > 65535)
    return fail(RUS_ERR_INVALID, "%s: h_q=%d must be a multiple of h_kv=%d, at most 65535", fn, h_q, h_kv);
  if (n_seq <= 0 || n_seq > (1 << 22) || n_q < 0 || n_k < 0 || n_q >= (int64_t(1) << 31) - 256 || n_k >= (int64_t(1) << 31) - 256 ||
      max_q < 0 || max_k < 0)
    return fail(RUS_ERR_INVALID, "%s: n_seq=%d n_q=%lld n_k=%lld max_q=%d max_k=%d", fn, n_seq, (long long)n_q,
                (long long)n_k, max_q, max_k);
  return RUS_OK;
}

int check_rows(const char* fn, const char* name, const void* p, int64_t n, int64_t st, int64_t sh) {
  if (n == 0) return RUS_OK;
  if (st >= (1 << 26)) return fail(RUS_ERR_UNSUPPORTED, "%s: %s has a token stride of 2^26 elements or more", fn, name);
  if (!p || !aligned(p, 16) || st % 8 || sh % 8 || st < 0 || sh < 0)
    return fail(RUS_ERR_INVALID, "%s: %s must be 16-byte aligned with strides that are multiples of 8", fn, name);
  return RUS_OK;
}

int check_call(const char* fn, const int32_t* cu_q, const int32_t* cu_k, float scale, float softcap, int32_t dtype) {
  if (!cu_q || !cu_k) return fail(RUS_ERR_INVALID, "%s: null cu_seqlens", fn);
  if (dtype != RUS_DTYPE_F16 && dtype != RUS_DTYPE_BF16)
    return fail(RUS_ERR_INVALID, "%s: dtype %d (fp16 or bf16)", fn, dtype);
  if (!(scale > 0.0f) || !(scale < INFINITY))
    return fail(RUS_ERR_INVALID, "%s: scale %g must be positive and finite", fn, static_cast<double>(scale));
  if (!(softcap >= 0.0f) || !(softcap < INFINITY))
    return fail(RUS_ERR_INVALID, "%s: softcap %g must be 0 (none) or positive and finite", fn,
                static_cast<double>(softcap));
  return RUS_OK;
}

void set_scores(MaskedArgs& a, float scale, float softcap, const float* slopes, const int32_t* prefix, int causal) {
  a.scale = scale;
  a.sl2 = scale * kLog2e;
  if (softcap > 0.0f) {
    a.kc = scale / softcap;
    a.k2 = 2.0f * kLog2e * a.kc;
    a.cap2 = softcap * kLog2e;
  }
  a.slopes = slopes;
  a.prefix = prefix;
  a.causal = causal != 0;
}

}  // namespace
}  // namespace rus

extern "C" int rus_attn_masked_workspace(int32_t n_seq, int64_t n_q, int64_t n_k, int32_t max_q, int32_t max_k,
                                         int32_t h_q, int32_t h_kv, int32_t head_dim, int32_t backward,
                                         int64_t* floats) {
  using namespace rus;
  const char* fn = "rus_attn_masked_workspace";
  if (!floats) return fail(RUS_ERR_INVALID, "%s: null result", fn);
  if (int e = check_sizes(fn, n_seq, n_q, n_k, max_q, max_k, h_q, h_kv, head_dim)) return e;
  if (backward) {
    *floats = bwd_floats(n_q, n_k, h_q, h_kv, head_dim);
    return RUS_OK;
  }
  const SplitPlan p = split_plan(n_seq, n_q, n_k, max_q, max_k, h_q, h_kv, head_dim);
  *floats = p.splits > 1 ? p.splits * n_q * h_q * (head_dim + 4) : 0;
  return RUS_OK;
}

extern "C" int rus_attn_masked_plan(int32_t n_seq, int64_t n_q, int64_t n_k, int32_t max_q, int32_t max_k, int32_t h_q,
                                    int32_t h_kv, int32_t head_dim, int32_t* plan) {
  using namespace rus;
  const char* fn = "rus_attn_masked_plan";
  if (!plan) return fail(RUS_ERR_INVALID, "%s: null result", fn);
  if (int e = check_sizes(fn, n_seq, n_q, n_k, max_q, max_k, h_q, h_kv, head_dim)) return e;
  const SplitPlan p = split_plan(n_seq, n_q, n_k, max_q, max_k, h_q, h_kv, head_dim);
  plan[0] = p.splits;
  plan[1] = p.tiles;
  plan[2] = narrow_bwd(n_seq, n_q, n_k, max_q, max_k, h_q) ? 32 : kRows;
  return RUS_OK;
}

extern "C" int rus_attn_masked_fwd(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k,
                                   int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                                   int64_t v_stride_h, const int32_t* cu_q, const int32_t* cu_k, int32_t n_seq,
                                   int64_t n_q, int64_t n_k, int32_t max_q, int32_t max_k, int32_t h_q, int32_t h_kv,
                                   int32_t head_dim, float scale, int32_t causal, const int32_t* prefix, float softcap,
                                   const float* slopes, int32_t dtype, void* out, float* lse, float* workspace,
                                   int64_t n_workspace, void* stream) {
  using namespace rus;
  const char* fn = "rus_attn_masked_fwd";
  if (int e = check_sizes(fn, n_seq, n_q, n_k, max_q, max_k, h_q, h_kv, head_dim)) return e;
  if (int e = check_call(fn, cu_q, cu_k, scale, softcap, dtype)) return e;
  if (int e = check_rows(fn, "q", q, n_q, q_stride_t, q_stride_h)) return e;
  if (int e = check_rows(fn, "k", k, n_k, k_stride_t, k_stride_h)) return e;
  if (int e = check_rows(fn, "v", v, n_k, v_stride_t, v_stride_h)) return e;
  if (n_q == 0) return RUS_OK;
  if (!out || !lse || !aligned(out, 16) || !aligned(lse, 4))
    return fail(RUS_ERR_INVALID, "%s: null or misaligned output", fn);
  MaskedArgs a{};
  a.q = q, a.q_st = q_stride_t, a.q_sh = q_stride_h;
  a.k = k, a.k_st = k_stride_t, a.k_sh = k_stride_h;
  a.v = v, a.v_st = v_stride_t, a.v_sh = v_stride_h;
  a.out = out, a.lse = lse;
  a.cu_q = cu_q, a.cu_k = cu_k, a.n_seq = n_seq, a.n_q = n_q, a.n_k = n_k, a.h_q = h_q, a.h_kv = h_kv;
  set_scores(a, scale, softcap, slopes, prefix, causal);
  const SplitPlan p = split_plan(n_seq, n_q, n_k, max_q, max_k, h_q, h_kv, head_dim);
  if (p.splits) {
    a.splits = p.splits;
    a.split_tiles = p.tiles;
    a.part = workspace;
    const int64_t need = p.splits > 1 ? p.splits * n_q * h_q * (head_dim + 4) : 0;
    if (need && (!workspace || n_workspace < need || !aligned(workspace, 16)))
      return fail(RUS_ERR_INVALID, "%s: workspace of %lld floats, %lld needed", fn, (long long)n_workspace,
                  (long long)need);
    const int64_t blocks = p.items * h_kv * p.splits;
    if (blocks * 64 * kWaves >= (int64_t(1) << 32))
      return fail(RUS_ERR_UNSUPPORTED, "%s: %lld blocks beyond one dispatch", fn, (long long)blocks);
    dispatch(dtype, head_dim, softcap > 0.0f, slopes != nullptr, [&](auto t, auto d, auto c, auto b) {
      hipLaunchKernelGGL((masked_split_kernel<decltype(t), decltype(d)::value, decltype(c)::value, decltype(b)::value>),
                         dim3(static_cast<unsigned>(blocks)), dim3(64 * kWaves), 0, static_cast<hipStream_t>(stream), a);
      auto join = [&](auto waves) {
        hipLaunchKernelGGL((masked_join_kernel<decltype(t), decltype(d)::value, decltype(c)::value, decltype(b)::value,
                                               decltype(waves)::value>),
                           dim3(static_cast<unsigned>(n_q * h_q)), dim3(64 * decltype(waves)::value), 0,
                           static_cast<hipStream_t>(stream), a);
      };
      // 8 tokens over caches up to 8,191 (32 parts) 4.1 us with 4 waves, 5.7 with 16; 131,071 keys (256 parts) 10.9, 7.9
      if (p.splits > 64)
        join(std::integral_constant<int, 16>{});
      else if (p.splits > 1)
        join(std::integral_constant<int, 4>{});
    });
    return check_launch(fn);
  }
  a.n_blocks = static_cast<int>(blocks_bound(n_q, n_seq, kRows));
  int64_t grid;
  if (int e = item_grid(fn, a.n_blocks, a, grid)) return e;
  dispatch(dtype, head_dim, softcap > 0.0f, slopes != nullptr, [&](auto t, auto d, auto c, auto b) {
    hipLaunchKernelGGL((masked_fwd_kernel<decltype(t), decltype(d)::value, decltype(c)::value, decltype(b)::value>),
                       dim3(grid), dim3(64 * kWaves), 0, static_cast<hipStream_t>(stream), a);
  });
  return check_launch(fn);
}

extern "C" int rus_attn_masked_bwd(const void* dout, int64_t do_stride_t, int64_t do_stride_h, const void* q,
                                   int64_t q_stride_t, int64_t q_stride_h, const void* k, int64_t k_stride_t,
                                   int64_t k_stride_h, const void* v, int64_t v_stride_t, int64_t v_stride_h,
                                   const void* out, const float* lse, const int32_t* cu_q, const int32_t* cu_k,
                                   int32_t n_seq, int64_t n_q, int64_t n_k, int32_t max_q, int32_t max_k, int32_t h_q,
                                   int32_t h_kv, int32_t head_dim, float scale, int32_t causal, const int32_t* prefix,
                                   float softcap, const float* slopes, int32_t dtype, void* dq, void* dk, void* dv,
                                   float* workspace, int64_t n_workspace, void* stream) {
  using namespace rus;
  const char* fn = "rus_attn_masked_bwd";
  if (int e = check_sizes(fn, n_seq, n_q, n_k, max_q, max_k, h_q, h_kv, head_dim)) return e;
  if (int e = check_call(fn, cu_q, cu_k, scale, softcap, dtype)) return e;
  if (int e = check_rows(fn, "dout", dout, n_q, do_stride_t, do_stride_h)) return e;
  if (int e = check_rows(fn, "q", q, n_q, q_stride_t, q_stride_h)) return e;
  if (int e = check_rows(fn, "k", k, n_k, k_stride_t, k_stride_h)) return e;
  if (int e = check_rows(fn, "v", v, n_k, v_stride_t, v_stride_h)) return e;
  if (n_q == 0 && n_k == 0) return RUS_OK;
  if ((n_q && (!out || !lse || !dq || !aligned(out, 16) || !aligned(lse, 4) || !aligned(dq, 16))) ||
      (n_k && (!dk || !dv || !aligned(dk, 16) || !aligned(dv, 16))))
    return fail(RUS_ERR_INVALID, "%s: null or misaligned argument", fn);
  MaskedArgs a{};
  a.dout = dout, a.do_st = do_stride_t, a.do_sh = do_stride_h;
  a.q = q, a.q_st = q_stride_t, a.q_sh = q_stride_h;
  a.k = k, a.k_st = k_stride_t, a.k_sh = k_stride_h;
  a.v = v, a.v_st = v_stride_t, a.v_sh = v_stride_h;
  a.o = out, a.lse = const_cast<float*>(lse);
  a.out = dq, a.dk = dk, a.dv = dv;
  a.cu_q = cu_q, a.cu_k = cu_k, a.n_seq = n_seq, a.n_q = n_q, a.n_k = n_k, a.h_q = h_q, a.h_kv = h_kv;
  set_scores(a, scale, softcap, slopes, prefix, causal);
  const bool narrow = narrow_bwd(n_seq, n_q, n_k, max_q, max_k, h_q);
  const int rows = narrow ? 32 : kRows;
  a.n_blocks = static_cast<int>(blocks_bound(n_q, n_seq, rows));
  a.n_kblocks = static_cast<int>(blocks_bound(n_k, n_seq, rows));
  int64_t dq_grid, dkdv_grid;
  if (int e = item_grid(fn, a.n_blocks, a, dq_grid)) return e;
  if (int e = item_grid(fn, a.n_kblocks, a, dkdv_grid)) return e;
  const int64_t need = bwd_floats(n_q, n_k, h_q, h_kv, head_dim);
  if (need && (!workspace || n_workspace < need || !aligned(workspace, 16)))
    return fail(RUS_ERR_INVALID, "%s: workspace of %lld floats, %lld needed", fn, (long long)n_workspace,
                (long long)need);
  a.dk_part = workspace;
  a.dv_part = workspace + static_cast<int64_t>(h_q) * n_k * head_dim;
  a.dsum = workspace + need - static_cast<int64_t>(h_q) * n_q;
  const dim3 dq_blocks(static_cast<unsigned>(dq_grid)), dkdv_blocks(static_cast<unsigned>(dkdv_grid)),
      threads(64 * kWaves);
  hipStream_t st = static_cast<hipStream_t>(stream);
  dispatch(dtype, head_dim, softcap > 0.0f, slopes != nullptr, [&](auto t, auto d, auto c, auto b) {
    using T = decltype(t);
    constexpr int kDim = decltype(d)::value;
    constexpr bool kCap = decltype(c)::value, kBias = decltype(b)::value;
    if (narrow) {
      if (n_q) hipLaunchKernelGGL((masked_narrow_dq_kernel<T, kDim, kCap, kBias>), dq_blocks, threads, 0, st, a);
      if (n_k) hipLaunchKernelGGL((masked_narrow_dkdv_kernel<T, kDim, kCap, kBias>), dkdv_blocks, threads, 0, st, a);
    } else {
      if (n_q) hipLaunchKernelGGL((masked_dq_kernel<T, kDim, kCap, kBias>), dq_blocks, threads, 0, st, a);
      if (n_k) hipLaunchKernelGGL((masked_dkdv_kernel<T, kDim, kCap, kBias>), dkdv_blocks, threads, 0, st, a);
    }
  });
  if (int e = check_launch(fn)) return e;
  if (h_q == h_kv || n_k == 0) return RUS_OK;
  const int hd4 = head_dim / 4;
  const dim3 sums(static_cast<unsigned>((n_k * h_kv * hd4 + 255) / 256), 2);
  if (dtype == RUS_DTYPE_F16)
    hipLaunchKernelGGL(masked_group_sum_kernel<f16>, sums, dim3(256), 0, st, a, hd4);
  else
    hipLaunchKernelGGL(masked_group_sum_kernel<bf16>, sums, dim3(256), 0, st, a, hd4);
  return check_launch(fn);
}
