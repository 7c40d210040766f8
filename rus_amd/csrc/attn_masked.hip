// Attention over packed rows with a tanh cap on the scores, a bias by distance, a prefix that every query sees, and
// fewer queries than keys where a cache is read: forward and backward, fp16 / bf16, head dims 64 and 128. The
// definition is in attn_masked.h.
#include "attn_masked.h"

namespace rus {
namespace {

constexpr int kWaves = 4, kRows = 128;  // waves of a block, tokens of a block

template <typename T, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * kWaves) void masked_fwd_kernel(MaskedArgs a) {
  int s, b, nb;
  if (!find_span_block<kRows>(a.cu_q, a.n_seq, static_cast<int>(a.n_q), blockIdx.x, s, b, nb)) return;
  const MaskedRow r = as_queries(masked_row(a, s), s, a.n_seq);
  const int wave = threadIdx.x >> 6;
  for (int i = b * kRows + wave; i < min((b + 1) * kRows, r.lq); i += kWaves)
    plain_fwd_row<T, HD, CAP, BIAS>(a, r, i, blockIdx.y);
}

template <typename T, int HD, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * kWaves) void masked_bwd_kernel(MaskedArgs a) {
  int s, b, nb;
  const int wave = threadIdx.x >> 6, blk = blockIdx.x;
  if (blk < a.n_kblocks) {
    const int grp = a.h_q / a.h_kv, head = blockIdx.y;
    if (head % grp) return;
    if (!find_span_block<kRows>(a.cu_k, a.n_seq, static_cast<int>(a.n_k), blk, s, b, nb)) return;
    const MaskedRow r = as_keys(masked_row(a, s), s, a.n_seq);
    for (int j = b * kRows + wave; j < min((b + 1) * kRows, r.lk); j += kWaves)
      plain_dkv_row<T, HD, CAP, BIAS>(a, r, j, head, head + grp, nullptr, nullptr);
    return;
  }
  if (!find_span_block<kRows>(a.cu_q, a.n_seq, static_cast<int>(a.n_q), blk - a.n_kblocks, s, b, nb)) return;
  const MaskedRow r = as_queries(masked_row(a, s), s, a.n_seq);
  for (int i = b * kRows + wave; i < min((b + 1) * kRows, r.lq); i += kWaves)
    plain_dq_row<T, HD, CAP, BIAS>(a, r, i, blockIdx.y);
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

int64_t blocks_bound(int64_t n, int32_t n_seq) { return (n + kRows - 1) / kRows + n_seq + 2; }

// Sizes that every entry point takes.
int check_sizes(const char* fn, int32_t n_seq, int64_t n_q, int64_t n_k, int32_t max_q, int32_t max_k, int32_t h_q,
                int32_t h_kv, int32_t head_dim) {
  if (head_dim != 64 && head_dim != 128)
    return fail(RUS_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", fn, head_dim);
  if (h_q <= 0 || h_kv <= 0 || h_q % h_kv || h_q > 65535)
    return fail(RUS_ERR_INVALID, "%s: h_q=%d must be a multiple of h_kv=%d, at most 65535", fn, h_q, h_kv);
  if (n_seq <= 0 || n_q < 0 || n_k < 0 || n_q >= (int64_t(1) << 31) - 256 || n_k >= (int64_t(1) << 31) - 256 ||
      max_q < 0 || max_k < 0)
    return fail(RUS_ERR_INVALID, "%s: n_seq=%d n_q=%lld n_k=%lld max_q=%d max_k=%d", fn, n_seq, (long long)n_q,
                (long long)n_k, max_q, max_k);
  return RUS_OK;
}

int check_rows(const char* fn, const char* name, const void* p, int64_t n, int64_t st, int64_t sh) {
  if (n == 0) return RUS_OK;
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
  *floats = 0;
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
  a.n_blocks = static_cast<int>(blocks_bound(n_q, n_seq));
  dispatch(dtype, head_dim, softcap > 0.0f, slopes != nullptr, [&](auto t, auto d, auto c, auto b) {
    hipLaunchKernelGGL((masked_fwd_kernel<decltype(t), decltype(d)::value, decltype(c)::value, decltype(b)::value>),
                       dim3(a.n_blocks, h_q), dim3(64 * kWaves), 0, static_cast<hipStream_t>(stream), a);
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
  a.n_blocks = static_cast<int>(blocks_bound(n_q, n_seq));
  a.n_kblocks = static_cast<int>(blocks_bound(n_k, n_seq));
  dispatch(dtype, head_dim, softcap > 0.0f, slopes != nullptr, [&](auto t, auto d, auto c, auto b) {
    hipLaunchKernelGGL((masked_bwd_kernel<decltype(t), decltype(d)::value, decltype(c)::value, decltype(b)::value>),
                       dim3(a.n_blocks + a.n_kblocks, h_q), dim3(64 * kWaves), 0, static_cast<hipStream_t>(stream), a);
  });
  return check_launch(fn);
}
