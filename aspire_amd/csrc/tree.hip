// Attention of drafted trees over a paged cache (gfx950): a request's tokens see its cached keys and, of its own last n keys,
// those of their ancestors.
//
// One workgroup a (token, q head): a wave takes every fourth key, a lane head_dim / 64 of its values; the running maximum and sum
// stay in registers and the four waves join through LDS.
#include <algorithm>
#include <cmath>

#include "common.h"

namespace aspire {
namespace {

constexpr float kNegInfT = -__builtin_huge_valf();

struct TreeParams {
  aspire_tree_attention_args a;
  float scale_log2;
};

template <bool kFp16>
__device__ __forceinline__ float widen(uint16_t x) {
  return kFp16 ? float(__builtin_bit_cast(_Float16, x)) : __uint_as_float(uint32_t(x) << 16);
}
template <bool kFp16>
__device__ __forceinline__ uint16_t narrow(float x) {
  return kFp16 ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(x)) : __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
}

template <bool kFp16, int kDim>
__global__ __launch_bounds__(256) void tree_attention_kernel(TreeParams p) {
  constexpr int kPer = kDim / 64;
  __shared__ float top[4], sum[4], part[4][kDim];
  const aspire_tree_attention_args& a = p.a;
  const int lane = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6);
  const int t = blockIdx.x, head = blockIdx.y, kv_head = head / (a.num_qo_heads / a.num_kv_heads);
  const int b = wave_last_le(a.qo_indptr, a.rows, t);
  if (b < 0 || t >= a.qo_indptr[b + 1]) return;
  const int q0 = a.qo_indptr[b], n = a.qo_indptr[b + 1] - q0;
  const int first = a.kv_indptr[b], pages = a.kv_indptr[b + 1] - first;
  const int len = pages > 0 ? (pages - 1) * a.page_size + a.kv_last_page_len[b] : 0;
  const uint16_t* const q = static_cast<const uint16_t*>(a.q) + t * a.q_stride_t + head * a.q_stride_h;
  float qv[kPer], o[kPer], m = kNegInfT, l = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) qv[i] = widen<kFp16>(q[lane * kPer + i]), o[i] = 0.f;
  for (int key = wave; key < len; key += 4) {
    const int j = key - (len - n);
    if (j >= 0 && !(j < 64 * a.mask_words && ((a.masks[t * a.mask_stride + (j >> 6)] >> (j & 63)) & 1))) continue;
    const int64_t entry = int64_t(first) + key / a.page_size;
    if (entry < 0 || entry >= a.num_page_indices) continue;
    const int page = a.kv_indices[entry];
    if (page < 0 || page >= a.num_pages) continue;
    const uint16_t* const k = static_cast<const uint16_t*>(a.kv_cache) + page * a.cache_stride_p +
                              (key % a.page_size) * a.cache_stride_t + kv_head * a.cache_stride_h + lane * kPer;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) x += qv[i] * widen<kFp16>(k[i]);
    x = wave_sum_f(x) * p.scale_log2;
    const float up = fmaxf(m, x), use = up == kNegInfT ? 0.f : up;
    const float keep = __builtin_amdgcn_exp2f(m - use), w = __builtin_amdgcn_exp2f(x - use);
    m = up;
    l = l * keep + w;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = o[i] * keep + (w != 0.f ? w * widen<kFp16>(k[a.cache_stride_kv + i]) : 0.f);
  }
  if (lane == 0) top[wave] = m, sum[wave] = l;
#pragma unroll
  for (int i = 0; i < kPer; ++i) part[wave][lane * kPer + i] = o[i];
  __syncthreads();
  if (wave != 0) return;
  m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  const float use = m == kNegInfT ? 0.f : m;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) o[i] = 0.f;
  for (int w = 0; w < 4; ++w) {
    const float keep = __builtin_amdgcn_exp2f(top[w] - use);
    l += keep * sum[w];
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] += keep * part[w][lane * kPer + i];
  }
  uint16_t* const out = static_cast<uint16_t*>(a.out) + t * a.out_stride_t + head * a.out_stride_h;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < kPer; ++i) out[lane * kPer + i] = narrow<kFp16>(o[i] * inv);
  if (a.lse != nullptr && lane == 0) a.lse[int64_t(t) * a.num_qo_heads + head] = l == 0.f ? kNegInfT : use + __builtin_log2f(l);
}

}  // namespace
}  // namespace aspire

extern "C" int64_t aspire_tree_attention_workspace(int32_t, int32_t, int32_t, int32_t, int32_t) { return 0; }

extern "C" int aspire_tree_attention(const aspire_tree_attention_args* a, void* stream) {
  using namespace aspire;
  ASPIRE_CHECK_ARG(a != nullptr, "null arguments");
  ASPIRE_CHECK_ARG(a->tokens >= 0 && a->rows >= 0 && a->mask_words >= 0 && a->num_pages >= 0 && a->num_page_indices >= 0, "bad sizes");
  ASPIRE_CHECK_ARG(a->num_kv_heads > 0 && a->num_qo_heads > 0 && a->num_qo_heads % a->num_kv_heads == 0 &&
                       a->num_qo_heads <= 1024, "q heads must be a multiple of the kv heads, at most 1,024");
  ASPIRE_CHECK_ARG(a->head_dim == 64 || a->head_dim == 128, "head_dim must be 64 or 128");
  ASPIRE_CHECK_ARG(a->page_size >= 16 && a->page_size <= 1024 && (a->page_size & (a->page_size - 1)) == 0, "page_size must be a power of two from 16 to 1,024");
  ASPIRE_CHECK_ARG(a->dtype == 0 || a->dtype == 1, "dtype must be 0 or 1");
  ASPIRE_CHECK_ARG(std::isfinite(a->sm_scale) && a->sm_scale > 0.f && a->sm_scale <= 1e30f, "sm_scale must be positive and finite");
  if (a->tokens == 0 || a->rows == 0) return ASPIRE_OK;
  ASPIRE_CHECK_ARG(a->q && a->out && a->qo_indptr && a->kv_indptr && a->kv_last_page_len &&
                       (a->masks || a->mask_words == 0) && (a->kv_cache || a->num_pages == 0) &&
                       (a->kv_indices || a->num_page_indices == 0), "null array");
  TreeParams p{*a, a->sm_scale * 1.4426950408889634f};
  const dim3 grid(a->tokens, a->num_qo_heads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == 1) {
    if (a->head_dim == 128) tree_attention_kernel<true, 128><<<grid, 256, 0, s>>>(p);
    else tree_attention_kernel<true, 64><<<grid, 256, 0, s>>>(p);
  } else {
    if (a->head_dim == 128) tree_attention_kernel<false, 128><<<grid, 256, 0, s>>>(p);
    else tree_attention_kernel<false, 64><<<grid, 256, 0, s>>>(p);
  }
  ASPIRE_CHECK_LAUNCH();
  return ASPIRE_OK;
}
