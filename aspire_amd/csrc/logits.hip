// Penalties for repeated tokens, biases and grammar masks on logits (gfx950).
//
// A workgroup takes one chunk of the vocabulary for one request. It counts the request's history tokens of the chunk in LDS
// once (one 32-bit word a token: output occurrences, bit 31 for the prompt's) and lays the chunk's biases beside them, then streams
// the chunk of each of the request's rows through: 16 bytes of logits a thread, their counts and biases from LDS,
// the mask's byte, one rounding. A drafted token's row first adds its path's tokens to the counts and takes them out after.
// HBM bounds it at batch sizes (logits once in, once out, and an eighth of a byte of mask a token); history is
// read once a chunk, from L2.
#include <algorithm>

#include "common.h"

namespace aspire {
namespace {

struct LogitsParams {
  aspire_adjust_logits_args a;
  int32_t chunk;  // tokens a workgroup takes, a multiple of 8
};

constexpr int kLogitThreads = 256;
constexpr uint32_t kPrompt = 0x80000000u;

template <typename T> struct Pack;
struct Bf16 {};
struct Fp16 {};
template <> struct Pack<Bf16> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float up(raw x) { return __uint_as_float(uint32_t(x) << 16); }
  static __device__ __forceinline__ raw down(float x) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x)); }
};
template <> struct Pack<Fp16> {
  typedef uint16_t raw;
  static __device__ __forceinline__ float up(raw x) { return float(__builtin_bit_cast(_Float16, x)); }
  static __device__ __forceinline__ raw down(float x) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x)); }
};
template <> struct Pack<float> {
  typedef float raw;
  static __device__ __forceinline__ float up(raw x) { return x; }
  static __device__ __forceinline__ raw down(float x) { return x; }
};

// n values at any 2- or 4-byte aligned place, in one access
template <typename R, int n> struct __attribute__((packed, aligned(sizeof(R)))) Vec { R v[n]; };

template <typename T, bool kCounts, bool kBias, bool kMask>
__global__ __launch_bounds__(kLogitThreads) void adjust_logits_kernel(LogitsParams p) {
  typedef typename Pack<T>::raw R;
  constexpr int kVec = 8;  // a byte of mask
  extern __shared__ uint32_t logits_lds[];
  uint32_t* const counts = logits_lds;
  float* const bias = reinterpret_cast<float*>(logits_lds + (kCounts ? p.chunk : 0));
  const aspire_adjust_logits_args& a = p.a;
  const int b = blockIdx.y, v0 = blockIdx.x * p.chunk, width = min(p.chunk, a.vocab - v0);
  const int64_t token0 = a.vocab_start + v0;  // the chunk's first token
  int row0 = b, row1 = b + 1;
  if (a.qo_indptr != nullptr) {
    row0 = max(a.qo_indptr[b], 0);
    row1 = min(a.qo_indptr[b + 1], a.tokens);
  }
  if (row0 >= row1) return;

  float repetition = 1.f, presence = 0.f, frequency = 0.f;
  if (kCounts || kBias) {
    for (int i = threadIdx.x; i < p.chunk; i += kLogitThreads) {
      if (kCounts) counts[i] = 0;
      if (kBias) bias[i] = 0.f;
    }
    __syncthreads();
  }
  if (kCounts) {
    if (a.repetition != nullptr) repetition = a.repetition[b];
    if (a.presence != nullptr) presence = a.presence[b];
    if (a.frequency != nullptr) frequency = a.frequency[b];
    if (a.history != nullptr) {
      const int32_t* const history = a.history + b * a.history_stride;
      const int len = min(a.history_lens[b], a.history_len), told = a.prompt_lens != nullptr ? a.prompt_lens[b] : 0;
      for (int i = threadIdx.x; i < len; i += kLogitThreads) {
        const int64_t at = int64_t(history[i]) - token0;
        if (at < 0 || at >= width) continue;
        if (i < told) atomicOr(&counts[at], kPrompt);
        else atomicAdd(&counts[at], 1u);
      }
    }
  }
  if (kBias) {
    const int end = min(a.bias_indptr[b + 1], a.bias_entries);
    for (int i = max(a.bias_indptr[b], 0) + threadIdx.x; i < end; i += kLogitThreads) {
      const int64_t at = int64_t(a.bias_ids[i]) - token0;
      if (at >= 0 && at < width) bias[at] = a.bias_values[i];
    }
  }
  if (kCounts || kBias) __syncthreads();

  // the tokens of a row's path come into the counts (or out again)
  const auto path = [&](int row, uint32_t by) {
    const int n = min(row1 - row0, 64 * a.mask_words);
    for (int i = threadIdx.x; i < n; i += kLogitThreads) {
      if (!((uint64_t(a.tree_masks[row * a.mask_stride + (i >> 6)]) >> (i & 63)) & 1)) continue;
      const int64_t at = int64_t(a.tree_tokens[row0 + i]) - token0;
      if (at >= 0 && at < width) atomicAdd(&counts[at], by);
    }
  };
  const auto adjust = [&](float x, int i, bool allowed) {
    if (kCounts) {
      const uint32_t c = counts[i];
      if (c != 0) {
        x = x > 0.f ? x / repetition : x * repetition;
        const uint32_t written = c & ~kPrompt;
        if (written != 0) x = (x - frequency * float(written)) - presence;
      }
    }
    if (kBias) x += bias[i];
    return allowed ? x : -__builtin_huge_valf();
  };
  for (int row = row0; row < row1; ++row) {
    const bool tree = kCounts && a.tree_masks != nullptr;
    if (tree) {
      path(row, 1u);
      __syncthreads();
    }
    const R* const in = static_cast<const R*>(a.logits) + row * a.stride + v0;
    R* const out = static_cast<R*>(a.out) + row * a.out_stride + v0;
    const uint8_t* mask = nullptr;
    if (kMask) {
      const int g = a.grammar_rows != nullptr ? a.grammar_rows[row] : row;
      if (g >= 0 && g < a.num_grammar_rows) mask = reinterpret_cast<const uint8_t*>(a.grammar + g * a.grammar_stride) + v0 / 8;
    }
    const int whole = width / kVec;
    for (int k = threadIdx.x; k < whole; k += kLogitThreads) {
      const int i = k * kVec;
      Vec<R, kVec> x = *reinterpret_cast<const Vec<R, kVec>*>(in + i);
      const uint32_t allowed = kMask && mask != nullptr ? mask[k] : 255u;
#pragma unroll
      for (int e = 0; e < kVec; ++e) x.v[e] = Pack<T>::down(adjust(Pack<T>::up(x.v[e]), i + e, (allowed >> e) & 1));
      *reinterpret_cast<Vec<R, kVec>*>(out + i) = x;
    }
    for (int i = whole * kVec + threadIdx.x; i < width; i += kLogitThreads) {
      const bool allowed = !kMask || mask == nullptr || ((mask[i >> 3] >> (i & 7)) & 1);
      out[i] = Pack<T>::down(adjust(Pack<T>::up(in[i]), i, allowed));
    }
    if (tree) {
      __syncthreads();
      path(row, ~0u);  // - 1
    }
  }
}

template <typename T, bool kCounts, bool kBias>
void launch_mask(const LogitsParams& p, dim3 grid, int lds, hipStream_t s) {
  if (p.a.grammar != nullptr) adjust_logits_kernel<T, kCounts, kBias, true><<<grid, kLogitThreads, lds, s>>>(p);
  else adjust_logits_kernel<T, kCounts, kBias, false><<<grid, kLogitThreads, lds, s>>>(p);
}
template <typename T>
void launch_logits(const LogitsParams& p, bool counts, bool bias, dim3 grid, int lds, hipStream_t s) {
  if (counts && bias) launch_mask<T, true, true>(p, grid, lds, s);
  else if (counts) launch_mask<T, true, false>(p, grid, lds, s);
  else if (bias) launch_mask<T, false, true>(p, grid, lds, s);
  else launch_mask<T, false, false>(p, grid, lds, s);
}

}  // namespace
}  // namespace aspire

extern "C" int aspire_adjust_logits(const aspire_adjust_logits_args* a, void* stream) {
  using namespace aspire;
  ASPIRE_CHECK_ARG(a != nullptr, "null arguments");
  ASPIRE_CHECK_ARG(a->tokens >= 0 && a->vocab >= 0 && a->requests >= 0 && a->history_len >= 0 && a->mask_words >= 0 &&
                       a->num_grammar_rows >= 0 && a->bias_entries >= 0 && a->dtype >= 0 && a->dtype <= 2, "bad sizes");
  ASPIRE_CHECK_ARG(a->requests <= 65535, "more than 65,535 requests");
  ASPIRE_CHECK_ARG(a->vocab <= (1 << 30), "more than 2^30 tokens in the vocabulary");
  if (a->tokens == 0 || a->vocab == 0 || a->requests == 0) return ASPIRE_OK;
  ASPIRE_CHECK_ARG(a->logits && a->out, "null logits");
  ASPIRE_CHECK_ARG(a->qo_indptr || a->requests <= a->tokens, "a request a row, and fewer rows");
  ASPIRE_CHECK_ARG(!a->history || a->history_lens, "a history needs its lengths");
  ASPIRE_CHECK_ARG(!a->tree_masks == !a->tree_tokens, "tree_tokens and tree_masks go together");
  ASPIRE_CHECK_ARG(!a->tree_masks || a->qo_indptr, "trees need qo_indptr");
  ASPIRE_CHECK_ARG(!a->bias_indptr || a->bias_entries == 0 || (a->bias_ids && a->bias_values), "null biases");
  const bool counts = (a->history || a->tree_masks) && (a->repetition || a->presence || a->frequency);
  const bool bias = a->bias_indptr != nullptr && a->bias_entries > 0;
  LogitsParams p{*a, 4096};
  const dim3 grid((a->vocab + p.chunk - 1) / p.chunk, a->requests);
  const int lds = p.chunk * 4 * ((counts ? 1 : 0) + (bias ? 1 : 0));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == 0) launch_logits<Bf16>(p, counts, bias, grid, lds, s);
  else if (a->dtype == 1) launch_logits<Fp16>(p, counts, bias, grid, lds, s);
  else launch_logits<float>(p, counts, bias, grid, lds, s);
  ASPIRE_CHECK_LAUNCH();
  return ASPIRE_OK;
}
