// Penalties for repeated tokens, biases and grammar masks on logits (gfx950).
//
// A workgroup takes one chunk of the vocabulary for one request (or some of its rows). It counts the request's history tokens of
// the chunk in LDS (a 32-bit word a token: occurrences in the output, one bit for the prompt's, one for tokens that the request's
// tree drafts) and lays the chunk's biases beside them, while its first logits are on their way; then the chunk of every row
// streams through: 16 or 32 bytes of logits a thread, their words from LDS, a byte of the mask, one rounding, two vectors a thread
// in flight. Rows only read the words: a token that the tree drafts is counted on a row's own path where it is met.
// HBM bounds it at batch sizes (logits once in, once out, and an eighth of a byte of mask a token); history is
// read once a chunk, from L2.
#include <algorithm>

#include "common.h"

namespace aspire {
namespace {

struct LogitsParams {
  aspire_adjust_logits_args a;
  int32_t chunk_log2;  // tokens a workgroup takes, 1,024 to 8,192
  int32_t row_parts;   // workgroups that share a request's rows of a chunk
};

constexpr int kLogitThreads = 512;
constexpr uint32_t kPrompt = 0x80000000u, kDrafted = 0x40000000u;  // the rest of a word counts
constexpr int kTreeList = 512;  // drafted tokens of a request, and words of rows' masks, that are held in LDS

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
  constexpr int kVec = 8, kAhead = 2;  // a byte of mask a vector; vectors in flight
  extern __shared__ uint32_t logits_lds[];
  __shared__ int32_t drafted[kCounts ? kTreeList : 1];
  __shared__ uint64_t paths[kCounts ? kTreeList : 1];
  const aspire_adjust_logits_args& a = p.a;
  const int chunk = 1 << p.chunk_log2;
  uint32_t* const counts = logits_lds;
  float* const bias = reinterpret_cast<float*>(logits_lds + (kCounts ? chunk : 0));
  const int b = blockIdx.y, v0 = blockIdx.x << p.chunk_log2, width = min(chunk, a.vocab - v0);
  const uint32_t token0 = uint32_t(a.vocab_start) + v0;  // the chunk's first token; its last one is below 2^31
  int first = b, end = b + 1;
  if (a.qo_indptr != nullptr) {
    first = max(a.qo_indptr[b], 0);
    end = min(a.qo_indptr[b + 1], a.tokens);
  }
  const int n = end - first;
  // this workgroup's rows
  const int row0 = first + int(int64_t(max(n, 0)) * blockIdx.z / p.row_parts);
  const int row1 = first + int(int64_t(max(n, 0)) * (blockIdx.z + 1) / p.row_parts);
  if (row0 >= row1) return;

  // Item i: vector i % per of row row0 + i / per. The last vector of the vocabulary may be short.
  const int per_log2 = p.chunk_log2 - 3, per = 1 << per_log2;
  const int64_t items = int64_t(row1 - row0) << per_log2;
  Vec<R, kVec> x[kAhead];
  uint32_t allowed[kAhead];
  const auto fetch = [&](int64_t i, int u) {
    const int row = row0 + int(i >> per_log2), at = int(i & (per - 1)) * kVec;
    allowed[u] = 255u;
    if (i >= items || at >= width) return;
    const R* const in = static_cast<const R*>(a.logits) + row * a.stride + v0 + at;
    if (at + kVec <= width) {
      x[u] = *reinterpret_cast<const Vec<R, kVec>*>(in);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (e < width - at) x[u].v[e] = in[e];
    }
    if (kMask) {
      const int g = a.grammar_rows != nullptr ? a.grammar_rows[row] : row;
      if (g >= 0 && g < a.num_grammar_rows)
        allowed[u] = reinterpret_cast<const uint8_t*>(a.grammar + g * a.grammar_stride)[(v0 + at) >> 3];
    }
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) fetch(threadIdx.x + u * kLogitThreads, u);

  float repetition = 1.f, inverse = 1.f, presence = 0.f, frequency = 0.f;
  if (kCounts || kBias) {
    for (int i = threadIdx.x * 4; i < chunk; i += kLogitThreads * 4) {
      if (kCounts) *reinterpret_cast<uint4*>(counts + i) = make_uint4(0, 0, 0, 0);
      if (kBias) *reinterpret_cast<float4*>(bias + i) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
  }
  const bool tree = kCounts && a.tree_masks != nullptr;
  const int words = min(a.mask_words, (n + 63) / 64);  // of a row's mask that hold its request's tokens
  const bool listed = int64_t(row1 - row0) * words <= kTreeList;
  if (kCounts) {
    if (a.repetition != nullptr) repetition = a.repetition[b];
    if (a.presence != nullptr) presence = a.presence[b];
    if (a.frequency != nullptr) frequency = a.frequency[b];
    inverse = 1.f / repetition;
    if (a.history != nullptr) {
      const int32_t* const history = a.history + b * a.history_stride;
      const int len = min(a.history_lens[b], a.history_len), told = a.prompt_lens != nullptr ? a.prompt_lens[b] : 0;
      constexpr int kRound = 4;  // 16-byte loads of a thread in flight: one trip to L2 for 4,096 tokens
      const auto count = [&](int32_t token, int i) {
        const uint32_t at = uint32_t(token) - token0;  // negative tokens wrap to beyond the chunk, too
        if (at >= uint32_t(width)) return;
        if (i < told) atomicOr(&counts[at], kPrompt);
        else atomicAdd(&counts[at], 1u);
      };
      int i0 = 0;
      for (; i0 + kRound * 4 * kLogitThreads <= len; i0 += kRound * 4 * kLogitThreads) {
        Vec<int32_t, 4> h[kRound];
#pragma unroll
        for (int u = 0; u < kRound; ++u)
          h[u] = *reinterpret_cast<const Vec<int32_t, 4>*>(history + i0 + (u * kLogitThreads + threadIdx.x) * 4);
#pragma unroll
        for (int u = 0; u < kRound; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) count(h[u].v[e], i0 + (u * kLogitThreads + threadIdx.x) * 4 + e);
      }
      for (; i0 < len; i0 += 8 * kLogitThreads) {
        int32_t h[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int i = i0 + u * kLogitThreads + threadIdx.x;
          h[u] = i < len ? history[i] : -1;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int i = i0 + u * kLogitThreads + threadIdx.x;
          if (i < len) count(h[u], i);
        }
      }
    }
    if (tree) {
      for (int i = threadIdx.x; i < min(n, 64 * a.mask_words); i += kLogitThreads) {
        const int32_t token = a.tree_tokens[first + i];
        if (i < kTreeList) drafted[i] = token;
        const uint32_t at = uint32_t(token) - token0;
        if (at < uint32_t(width)) atomicOr(&counts[at], kDrafted);
      }
      if (listed)
        for (int i = threadIdx.x; i < (row1 - row0) * words; i += kLogitThreads)
          paths[i] = uint64_t(a.tree_masks[(row0 + i / words) * a.mask_stride + i % words]);
    }
  }
  if (kBias) {
    const int last = min(a.bias_indptr[b + 1], a.bias_entries);
    for (int i = max(a.bias_indptr[b], 0) + threadIdx.x; i < last; i += kLogitThreads) {
      const uint32_t at = uint32_t(a.bias_ids[i]) - token0;
      if (at < uint32_t(width)) bias[at] = a.bias_values[i];
    }
  }
  if (kCounts || kBias) __syncthreads();

  // Adds to the words c of this lane's 8 tokens how often the row's path has them: the wave walks the path together, node tokens in
  // lanes, and passes over those outside its 512 tokens from token base on.
  const auto add_path = [&](int row, uint32_t base, uint32_t (&c)[kVec]) {
    const int lane = threadIdx.x & 63;
    for (int w = 0; w < words; ++w) {
      const int i = 64 * w + lane;
      const int32_t token = i >= n ? -1 : i < kTreeList ? drafted[i] : a.tree_tokens[first + i];
      uint64_t bits = listed ? paths[(row - row0) * words + w] : uint64_t(a.tree_masks[row * a.mask_stride + w]);
      bits = (uint64_t(uint32_t(wave_uniform(int(bits >> 32)))) << 32) | uint32_t(wave_uniform(int(uint32_t(bits))));
      if (n - 64 * w < 64) bits &= (uint64_t(1) << (n - 64 * w)) - 1;
      for (; bits != 0; bits &= bits - 1) {
        const uint32_t at = uint32_t(__builtin_amdgcn_readlane(token, __builtin_ctzll(bits))) - base;
        if (at >= 64 * kVec) continue;
#pragma unroll
        for (int e = 0; e < kVec; ++e) c[e] += at == uint32_t(lane * kVec + e) ? 1u : 0u;
      }
    }
  };
  for (int64_t i0 = threadIdx.x; i0 < items; i0 += kAhead * kLogitThreads) {
    Vec<R, kVec> y[kAhead];
    uint32_t now[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) y[u] = x[u], now[u] = allowed[u];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) fetch(i0 + (kAhead + u) * kLogitThreads, u);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t i = i0 + u * kLogitThreads;
      const int row = row0 + int(i >> per_log2), at = int(i & (per - 1)) * kVec;
      const bool live = i < items && at < width;
      float f[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) f[e] = Pack<T>::up(y[u].v[e]);
      if (kCounts) {
        uint4 c0 = make_uint4(0, 0, 0, 0), c1 = c0;
        if (live) c0 = *reinterpret_cast<const uint4*>(counts + at), c1 = *reinterpret_cast<const uint4*>(counts + at + 4);
        uint32_t c[kVec] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
        const uint32_t some = c0.x | c0.y | c0.z | c0.w | c1.x | c1.y | c1.z | c1.w;
        if (tree && __ballot(some & kDrafted)) {  // a wave's vectors are one row's
#pragma unroll
          for (int e = 0; e < kVec; ++e) c[e] &= ~kDrafted;
          add_path(wave_uniform(row), token0 + wave_uniform(at), c);
        }
        if (some != 0) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) {
            const uint32_t written = c[e] & ~kPrompt;
            // (a product by the rounded inverse is off by one rounding more than the quotient)
            const float seen = f[e] * (f[e] > 0.f ? inverse : repetition);
            f[e] = c[e] != 0 ? seen : f[e];
            f[e] = written != 0 ? (f[e] - frequency * float(written)) - presence : f[e];
          }
        }
      }
      if (!live) continue;
      if (kBias) {
        const float4 b0 = *reinterpret_cast<const float4*>(bias + at), b1 = *reinterpret_cast<const float4*>(bias + at + 4);
        f[0] += b0.x, f[1] += b0.y, f[2] += b0.z, f[3] += b0.w;
        f[4] += b1.x, f[5] += b1.y, f[6] += b1.z, f[7] += b1.w;
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        if (kMask) f[e] = (now[u] >> e) & 1 ? f[e] : -__builtin_huge_valf();
        y[u].v[e] = Pack<T>::down(f[e]);
      }
      R* const out = static_cast<R*>(a.out) + row * a.out_stride + v0 + at;
      if (at + kVec <= width) {
        *reinterpret_cast<Vec<R, kVec>*>(out) = y[u];
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (e < width - at) out[e] = y[u].v[e];
      }
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
  ASPIRE_CHECK_ARG(a->vocab_start >= 0 && a->vocab_start + a->vocab <= (int64_t(1) << 31), "tokens past 2^31");
  if (a->tokens == 0 || a->vocab == 0 || a->requests == 0) return ASPIRE_OK;
  ASPIRE_CHECK_ARG(a->logits && a->out, "null logits");
  ASPIRE_CHECK_ARG(a->qo_indptr || a->requests <= a->tokens, "a request a row, and fewer rows");
  ASPIRE_CHECK_ARG(!a->history || a->history_lens, "a history needs its lengths");
  ASPIRE_CHECK_ARG(!a->tree_masks == !a->tree_tokens, "tree_tokens and tree_masks go together");
  ASPIRE_CHECK_ARG(!a->tree_masks || a->qo_indptr, "trees need qo_indptr");
  ASPIRE_CHECK_ARG(!a->bias_indptr || a->bias_entries == 0 || (a->bias_ids && a->bias_values), "null biases");
  const bool counts = (a->history || a->tree_masks) && (a->repetition || a->presence || a->frequency);
  const bool bias = a->bias_indptr != nullptr && a->bias_entries > 0;
  // Chunks of 8,192 tokens, shorter while that leaves fewer than two workgroups a CU; then a request's rows are shared by several, four
  // rows or more each, up to eight workgroups a CU. (A history is counted once a workgroup; without enough of them too few loads are
  // in flight: 16 trees of 1 to 24 tokens over 128,257 took 68 us on 256 workgroups.)
  LogitsParams p{*a, 13, 1};
  const auto chunks = [&] { return (int64_t(a->vocab) + (1 << p.chunk_log2) - 1) >> p.chunk_log2; };
  while (p.chunk_log2 > 10 && chunks() * a->requests < 512) --p.chunk_log2;
  const int64_t wgs = chunks() * a->requests, mean = a->qo_indptr ? a->tokens / a->requests : 1;
  p.row_parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({mean / 4, 2048 / wgs, 65535})));
  ASPIRE_CHECK_ARG(chunks() <= (1 << 24) / a->requests, "vocabulary times requests too large");
  const dim3 grid(static_cast<uint32_t>(chunks()), a->requests, p.row_parts);
  const int lds = (4 << p.chunk_log2) * ((counts ? 1 : 0) + (bias ? 1 : 0));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == 0) launch_logits<Bf16>(p, counts, bias, grid, lds, s);
  else if (a->dtype == 1) launch_logits<Fp16>(p, counts, bias, grid, lds, s);
  else launch_logits<float>(p, counts, bias, grid, lds, s);
  ASPIRE_CHECK_LAUNCH();
  return ASPIRE_OK;
}
