// Penalties for repeated tokens, biases and grammar masks on logits (gfx950).
//
// A workgroup takes one chunk of the vocabulary for one request (or some of its rows). It counts the request's history tokens of
// the chunk in LDS (a 32-bit word a token: occurrences in the output, one bit for the prompt's, one for tokens that the request's
// tree drafts) and lays the chunk's biases beside them, while its first logits are on their way; then the chunk of every row
// streams through: vectors of 8 logits, their words from LDS, a byte of the mask, one rounding, the next row's in flight
// meanwhile. (Counts and biases kept in registers over the rows take 121 VGPRs, half the waves, and as long.) A token that the
// tree drafts is counted on a row's own path where it is met. Chunks of low tokens, which histories and trees meet most, start first.
// HBM bounds it at batch sizes (logits once in, once out, and an eighth of a byte of mask a token); history is
// read once a chunk, from L2. Measured: 64 x 151,936 bf16 logits with histories and masks 15 us = 2.8 TB/s, the history's chain (lengths,
// tokens, LDS) before the first store; 16 trees of up to 24 tokens over 128,257 with 20,000 tokens of history and 100 biases 46 us = 3.1
// TB/s, of which counting takes its part and rows whose trees draft tokens of the chunk theirs; one row of 32,000 4.3 us, latency.
#include <algorithm>

#include "common.h"

namespace aspire {
namespace {

struct LogitsParams {
  aspire_adjust_logits_args a;
  int32_t row_parts;  // workgroups that share a request's rows of a chunk
};

constexpr int kLogitThreads = 512;
constexpr int kVec = 8;          // logits of a vector: a byte of mask
constexpr uint32_t kPrompt = 0x80000000u, kDrafted = 0x40000000u;  // the rest of a word counts
constexpr int kTreeList = 512;   // drafted tokens of a request, and words of rows' masks, that are held in LDS

template <typename T> struct Pack;
struct Bf16 {};
struct Fp16 {};
template <> struct Pack<Bf16> {
  typedef uint16_t raw;
  static constexpr bool kLean = true;  // fits in 64 registers with two vectors a thread
  static __device__ __forceinline__ float up(raw x) { return __uint_as_float(uint32_t(x) << 16); }
  static __device__ __forceinline__ raw down(float x) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x)); }
};
template <> struct Pack<Fp16> {
  typedef uint16_t raw;
  static constexpr bool kLean = false;
  static __device__ __forceinline__ float up(raw x) { return float(__builtin_bit_cast(_Float16, x)); }
  static __device__ __forceinline__ raw down(float x) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x)); }
};
template <> struct Pack<float> {
  typedef float raw;
  static constexpr bool kLean = false;
  static __device__ __forceinline__ float up(raw x) { return x; }
  static __device__ __forceinline__ raw down(float x) { return x; }
};

// n values at any 2- or 4-byte aligned place, in one access
template <typename R, int n> struct __attribute__((packed, aligned(sizeof(R)))) Vec { R v[n]; };

// 1 / r = (high + low) scale, scale a power of two: with m = |r| scale, fma(x, high, x low) is x / m within half a step and 2^-46, and times
// scale x / r (rounded once more where that lies below the normal numbers). m is a normal number: as r is from 2^-60 to 2^60, past that 1 to
// 2^68 and below 2^-60 to 2^-30, so that x / m only overflows where x / r does, and holds a small x's bits. high lies towards zero; low has
// its sign and is not 0, so that infinite x stay so.
// With two vectors a thread its three values leave the registers and each penalised logit is divided. 16 trees over 128,257 logits (one
// vector) and 64 requests over 151,936 (two), us in a graph: one product by a rounded reciprocal 51.6 and 19.9; the parts 52.4 and 22.0;
// divisions 56.6 and 20.6.
__device__ __forceinline__ void reciprocal(float r, float& high, float& low, float& scale) {
  float m = fabsf(r);
  scale = m > 0x1p60f ? 0x1p-60f : m >= 0x1p-60f ? 1.f : m >= 0x1p-90f ? 0x1p30f : m >= 0x1p-120f ? 0x1p60f : 0x1p90f;
  m *= scale;
  high = __builtin_amdgcn_rcpf(m);  // within a step: what it lacks is low's
  if (fmaf(-m, high, 1.f) < 0.f) high = __int_as_float(__float_as_int(high) - 2);
  low = m < __builtin_huge_valf() ? fmaxf(fmaf(-m, high, 1.f) * high, 0x1p-149f) : 0.f;
  high = copysignf(high, r), low = copysignf(low, r);
}

// A workgroup's chunk is kJ vectors a thread.
template <typename T, int kJ, bool kCounts, bool kBias, bool kMask>
__global__ __launch_bounds__(kLogitThreads, kJ == 1 || Pack<T>::kLean ? 8 : 6) void adjust_logits_kernel(LogitsParams p) {
  typedef typename Pack<T>::raw R;
  constexpr int kChunk = kJ * kVec * kLogitThreads;
  extern __shared__ uint4 logits_lds[];
  uint32_t* const counts = reinterpret_cast<uint32_t*>(logits_lds);
  float* const bias = reinterpret_cast<float*>(counts + (kCounts ? kChunk : 0));
  uint64_t* const paths = reinterpret_cast<uint64_t*>(bias + (kBias ? kChunk : 0));  // there only for trees
  int32_t* const drafted = reinterpret_cast<int32_t*>(paths + kTreeList);
  const aspire_adjust_logits_args& a = p.a;
  const int nth = wave_uniform(int(blockIdx.x / uint32_t(a.requests))), b = int(blockIdx.x) - nth * a.requests, v0 = nth * kChunk, width = min(kChunk, a.vocab - v0);
  const uint32_t token0 = uint32_t(a.vocab_start) + v0;  // the chunk's first token; its last one is below 2^31
  int first = b, end = b + 1;
  if (a.qo_indptr != nullptr) {
    first = max(a.qo_indptr[b], 0);
    end = min(a.qo_indptr[b + 1], a.tokens);
  }
  const int n = max(end - first, 0);
  // this workgroup's rows
  const int row0 = first + int(int64_t(n) * blockIdx.y / p.row_parts), row1 = first + int(int64_t(n) * (blockIdx.y + 1) / p.row_parts);
  if (row0 >= row1) return;

  const int whole = width / kVec;  // whole vectors; the vocabulary's last logits come one by one, to the first threads
  const int tail = whole * kVec + int(threadIdx.x);
  Vec<R, kVec> x[kJ];
  uint32_t allowed[kJ];
  const auto mask_of = [&](int row) -> const uint8_t* {
    const int g = !kMask ? -1 : a.grammar_rows != nullptr ? a.grammar_rows[row] : row;
    return g >= 0 && g < a.num_grammar_rows ? reinterpret_cast<const uint8_t*>(a.grammar + g * a.grammar_stride) + (v0 >> 3) : nullptr;
  };
  const auto fetch = [&](int row) {
    const R* const in = static_cast<const R*>(a.logits) + row * a.stride + v0;
    const uint8_t* const mask = mask_of(row);
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      const int k = j * kLogitThreads + threadIdx.x;
      if (k >= whole) break;
      x[j] = *reinterpret_cast<const Vec<R, kVec>*>(in + k * kVec);
      allowed[j] = kMask && mask != nullptr ? mask[k] : 255u;
    }
  };
  fetch(row0);

  if (kCounts || kBias) {
    for (int i = threadIdx.x; i < (kChunk / 4) * ((kCounts ? 1 : 0) + (kBias ? 1 : 0)); i += kLogitThreads) {
      const uint32_t none = kBias && i >= (kCounts ? kChunk / 4 : 0) ? 0x80000000u : 0u;  // a bias of -0 leaves every logit as it is
      logits_lds[i] = make_uint4(none, none, none, none);
    }
    __syncthreads();
  }
  const bool tree = kCounts && a.tree_masks != nullptr;
  const int words = min(a.mask_words, (n + 63) / 64);  // of a row's mask that hold its request's tokens
  const bool listed = int64_t(row1 - row0) * words <= kTreeList;
  float repetition = 1.f, presence = 0.f, frequency = 0.f;
  if (kCounts) {
    if (a.repetition != nullptr) repetition = a.repetition[b];
    if (a.presence != nullptr) presence = a.presence[b];
    if (a.frequency != nullptr) frequency = a.frequency[b];
    if (a.history != nullptr) {
      const int32_t* const history = a.history + b * a.history_stride;
      const int len = min(a.history_lens[b], a.history_len), told = a.prompt_lens != nullptr ? a.prompt_lens[b] : 0;
      constexpr int kRound = 4;  // 16-byte loads of a thread in flight: one trip to L2 for 8,192 tokens
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
          h[u] = i < len ? history[i] : -1;  // of no column
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) count(h[u], i0 + u * kLogitThreads + threadIdx.x);
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
  float high = 1.f, low = 0.f, scale = 1.f;
  if (kCounts && kJ == 1) reciprocal(repetition, high, low, scale);
  if (kBias) {
    const int last = min(a.bias_indptr[b + 1], a.bias_entries);
    for (int i = max(a.bias_indptr[b], 0) + threadIdx.x; i < last; i += kLogitThreads) {
      const uint32_t at = uint32_t(a.bias_ids[i]) - token0;
      if (at < uint32_t(width)) bias[at] = a.bias_values[i];
    }
  }
  if (kCounts || kBias) __syncthreads();

  // the bits of word w of a row's path, and the drafted token of a node
  const auto path_word = [&](int row, int w) {
    const uint64_t bits = listed ? paths[(row - row0) * words + w] : uint64_t(a.tree_masks[row * a.mask_stride + w]);
    return n - 64 * w < 64 ? bits & ((uint64_t(1) << (n - 64 * w)) - 1) : bits;
  };
  const auto node_token = [&](int i) { return i < kTreeList ? drafted[i] : a.tree_tokens[first + i]; };
  // Adds to the words c of this lane's 8 tokens how often the row's path has them: the wave walks the path together, node tokens in
  // lanes, and passes over those outside its 512 tokens from token base on.
  const auto add_path = [&](int row, uint32_t base, uint32_t (&c)[kVec]) {
    const int lane = threadIdx.x & 63;
    for (int w = 0; w < words; ++w) {
      const int32_t token = 64 * w + lane < n ? node_token(64 * w + lane) : -1;
      uint64_t bits = path_word(row, w);
      bits = (uint64_t(uint32_t(wave_uniform(int(bits >> 32)))) << 32) | uint32_t(wave_uniform(int(uint32_t(bits))));
      for (; bits != 0; bits &= bits - 1) {
        const uint32_t at = uint32_t(__builtin_amdgcn_readlane(token, __builtin_ctzll(bits))) - base;
        if (at >= 64 * kVec) continue;
#pragma unroll
        for (int e = 0; e < kVec; ++e) c[e] += at == uint32_t(lane * kVec + e) ? 1u : 0u;
      }
    }
  };
  const auto penalty = [&](float f, uint32_t c) {
    const uint32_t written = c & ~kPrompt;
    if constexpr (kJ == 1) {
      const float seen = f > 0.f ? fmaf(f, high, f * low) * scale : f * repetition;
      f = c != 0 ? seen : f;
    } else if (c != 0) {
      f = f > 0.f ? f / repetition : f * repetition;
    }
    return written != 0 ? (f - frequency * float(written)) - presence : f;
  };
  for (int row = row0; row < row1; ++row) {
    R* const out = static_cast<R*>(a.out) + row * a.out_stride + v0;
    Vec<R, kVec> y[kJ];
    uint32_t now[kJ];
#pragma unroll
    for (int j = 0; j < kJ; ++j) y[j] = x[j], now[j] = allowed[j];
    if (row + 1 < row1) fetch(row + 1);
#pragma unroll
    for (int j = 0; j < kJ; ++j) {
      const int k = j * kLogitThreads + threadIdx.x;
      if (k - int(threadIdx.x & 63) >= whole) break;  // of the whole wave
      float f[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) f[e] = Pack<T>::up(y[j].v[e]);
      const int at = k * kVec;
      if (kCounts) {
        const uint4 c0 = *reinterpret_cast<const uint4*>(counts + at), c1 = *reinterpret_cast<const uint4*>(counts + at + 4);
        uint32_t c[kVec] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
        const uint32_t some = c0.x | c0.y | c0.z | c0.w | c1.x | c1.y | c1.z | c1.w;
        if (tree && __ballot((some & kDrafted) != 0)) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) c[e] &= ~kDrafted;
          add_path(row, token0 + wave_uniform(at), c);
        }
        if (some != 0) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) f[e] = penalty(f[e], c[e]);
        }
      }
      if (kBias) {
        const float4 b0 = *reinterpret_cast<const float4*>(bias + at), b1 = *reinterpret_cast<const float4*>(bias + at + 4);
        f[0] += b0.x, f[1] += b0.y, f[2] += b0.z, f[3] += b0.w;
        f[4] += b1.x, f[5] += b1.y, f[6] += b1.z, f[7] += b1.w;
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        if (kMask) f[e] = (now[j] >> e) & 1 ? f[e] : -__builtin_huge_valf();
        y[j].v[e] = Pack<T>::down(f[e]);
      }
      if (k < whole) *reinterpret_cast<Vec<R, kVec>*>(out + at) = y[j];
    }
    if (tail < width) {  // up to 7 threads
      float f = Pack<T>::up((static_cast<const R*>(a.logits) + row * a.stride + v0)[tail]);
      if (kCounts) {
        uint32_t c = counts[tail];
        if (c & kDrafted) {
          c &= ~kDrafted;
          for (int w = 0; w < words; ++w)
            for (uint64_t bits = path_word(row, w); bits != 0; bits &= bits - 1)
              c += uint32_t(node_token(64 * w + __builtin_ctzll(bits))) == token0 + tail ? 1u : 0u;
        }
        f = penalty(f, c);
      }
      if (kBias) f += bias[tail];
      const uint8_t* const mask = mask_of(row);
      if (kMask && mask != nullptr && !((mask[tail >> 3] >> (tail & 7)) & 1)) f = -__builtin_huge_valf();
      out[tail] = Pack<T>::down(f);
    }
  }
}

struct LogitsLaunch {
  int vectors;  // of a thread
  bool counts, bias;
  dim3 grid;
  int lds;
  hipStream_t stream;
};
template <typename T, int kJ, bool kCounts, bool kBias>
void launch_mask(const LogitsParams& p, const LogitsLaunch& l) {
  if (p.a.grammar != nullptr) adjust_logits_kernel<T, kJ, kCounts, kBias, true><<<l.grid, kLogitThreads, l.lds, l.stream>>>(p);
  else adjust_logits_kernel<T, kJ, kCounts, kBias, false><<<l.grid, kLogitThreads, l.lds, l.stream>>>(p);
}
template <typename T, int kJ>
void launch_parts(const LogitsParams& p, const LogitsLaunch& l) {
  if (l.counts && l.bias) launch_mask<T, kJ, true, true>(p, l);
  else if (l.counts) launch_mask<T, kJ, true, false>(p, l);
  else if (l.bias) launch_mask<T, kJ, false, true>(p, l);
  else launch_mask<T, kJ, false, false>(p, l);
}
template <typename T>
void launch_logits(const LogitsParams& p, const LogitsLaunch& l) {
  if (l.vectors == 2) launch_parts<T, 2>(p, l);
  else launch_parts<T, 1>(p, l);
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
  // Chunks of 8,192 tokens, or 4,096 with two tables in LDS (four workgroups a CU either way; three with 8,192 fp16 or fp32 logits, whose
  // registers leave six waves a SIMD) or while longer ones leave fewer than two workgroups a CU; then a request's rows are shared by
  // several, eight rows or more each, up to eight workgroups a CU (a history is counted once a workgroup: 16 trees of up to 24 tokens,
  // 128,257 logits, took 54 us so, 59 with four rows or more each, in one build).
  LogitsLaunch l{counts && bias ? 1 : 2, counts, bias, dim3(), 0, static_cast<hipStream_t>(stream)};
  const auto chunk = [&] { return l.vectors * kVec * kLogitThreads; };
  const auto chunks = [&] { return (int64_t(a->vocab) + chunk() - 1) / chunk(); };
  if (chunks() * a->requests < 512) l.vectors = 1;
  const int64_t wgs = chunks() * a->requests, mean = a->qo_indptr ? a->tokens / a->requests : 1;
  LogitsParams p{*a, static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({mean / 8, 2048 / wgs, 65535})))};
  // (a launch has less than 2^32 threads)
  ASPIRE_CHECK_ARG(wgs < (int64_t(1) << 32) / kLogitThreads, "vocabulary times requests too large");
  l.grid = dim3(static_cast<uint32_t>(wgs), p.row_parts);
  l.lds = chunk() * 4 * ((counts ? 1 : 0) + (bias ? 1 : 0)) + (counts && a->tree_masks ? kTreeList * 12 : 0);
  if (a->dtype == 0) launch_logits<Bf16>(p, l);
  else if (a->dtype == 1) launch_logits<Fp16>(p, l);
  else launch_logits<float>(p, l);
  ASPIRE_CHECK_LAUNCH();
  return ASPIRE_OK;
}
