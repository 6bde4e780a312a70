// Products with 4-bit weights: y[m, n] = sum_k x[m, k] s[n, g(k)] (c[n, k] - z[n, g(k)]), codes c of 4 bits,
// a 16-bit scale s and a whole-numbered zero point z (8 without) for each group of 32, 64 or 128 k.
//
// Nothing is rounded on the way: a code becomes the 16-bit float kOffset + c (exact: bf16 128 + c, fp16 1024 + c)
// by putting its bits into the constant's mantissa, MFMAs sum it against x in fp32, and what the offset adds is
// taken off for each group before the scale goes on,
//     y += s (sum (kOffset + c) x - (kOffset + z) sum x),
// the sums of x from one more MFMA with ones in the weights' place. fp16 has packed subtraction, so there
// kOffset + z comes off the weights themselves, exactly, and no sums of x are needed.
//
// Weights are laid out once (aspire_int4_pack's order): 16 rows x 128 k make a block of 1 KiB in which lane l of a
// wave finds its 32 codes (row l % 16, and for each 32 k the 8 from 8 (l / 16) on) in one 16-byte load; blocks of 16
// rows follow each other along k. A word's nibbles are ordered so that shifts by 0, 4, 8, 12 leave neighbours in
// the low and high half.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace aspire {
namespace {

struct Int4Params {
  const uint16_t* x;
  int64_t x_st;
  const uint4* w;
  const uint16_t* scales;    // [groups][n_pad]
  const uint8_t* zeros;      // [groups][n_pad], or null: 8
  uint16_t* out;
  int64_t o_st;
  int32_t rows, n, n_pad, k, blocks;   // n: output columns; blocks: of 128 k
  int32_t up_tile;           // swiglu: 16-row tile where the up rows begin
  int32_t scale_fp16;
  int32_t wide_out;          // output rows take 8-byte stores
};

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

struct Bf16 {
  static constexpr uint32_t kMagic = 0x43004300u;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint16_t narrow(float f) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f)); }
};
struct Fp16 {
  static constexpr uint32_t kMagic = 0x64006400u;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint16_t narrow(float f) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f)); }
};

// 8 codes as 8 values kOffset + c, in k's order.
template <class T>
__device__ __forceinline__ u32x4 spread(uint32_t w) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = ((w >> (4 * i)) & 0x000f000fu) | T::kMagic;
  return v;
}

__device__ __forceinline__ float scale_of(uint32_t bits, int fp16) {
  return fp16 ? float(__builtin_bit_cast(_Float16, uint16_t(bits))) : __uint_as_float(bits << 16);
}

constexpr int kWaves = 8;

// A workgroup takes TN tiles of 16 weight rows and TM of 16 rows of x; its waves take the blocks of 128 k in
// turn and add up through LDS at the end, in a fixed order.
template <class T, int G, int TM, int TN, bool kSwiglu>
__global__ __launch_bounds__(64 * kWaves) void int4_stream_kernel(Int4Params p) {
  constexpr int kParts = 128 / G;   // groups of a block
  constexpr bool kIsBf16 = std::is_same<T, Bf16>::value;
  __shared__ float4 sums[kWaves][TM * TN][64];
  const int lane = threadIdx.x & 63;
  const int wave = wave_uniform(threadIdx.x >> 6);
  const int r = lane & 15, grp = lane >> 4;
  const int64_t m0 = int64_t(blockIdx.y) * (16 * TM);
  int tile[TN];                     // 16-row tiles of the weights
#pragma unroll
  for (int j = 0; j < TN; ++j)
    tile[j] = kSwiglu ? (j < TN / 2 ? blockIdx.x * (TN / 2) + j : p.up_tile + blockIdx.x * (TN / 2) + j - TN / 2)
                      : blockIdx.x * TN + j;
  const int last_tile = p.n_pad / 16 - 1;
  const uint16_t* xrow[TM];
  bool live[TM];
#pragma unroll
  for (int t = 0; t < TM; ++t) {
    const int64_t m = m0 + t * 16 + r;
    live[t] = m < p.rows;
    xrow[t] = p.x + (live[t] ? m : 0) * p.x_st + 8 * grp;
  }
  f32x4 acc[TM][TN];
#pragma unroll
  for (int t = 0; t < TM; ++t)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const f32x4 none = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int kb = wave; kb < p.blocks; kb += kWaves) {
    uint4 w[TN];
    uint2 sc[TN][kParts];
    uint32_t zp[TN][kParts];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int at = min(tile[j], last_tile);
      w[j] = p.w[(int64_t(at) * p.blocks + kb) * 64 + lane];
#pragma unroll
      for (int g = 0; g < kParts; ++g) {
        const int64_t row = (int64_t(kb) * kParts + g) * p.n_pad + at * 16;
        sc[j][g] = *reinterpret_cast<const uint2*>(p.scales + row + 4 * grp);
        zp[j][g] = 0x08080808u;
        if (p.zeros) zp[j][g] = kIsBf16 ? *reinterpret_cast<const uint32_t*>(p.zeros + row + 4 * grp) : p.zeros[row + r];
      }
    }
    u32x4 xs[TM][4];
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        xs[t][c] = u32x4{0, 0, 0, 0};
        const int k = kb * 128 + c * 32;
        if (live[t] && k < p.k) xs[t][c] = *reinterpret_cast<const u32x4*>(xrow[t] + k);
      }
#pragma unroll
    for (int g = 0; g < kParts; ++g) {
      f32x4 part[TM][TN], ones[TM];
#pragma unroll
      for (int t = 0; t < TM; ++t) {
        ones[t] = none;
#pragma unroll
        for (int j = 0; j < TN; ++j) part[t][j] = none;
      }
#pragma unroll
      for (int c = g * (4 / kParts); c < (g + 1) * (4 / kParts); ++c) {
        if (kIsBf16) {
          constexpr uint32_t one = 0x3f803f80u;
#pragma unroll
          for (int t = 0; t < TM; ++t) ones[t] = T::mfma(u32x4{one, one, one, one}, xs[t][c], ones[t]);
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const uint32_t word = c == 0 ? w[j].x : c == 1 ? w[j].y : c == 2 ? w[j].z : w[j].w;
          u32x4 a = spread<T>(word);
          if (!kIsBf16) {
            const uint32_t off = 0x6400u | (zp[j][g] & 15u);
            const f16x2 z = __builtin_bit_cast(f16x2, off | off << 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, uint32_t(a[i])) - z);
          }
#pragma unroll
          for (int t = 0; t < TM; ++t) part[t][j] = T::mfma(a, xs[t][c], part[t][j]);
        }
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const uint32_t sw[2] = {sc[j][g].x, sc[j][g].y};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float s = scale_of((sw[i / 2] >> (16 * (i & 1))) & 0xffffu, p.scale_fp16);
          const float z = 128.f + float((zp[j][g] >> (8 * i)) & 0xffu);
#pragma unroll
          for (int t = 0; t < TM; ++t)
            acc[t][j][i] = fmaf(s, kIsBf16 ? fmaf(-z, ones[t][i], part[t][j][i]) : part[t][j][i], acc[t][j][i]);
        }
      }
    }
  }

#pragma unroll
  for (int t = 0; t < TM; ++t)
#pragma unroll
    for (int j = 0; j < TN; ++j)
      sums[wave][t * TN + j][lane] = make_float4(acc[t][j][0], acc[t][j][1], acc[t][j][2], acc[t][j][3]);
  __syncthreads();
  constexpr int kOuts = kSwiglu ? TN / 2 : TN;
  for (int i = wave; i < TM * kOuts; i += kWaves) {
    const int t = i / kOuts, j = i % kOuts;
    const auto total = [&](int tj) {
      float4 v = sums[0][tj][lane];
#pragma unroll
      for (int q = 1; q < kWaves; ++q) {
        const float4 u = sums[q][tj][lane];
        v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
      }
      return v;
    };
    float4 v = total(t * TN + j);
    if (kSwiglu) {
      const float4 u = total(t * TN + j + TN / 2);
      v.x = v.x / (1.f + expf(-v.x)) * u.x;
      v.y = v.y / (1.f + expf(-v.y)) * u.y;
      v.z = v.z / (1.f + expf(-v.z)) * u.z;
      v.w = v.w / (1.f + expf(-v.w)) * u.w;
    }
    const int64_t m = m0 + t * 16 + r;
    const int col = tile[j] * 16 + 4 * grp;
    if (m >= p.rows) continue;
    uint16_t* to = p.out + m * p.o_st + col;
    const uint16_t o[4] = {T::narrow(v.x), T::narrow(v.y), T::narrow(v.z), T::narrow(v.w)};
    if (p.wide_out && col + 4 <= p.n) {
      *reinterpret_cast<uint2*>(to) = make_uint2(o[0] | uint32_t(o[1]) << 16, o[2] | uint32_t(o[3]) << 16);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < p.n) to[e] = o[e];
    }
  }
}

template <class T, int G, int TM, bool kSwiglu>
void launch(const Int4Params& p, hipStream_t s) {
  constexpr int TN = kSwiglu ? 2 : 1, kOuts = kSwiglu ? TN / 2 : TN;
  const dim3 grid((p.n + 16 * kOuts - 1) / (16 * kOuts), (p.rows + 16 * TM - 1) / (16 * TM));
  hipLaunchKernelGGL((int4_stream_kernel<T, G, TM, TN, kSwiglu>), grid, dim3(64 * kWaves), 0, s, p);
}

template <class T, int G>
void pick(const Int4Params& p, bool swiglu, hipStream_t s) {
  const auto rows = [&](auto sw) {
    if (p.rows <= 16) launch<T, G, 1, sw()>(p, s);
    else if (p.rows <= 32) launch<T, G, 2, sw()>(p, s);
    else launch<T, G, 4, sw()>(p, s);
  };
  if (swiglu) rows(std::true_type{});
  else rows(std::false_type{});
}

template <class T>
void pick_group(const Int4Params& p, int group, bool swiglu, hipStream_t s) {
  if (group == 32) pick<T, 32>(p, swiglu, s);
  else if (group == 64) pick<T, 64>(p, swiglu, s);
  else pick<T, 128>(p, swiglu, s);
}

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace
}  // namespace aspire

extern "C" int aspire_linear_int4(const aspire_int4_args* a, void* stream) {
  using namespace aspire;
  ASPIRE_CHECK_ARG(a != nullptr, "null arguments");
  ASPIRE_CHECK_ARG(a->rows >= 0 && a->n >= 0 && a->k > 0, "bad sizes");
  ASPIRE_CHECK_ARG(a->rows <= (1 << 22) - 64, "at most 4,194,240 rows");
  ASPIRE_CHECK_ARG(a->group == 32 || a->group == 64 || a->group == 128, "groups of 32, 64 or 128");
  ASPIRE_CHECK_ARG(a->k % a->group == 0, "k must be a multiple of the group");
  ASPIRE_CHECK_ARG(!a->swiglu || a->n % 32 == 0, "swiglu needs whole 16-row tiles of gate and up rows");
  if (a->rows == 0 || a->n == 0) return ASPIRE_OK;
  ASPIRE_CHECK_ARG(a->x && a->weights && a->scales && a->out, "null pointer");
  ASPIRE_CHECK_ARG(aligned(a->x, 16) && a->x_stride % 8 == 0 && a->x_stride >= a->k, "x rows must be 16-byte aligned");
  ASPIRE_CHECK_ARG(aligned(a->weights, 16) && aligned(a->scales, 16) && aligned(a->zeros, 16),
                   "weights, scales and zeros must be 16-byte aligned");
  const int outs = a->swiglu ? a->n / 2 : a->n;
  ASPIRE_CHECK_ARG(a->out_stride >= outs, "out rows must hold the output columns");
  Int4Params p{};
  p.x = static_cast<const uint16_t*>(a->x);
  p.x_st = a->x_stride;
  p.w = static_cast<const uint4*>(a->weights);
  p.scales = static_cast<const uint16_t*>(a->scales);
  p.zeros = static_cast<const uint8_t*>(a->zeros);
  p.out = static_cast<uint16_t*>(a->out);
  p.o_st = a->out_stride;
  p.rows = a->rows;
  p.n = outs;
  p.n_pad = (a->n + 15) / 16 * 16;
  p.k = a->k;
  p.blocks = (a->k + 127) / 128;
  p.up_tile = outs / 16;
  p.scale_fp16 = a->scales_fp16;
  p.wide_out = aligned(a->out, 8) && a->out_stride % 4 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->fp16) pick_group<Fp16>(p, a->group, a->swiglu != 0, s);
  else pick_group<Bf16>(p, a->group, a->swiglu != 0, s);
  ASPIRE_CHECK_LAUNCH();
  return ASPIRE_OK;
}
