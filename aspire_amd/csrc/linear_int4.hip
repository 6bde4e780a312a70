// Products with 4-bit weights: y[m, n] = sum_k x[m, k] s[n, g(k)] (c[n, k] - z[n, g(k)]), codes c of 4 bits,
// a 16-bit scale s and a whole-numbered zero point z (8 without) for each group of 32, 64 or 128 k.
//
// Weights are never rounded. fp16: a code's bits in the mantissa of 1024 give 1024 + c, and a packed subtraction of 1024 + z
// leaves c - z exactly. bf16 has no packed arithmetic, but the bits of 192 + d are those of 192 (0x4340) plus d for every
// d = c - z from -15 to 15 (one binade, steps of 1), so bytes 0x40 + d, four to an addition, get their upper byte 0x43 from a
// byte permutation, and the sum over a group starts from -192 sum x, which one MFMA with -192 in the weights' place gives for all of them:
//     part = sum (192 + d) x - 192 sum x (fp32),  y += s part  for each group.
// The offset costs the sums of a group up to 5 of fp32's 24 bits, which bf16 outputs have to spare: of 12 x 24,576 x 4,096 with swiglu 0.4% are
// rounded to another side than plain fp32 sums are, and both are 0.00167 off the exact values (2-norm).
//
// Weights are laid out once (aspire_hip.h): 16 rows x 128 k make a block of 1 KiB in which lane l of a
// wave finds its 32 codes (row l % 16, and for each 32 k the 8 from 8 (l / 16) on) in one 16-byte load; blocks of 16
// rows follow each other along k. A word's nibbles are ordered so that shifts by 0, 4, 8, 12 leave neighbours in
// the low and high half.
//
// Bound by the weights' stream up to 16 rows (151,936 x 4,096: 4.4 TB/s, where a mere read runs at 7.3; smaller ones start up for
// some 5 us), above by the steps of the tiles, whose matrix cores are busy 36 to 39% of the time and the VALU beside them 34 to 46%, hardly
// at once. us on MI355X, bf16, groups of 128 with zero points, weights cold / the bf16 products of linear.hip (slabs whose sum
// is their consumer's; whole for the two wide ones) / torch's (swiglu with silu_mul behind it):
//   rows     4,096 x 4,096   24,576 x 4,096 + swiglu    4,096 x 12,288      151,936 x 4,096
//      1     5.8 / 7.9 / 16      17 / 39 / 48           13.8 / 17.6 / 21     78 / 202 / 244
//     12     7.6 / 8.1 / 16      17 / 37 / 47           15.7 / 17.6 / 22     74 / 200 / 255 (16 rows)
//     48    14.4 / 10.0 / 14     31 / 43 / 48           20.9 / 20.7 / 32    124 / 214 / 260
//    208    25.5 / 18.1 / 22     57 / 60 / 68           35.4 / 39.1 / 51    318 / 357 / 330
//  2,048      67 /  -   / 60    384 /  - / 317           188 /   -  / 177
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace aspire {
namespace {

struct Int4Params {
  const uint16_t* x;
  int64_t x_st;
  const uint4* w;
  const uint8_t* scales;     // [tiles][blocks][4][128 / group][4] 16-bit floats
  const uint8_t* zeros;      // [tiles][blocks][16][128 / group] bytes, or null: 8
  uint16_t* out;
  int64_t o_st;
  int32_t rows, n, n_pad, k, blocks;   // n: output columns; blocks: of 128 k
  int32_t swiglu;            // the up rows' first 16-row tile is n / 16
  int32_t wide_out;          // output rows take 8-byte stores
  int32_t splits;            // of the blocks along k
  float* partials;           // [splits][rows][n_pad]
};

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

// A type's MFMA, and 8 codes as its weights in k's order, with what a row's zero point makes of them (`Row`).
struct Bf16 {
  static constexpr bool kOffset = true;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint16_t narrow(float f) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f)); }
  static __device__ __forceinline__ float low(uint32_t v) { return __uint_as_float(v << 16); }
  static __device__ __forceinline__ float high(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
  typedef uint32_t Row;             // 0x40 - z in each byte
  static __device__ __forceinline__ Row row(uint32_t z) { return 0x40404040u - z * 0x01010101u; }
  // bytes 0x40 + c - z, then 0x43 above each
  static __device__ __forceinline__ u32x4 weights(uint32_t w, Row z) {
    const uint32_t lo = (w & 0x0f0f0f0fu) + z, hi = ((w >> 4) & 0x0f0f0f0fu) + z;
    return u32x4{__builtin_amdgcn_perm(0x43434343u, lo, 0x04020400u), __builtin_amdgcn_perm(0x43434343u, hi, 0x04020400u),
                 __builtin_amdgcn_perm(0x43434343u, lo, 0x04030401u), __builtin_amdgcn_perm(0x43434343u, hi, 0x04030401u)};
  }
};
struct Fp16 {
  static constexpr bool kOffset = false;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint16_t narrow(float f) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f)); }
  static __device__ __forceinline__ float low(uint32_t v) { return float(__builtin_bit_cast(_Float16, uint16_t(v))); }
  static __device__ __forceinline__ float high(uint32_t v) { return float(__builtin_bit_cast(_Float16, uint16_t(v >> 16))); }
  struct Row { f16x2 low, high; };  // -(1024 + z) and -(64 + z), twice
  static __device__ __forceinline__ Row row(uint32_t z) {
    const _Float16 f = static_cast<_Float16>(float(z));
    const _Float16 low = _Float16(-1024) - f, high = _Float16(-64) - f;
    return Row{f16x2{low, low}, f16x2{high, high}};
  }
  // a nibble in bits 4 to 7 makes 1024 + 16 c
  static __device__ __forceinline__ u32x4 weights(uint32_t w, Row z) {
    const f16x2 sixteenth = f16x2{_Float16(0.0625f), _Float16(0.0625f)};
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t b = w >> (8 * i);
      v[2 * i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, (b & 0x000f000fu) | 0x64006400u) + z.low);
      v[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (b & 0x00f000f0u) | 0x64006400u), sixteenth, z.high));
    }
    return v;
  }
};
constexpr uint32_t kMinusOffset = 0xc340c340u;  // -192 twice

__device__ __forceinline__ float silu(float x) { return x / (1.f + expf(-x)); }

// A row's zero points of a block's groups, a byte each.
template <int kParts>
__device__ __forceinline__ uint32_t zero_points(const uint8_t* at) {
  if (kParts == 4) return *reinterpret_cast<const uint32_t*>(at);
  if (kParts == 2) return *reinterpret_cast<const uint16_t*>(at);
  return *at;
}

// 4 neighbouring outputs of a row.
template <class T>
__device__ __forceinline__ void store4(const Int4Params& p, int64_t m, int col, const float* v) {
  uint16_t* to = p.out + m * p.o_st + col;
  const uint16_t o[4] = {T::narrow(v[0]), T::narrow(v[1]), T::narrow(v[2]), T::narrow(v[3])};
  if (p.wide_out && col + 4 <= p.n) {
    *reinterpret_cast<uint2*>(to) = make_uint2(o[0] | uint32_t(o[1]) << 16, o[2] | uint32_t(o[3]) << 16);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < p.n) to[e] = o[e];
  }
}

constexpr int kWaves = 8;
// Blocks of 1 KiB a wave has, and has in flight, of a tile: at most 6, or 8 where that saves the splits and their join (groups
// of 32 have no registers for it).
constexpr int most_ahead(int blocks, int group) { return group > 32 && blocks <= 8 * kWaves ? 8 : 6; }

// Few rows (16 to a blockIdx.z): bound by the weights' stream. A workgroup walks over output tiles of 16 columns (with swiglu over pairs of a
// gate and an up tile), for all of k or the split blockIdx.y of at most 6 or 8 blocks a wave; its waves take the blocks of
// 128 k in turn, keep their x in registers, and add up through LDS, in a fixed order. A block is asked for as soon as
// the one before it in its registers is multiplied, across the ends of tiles (once a tile the compiled loop still waits for all
// of a wave's loads where it has 2 blocks or more: one wait serves the first tile, whose loads go out in another order). kAhead is the
// blocks that a wave has, so that a short k loads none twice: 16 x 24,576 x 1,024 with 1 7.3 us, with 4 14.9; 16 x 24,576 x
// 2,048 with 2 11.4, with 4 16.6. More than 4 leave a CU one workgroup, and are still faster than splits of at most 4 with
// their join: 1 x 4,096 x 6,144 with 6 7.5 us, in two splits 9.2; 16 x 24,576 x 8,192 with 8 32.0, in two 34.6; 16 x 4,096 x
// 12,288 in two splits of 6 17.2, in three of 4 19.0. Two splits of 8 are not: 1 x 4,096 x 16,384 17.2, four of 4 16.2.
template <class T, class S, int G, int kAhead>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(kAhead > 4 ? 2 : G == 128 || kAhead < 4 ? 4 : 3))) void int4_stream_kernel(Int4Params p) {
  constexpr int kParts = 128 / G;   // groups of a block
  constexpr int kSteps = 4 / kParts;
  __shared__ float4 sums[2][kWaves][64];
  const int lane = threadIdx.x & 63;
  const int wave = wave_uniform(threadIdx.x >> 6);
  const int r = lane & 15, grp = lane >> 4;
  const int first = wave_uniform(int(int64_t(p.blocks) * blockIdx.y / p.splits));
  const int blocks = wave_uniform(int(int64_t(p.blocks) * (blockIdx.y + 1) / p.splits)) - first;
  const int tiles = p.swiglu ? p.n / 16 : p.splits > 1 ? p.n_pad / 16 : (p.n + 15) / 16, halves = p.swiglu ? 2 : 1;

  // No load depends on a branch (the compiler could not count the loads in flight, and would wait for all of them): past
  // an end it reads what is there before it. Rows past the last are not stored; k past the end has codes and scales of 0.
  struct Block {
    uint4 w;
    uint2 sc[kParts];
    uint32_t zp;                    // a byte a group
  };
  const uint8_t* zeros = p.zeros ? p.zeros : p.scales;
  const int64_t zero_block = p.zeros ? 16 * kParts : 0;
  const auto fetch = [&](Block& f, int tile, int i) {
    const int64_t at = int64_t(tile) * p.blocks + first + min(i * kWaves + wave, blocks - 1);
    f.w = p.w[at * 64 + lane];
#pragma unroll
    for (int g = 0; g < kParts; ++g)
      f.sc[g] = *reinterpret_cast<const uint2*>(p.scales + at * (32 * kParts) + grp * (8 * kParts) + 8 * g);
    f.zp = zero_points<kParts>(zeros + at * zero_block + r * kParts);
  };
  const auto multiply = [&](const Block& f, const u32x4* x, f32x4 acc) {
    const uint32_t words[4] = {f.w.x, f.w.y, f.w.z, f.w.w};
#pragma unroll
    for (int g = 0; g < kParts; ++g) {
      f32x4 part = f32x4{0.f, 0.f, 0.f, 0.f};
      if (T::kOffset)  // -192 times the sum of x over the group, the same for all 16 weight rows
#pragma unroll
        for (int c = g * kSteps; c < (g + 1) * kSteps; ++c)
          part = T::mfma(u32x4{kMinusOffset, kMinusOffset, kMinusOffset, kMinusOffset}, x[c], part);
      const typename T::Row base = T::row(p.zeros ? (f.zp >> (8 * g)) & 15u : 8u);
#pragma unroll
      for (int c = g * kSteps; c < (g + 1) * kSteps; ++c) part = T::mfma(T::weights(words[c], base), x[c], part);
      const float sc[4] = {S::low(f.sc[g].x), S::high(f.sc[g].x), S::low(f.sc[g].y), S::high(f.sc[g].y)};
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(sc[i], part[i], acc[i]);
    }
    return acc;
  };

  int tile = blockIdx.x, half = 0;  // half 1: the up tile
  Block ring[kAhead];
  u32x4 x[kAhead][4];
  const int64_t m = int64_t(blockIdx.z) * 16 + r;
  const uint16_t* xrow = p.x + min(m, int64_t(p.rows) - 1) * p.x_st + 8 * grp;
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    fetch(ring[i], tile, i);
    const int k = (first + min(i * kWaves + wave, blocks - 1)) * 128;
#pragma unroll
    for (int c = 0; c < 4; ++c) x[i][c] = *reinterpret_cast<const u32x4*>(xrow + min(k + c * 32, p.k - 32));
  }
  float4 gate = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int done = 0; tile < tiles; ++done) {
    const bool last = half + 1 == halves;
    const int next = last ? tile + int(gridDim.x) : tile, next_half = last ? 0 : half + 1;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i * kWaves + wave < blocks) acc = multiply(ring[i], x[i], acc);
      fetch(ring[i], min(next, tiles - 1) + next_half * (p.n / 16), i);
    }
    // a wave in turn adds up, while the others go on
    float4 (*to)[64] = sums[done & 1];
    to[wave][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    if (wave == (done / halves) % kWaves) {
      float4 v = to[0][lane];
#pragma unroll
      for (int q = 1; q < kWaves; ++q) {
        const float4 u = to[q][lane];
        v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
      }
      if (!last) {
        gate = v;
      } else if (m < p.rows) {
        if (p.swiglu) v = make_float4(silu(gate.x) * v.x, silu(gate.y) * v.y, silu(gate.z) * v.z, silu(gate.w) * v.w);
        const float o[4] = {v.x, v.y, v.z, v.w};
        const int col = tile * 16 + 4 * grp;
        if (p.splits > 1)
          *reinterpret_cast<float4*>(p.partials + (int64_t(blockIdx.y) * p.rows + m) * p.n_pad + col) = v;
        else
          store4<T>(p, m, col, o);
      }
    }
    tile = next, half = next_half;
  }
}

// ---------------------------------------------------------------- more rows
constexpr uint32_t kBufferConfig = 0x00020000u;  // gfx9 raw buffer dword 3

__device__ __forceinline__ u32x4 buffer_desc(const char* base, int span) {
  const uint64_t v = reinterpret_cast<uint64_t>(base);
  return u32x4{uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(v))),
               uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(v >> 32))) & 0xffffu, uint32_t(span), kBufferConfig};
}

// 64 lanes x 16 bytes from the buffer straight into 1 KiB of LDS at address `at` (no register output); loads past the
// buffer's span return zeros.
__device__ __forceinline__ void load_lds(u32x4 desc, int voff, uint32_t at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(wave_uniform(int(at))), "v"(voff), "s"(desc) : "memory");
}

// All but the newest kLoads of this wave's loads have landed, and its LDS accesses are done (gfx9's encoding of vmcnt(kLoads)
// lgkmcnt(0): vmcnt in bits 3:0 and 15:14, expcnt 6:4 at 7).
template <int kLoads>
__device__ __forceinline__ void wait_for() {
  static_assert(kLoads < 64, "vmcnt has 6 bits");
  __builtin_amdgcn_s_waitcnt((kLoads & 15) | ((kLoads >> 4) << 14) | 0x70);
}

// Bytes of a ring stage of 128 k: x rows, weight tiles, their scales and zero points; and the stages that fit a CU.
constexpr int stage_bytes(int bm, int tiles, int parts) { return bm * 256 + tiles * (1024 + 48 * parts); }
constexpr int sum_bytes(int bm, int parts) { return 2 * parts * bm * 4; }
constexpr int stages(int bm, int tiles, int parts) {
  // two workgroups a CU where three stages each leave room for them
  const int half = (80 * 1024 - sum_bytes(bm, parts)) / stage_bytes(bm, tiles, parts);
  return half >= 3 ? std::min(half, 5) : std::max(3, std::min(5, (160 * 1024 - sum_bytes(bm, parts)) / stage_bytes(bm, tiles, parts)));
}

// WM x 8 / WM waves; a wave multiplies TM tiles of 16 rows of x with TN tiles of 16 weight rows. Everything travels
// HBM -> LDS directly, into a ring of 3 to 5 stages of 128 k (chunk c of x's row q lies at c ^ (q % 16), so that a
// fragment read covers every bank); one barrier a step. While a wave multiplies 32 k it reads the next
// 32 k's fragments of x and makes the next weights.
// The sums of x (bf16) are made once for all waves, a tile of rows each, a step ahead.
template <class T, class S, int G, int WM, int TM, int TN>
__global__ __launch_bounds__(512) void int4_tile_kernel(Int4Params p) {
  constexpr int kWN = 8 / WM, kBM = 16 * TM * WM, kTiles = kWN * TN;
  constexpr int kParts = 128 / G, kSteps = 4 / kParts;
  constexpr int kDepth = stages(kBM, kTiles, kParts), kStage = stage_bytes(kBM, kTiles, kParts);
  constexpr int kW = kBM * 256, kSc = kW + kTiles * 1024, kZp = kSc + kTiles * 32 * kParts;  // offsets in a stage
  // 1 KiB loads of a wave and stage (of x some twice where they do not come out even: the same bytes to the same place)
  constexpr int kLoadX = (kBM / 4 + 7) / 8, kLoadW = kTiles / 8;
  static_assert(kTiles % 8 == 0, "whole loads a wave");
  constexpr int kLater = kDepth - 3;       // stages whose loads may be in flight at a barrier
  __shared__ uint4 ring[kDepth * kStage / 16];
  __shared__ float x_sums[T::kOffset ? 2 * kParts * kBM : 1];
  const char* lds = reinterpret_cast<const char*>(ring);
  const uint32_t lds_at = uint32_t(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)&ring[0]));
  const int lane = threadIdx.x & 63;
  const int wave = wave_uniform(threadIdx.x >> 6);
  const int r = lane & 15, grp = lane >> 4;
  const int wm = wave % WM, wn = wave / WM;
  const int z = wave_uniform(int(blockIdx.x) % p.splits), bx = wave_uniform(int(blockIdx.x) / p.splits);
  const int64_t m0 = int64_t(blockIdx.y) * kBM;
  const int s0 = wave_uniform(int(int64_t(p.blocks) * z / p.splits));
  const int steps = wave_uniform(int(int64_t(p.blocks) * (z + 1) / p.splits)) - s0;
  const int last_tile = p.n_pad / 16 - 1;
  // tile i of the workgroup; with swiglu a wave's first TN / 2 tiles are gate rows, the others the same columns' up rows
  const auto tile_of = [&](int i) {
    const int w = i / TN, j = i % TN;
    return p.swiglu ? (bx * kWN + w) * (TN / 2) + j % (TN / 2 + (TN == 1)) + (j < TN / 2 ? 0 : p.n / 16) : bx * kTiles + i;
  };

  // ---- loads: an eighth of x's rows and of the weight tiles; the scales and zero points of those tiles
  const int x_row_bytes = int(p.x_st) * 2;
  const char* x_base = reinterpret_cast<const char*>(p.x + m0 * p.x_st) + int64_t(s0) * 256;
  const int rows = int(min(int64_t(kBM), p.rows - m0));
  const int x_row = (lane / 16) * x_row_bytes, x_chunk = ((lane % 16) ^ (lane / 16)) * 16;
  int at[kLoadW];                     // first block of a tile
#pragma unroll
  for (int i = 0; i < kLoadW; ++i) at[i] = min(tile_of(wave * kLoadW + i), last_tile) * p.blocks + s0;
  // Scales and zero points of all tiles: waves 0 and 1, 16 bytes a lane. A load costs about the same however few lanes it has
  // (with one each a wave, 16 a step, the steps of 64 x 128 tiles took 1.0 us).
  constexpr int kLoadS = (kTiles * kParts * 2 + 63) / 64, kLoadZ = (kTiles * kParts + 63) / 64;
  int s_off[kLoadS], z_off[kLoadZ];
#pragma unroll
  for (int i = 0; i < kLoadS; ++i) {
    const int n = i * 64 + lane;
    s_off[i] = (min(tile_of(min(n / (2 * kParts), kTiles - 1)), last_tile) * p.blocks + s0) * (32 * kParts) + n % (2 * kParts) * 16;
  }
#pragma unroll
  for (int i = 0; i < kLoadZ; ++i) {
    const int n = i * 64 + lane;
    z_off[i] = (min(tile_of(min(n / kParts, kTiles - 1)), last_tile) * p.blocks + s0) * (16 * kParts) + n % kParts * 16;
  }
  constexpr int kLoads = kLoadX + kLoadW;
  const int all = p.n_pad / 16 * p.blocks * (16 * kParts);  // bytes of zero points
  // load number d of step s's stage; past the end no bytes, so that every stage counts the same loads
  const auto issue = [&](int s, int d) {
    const uint32_t to = lds_at + uint32_t(s % kDepth) * kStage;
    const bool real = s < steps;
    if (d < kLoadX) {
      const int left = (p.k - (s0 + s) * 128) * 2, n = min(wave * kLoadX + d, kBM / 4 - 1), chunk = x_chunk ^ ((n & 3) * 64);
      const u32x4 dx = buffer_desc(x_base + int64_t(s) * 256, real ? (rows - 1) * x_row_bytes + left : 0);
      // k past the end: zeros (an offset past the span), whatever lies behind x's rows
      load_lds(dx, chunk >= left ? 0x7ffffff0 : n * 4 * x_row_bytes + x_row + chunk, to + n * 1024);
    } else {
      const u32x4 dw = buffer_desc(reinterpret_cast<const char*>(p.w) + int64_t(at[d - kLoadX] + s) * 1024, real ? 1024 : 0);
      load_lds(dw, lane * 16, to + kW + (wave * kLoadW + d - kLoadX) * 1024);
    }
  };
  const auto issue_groups = [&](int s) {
    const uint32_t to = lds_at + uint32_t(s % kDepth) * kStage;
    const bool real = s < steps;
    if (wave == 0) {
      const u32x4 ds = buffer_desc(reinterpret_cast<const char*>(p.scales), real ? 2 * all : 0);
#pragma unroll
      for (int i = 0; i < kLoadS; ++i)
        if (i * 64 + lane < kTiles * kParts * 2) load_lds(ds, s_off[i] + s * (32 * kParts), to + kSc + i * 1024);
    } else if (wave == 1) {
      const u32x4 dz = buffer_desc(reinterpret_cast<const char*>(p.zeros), real && p.zeros ? all : 0);
#pragma unroll
      for (int i = 0; i < kLoadZ; ++i)
        if (i * 64 + lane < kTiles * kParts) load_lds(dz, z_off[i] + s * (16 * kParts), to + kZp + i * 1024);
    }
  };

  const f32x4 none = f32x4{0.f, 0.f, 0.f, 0.f};
  f32x4 acc[TM][TN];
#pragma unroll
  for (int t = 0; t < TM; ++t)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[t][j] = none;
  const int x_at = r * 256 + wm * (TM * 4096);  // this lane's row of the wave's first tile
  const int c_at = (grp ^ r) * 16;              // its chunk of 32 k number c: c_at ^ (64 c)
  const auto meet = [&]() {
    if (kLater == 0 || wave >= 2) wait_for<kLater * (kLoadX + kLoadW)>();
    else if (wave == 0) wait_for<kLater * (kLoadX + kLoadW + kLoadS)>();
    else wait_for<kLater * (kLoadX + kLoadW + kLoadZ)>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // -192 times the sums of x's rows: each wave makes those of one tile (some twice where there are fewer than 8)
  const int sum_tile = wave % (TM * WM);
  const auto sum_chunk = [&](const char* stage, int c) { return *reinterpret_cast<const u32x4*>(stage + sum_tile * 4096 + r * 256 + (c_at ^ (64 * c))); };
  const auto sum_step = [&](u32x4 x, f32x4 v) { return T::mfma(u32x4{kMinusOffset, kMinusOffset, kMinusOffset, kMinusOffset}, x, v); };
  const auto sum_at = [&](int s, int g) { return &x_sums[T::kOffset ? ((s & 1) * kParts + g) * kBM : 0]; };

  for (int s = 0; s < kDepth - 1; ++s) {
    issue_groups(s);
#pragma unroll
    for (int d = 0; d < kLoads; ++d) issue(s, d);
  }
  wait_for<0>();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (T::kOffset) {
#pragma unroll
    for (int g = 0; g < kParts; ++g) {
      f32x4 v = none;
#pragma unroll
      for (int c = g * kSteps; c < (g + 1) * kSteps; ++c) v = sum_step(sum_chunk(lds, c), v);
      if (grp == 0) sum_at(0, g)[sum_tile * 16 + r] = v[0];
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  uint4 w[TN];
  uint32_t zp[TN];
  typename T::Row base[TN];
  u32x4 xf[TM], a[2][TN];
  const auto read_w = [&](const char* stage, int j) {
    w[j] = *reinterpret_cast<const uint4*>(stage + kW + (wn * TN + j) * 1024 + lane * 16);
    zp[j] = zero_points<kParts>(reinterpret_cast<const uint8_t*>(stage) + kZp + ((wn * TN + j) * 16 + r) * kParts);
    if (!p.zeros) zp[j] = 0x08080808u;
  };
  const auto make_a = [&](int c, int j) {
    const uint32_t words[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
    if (c % kSteps == 0) base[j] = T::row((zp[j] >> (8 * (c / kSteps))) & 15u);
    a[c & 1][j] = T::weights(words[c], base[j]);
    asm volatile("" : "+v"(a[c & 1][j]));
  };
  const auto read_x = [&](const char* stage, int c, int t) {
    xf[t] = *reinterpret_cast<const u32x4*>(stage + x_at + t * 4096 + (c_at ^ (64 * c)));
  };
  uint2 s4[TN];
  const auto read_scales = [&](const char* stage, int g) {
#pragma unroll
    for (int j = 0; j < TN; ++j) s4[j] = *reinterpret_cast<const uint2*>(stage + kSc + (((wn * TN + j) * 4 + grp) * kParts + g) * 8);
  };
  constexpr int kSoon = 4;
  const char* stage = lds;
  if (kSteps == 1) read_scales(stage, 0);
#pragma unroll
  for (int j = 0; j < TN; ++j) read_w(stage, j), make_a(0, j);
#pragma unroll
  for (int t = 0; t < TM; ++t) read_x(stage, 0, t);
  int slot = 0;
  for (int s = 0; s < steps; ++s) {
    slot = slot + 1 == kDepth ? 0 : slot + 1;
    const char* following = lds + slot * kStage;  // landed, too; past the last step its values are not used
    f32x4 part[TM][TN], sum = none;
    float sc[TN][4];
    u32x4 sum_x;
    issue_groups(s + kDepth - 1);  // into the slot that the step before read
    const auto take = [&](int t) {     // a finished group of row tile t
#pragma unroll
      for (int j = 0; j < TN; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][j][i] = fmaf(sc[j][i], part[t][j][i], acc[t][j][i]);
        asm volatile("" : "+v"(acc[t][j]));  // here: pure arithmetic would drift to the loop's end, past every fence
      }
    };
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int g = c / kSteps;
      const bool begins = c % kSteps == 0, ends = c % kSteps == kSteps - 1;
      float v[TM];                     // read kSoon slices ahead
      if (begins)
#pragma unroll
        for (int t = 0; t < kSoon && t < TM; ++t) v[t] = T::kOffset ? sum_at(s, g)[(wm * TM + t) * 16 + r] : 0.f;
      // A slice reads a row tile's next fragment and makes its share of the next weights beside a row tile's
      // products (the fences keep that order: left alone, the compiler makes all weights first, and VALU and matrix cores take turns).
#pragma unroll
      for (int t = 0; t < TM; ++t) {
        if (ends && t == 0)
#pragma unroll
          for (int j = 0; j < TN; ++j)
            sc[j][0] = S::low(s4[j].x), sc[j][1] = S::high(s4[j].x), sc[j][2] = S::low(s4[j].y), sc[j][3] = S::high(s4[j].y);
#pragma unroll
        for (int j = t * TN / TM; j < (t + 1) * TN / TM; ++j) {
          make_a(c < 3 ? c + 1 : 0, j);
          if (c == 2) read_w(following, j);
        }
#pragma unroll
        for (int j = 0; j < TN; ++j)
          part[t][j] = T::mfma(a[c & 1][j], xf[t], begins ? f32x4{v[t], v[t], v[t], v[t]} : part[t][j]);
        // The next stage's loads are spread over the first half of the step: together after the barrier they held up every wave.
#pragma unroll
        for (int d = 0; d < kLoads; ++d)
          if (d * 2 * TM / kLoads == c * TM + t) issue(s + kDepth - 1, d);
        // (kept in vector registers, where the compiler needs 10 fewer than with part of them in accumulation registers)
#pragma unroll
        for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(part[t][j]));
        if (c < 3) read_x(stage, c + 1, t);
        else read_x(following, 0, t);
        if (begins && t + kSoon < TM) v[t + kSoon] = T::kOffset ? sum_at(s, g)[(wm * TM + t + kSoon) * 16 + r] : 0.f;
        // the scales of a group that ends in the next phase
        if (t == TM - 1 && (c + 1) % kSteps == kSteps - 1) read_scales(c < 3 ? stage : following, (c + 1) % 4 / kSteps);
        if (ends && t > 0) take(t - 1);
        // (where a phase is short, its chunk is read a phase ahead)
        if (T::kOffset && t == (TM > 4 ? 2 : 0) && (TM > 4 || c == 0)) sum_x = sum_chunk(following, c);
        if (T::kOffset && t == TM - 1) {
          sum = sum_step(sum_x, begins ? none : sum);
          if (TM <= 4 && c < 3) sum_x = sum_chunk(following, c + 1);
          if (ends && grp == 0) sum_at(s + 1, g)[sum_tile * 16 + r] = sum[0];
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      }
      if (ends) take(TM - 1);
    }
    meet();          // every wave has read this stage, and the next two have landed
    stage = following;
  }
  __builtin_amdgcn_s_waitcnt(0x70);  // vmcnt(0): no load may land after the ring is given up
  asm volatile("" ::: "memory");

#pragma unroll
  for (int t = 0; t < TM; ++t) {
    const int64_t m = m0 + (wm * TM + t) * 16 + r;
    if (m >= p.rows) continue;
    if (p.splits > 1) {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int col = tile_of(wn * TN + j) * 16 + 4 * grp;
        const f32x4 v = acc[t][j];
        if (col < p.n_pad)
          *reinterpret_cast<float4*>(p.partials + (int64_t(z) * p.rows + m) * p.n_pad + col) = make_float4(v[0], v[1], v[2], v[3]);
      }
    } else if (p.swiglu) {
#pragma unroll
      for (int j = 0; j < TN / 2; ++j) {
        const f32x4 v = acc[t][j], u = acc[t][j + TN / 2];
        const float o[4] = {silu(v[0]) * u[0], silu(v[1]) * u[1], silu(v[2]) * u[2], silu(v[3]) * u[3]};
        const int col = tile_of(wn * TN + j) * 16 + 4 * grp;
        if (col < p.n) store4<T>(p, m, col, o);
      }
    } else {
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const float o[4] = {acc[t][j][0], acc[t][j][1], acc[t][j][2], acc[t][j][3]};
        store4<T>(p, m, tile_of(wn * TN + j) * 16 + 4 * grp, o);
      }
    }
  }
}

// The sum of the split tiles' slabs, in their order, with the epilogue.
template <class T>
__global__ __launch_bounds__(256) void int4_join_kernel(Int4Params p) {
  const int quads = (p.n + 3) / 4;
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= int64_t(quads) * p.rows) return;
  const int64_t m = i / quads;
  const int col = int(i - m * quads) * 4;
  const auto total = [&](int at) {
    const float* from = p.partials + m * p.n_pad + at;
    const int64_t slab = int64_t(p.rows) * p.n_pad;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q = 0; q < p.splits; q += 8) {  // 8 loads in flight (16 slabs of 33 x 4,016: 4.0 us; one by one 5.7)
      float4 u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = *reinterpret_cast<const float4*>(from + min(q + i, p.splits - 1) * slab);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (q + i < p.splits) v.x += u[i].x, v.y += u[i].y, v.z += u[i].z, v.w += u[i].w;
    }
    return v;
  };
  const float4 v = total(col);
  float o[4] = {v.x, v.y, v.z, v.w};
  if (p.swiglu) {
    const float4 u = total(p.n + col);
    const float up[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = silu(o[e]) * up[e];
  }
  store4<T>(p, m, col, o);
}

template <class T>
void launch_join(const Int4Params& p, hipStream_t s) {
  const int64_t quads = int64_t((p.n + 3) / 4) * p.rows;
  hipLaunchKernelGGL((int4_join_kernel<T>), dim3(unsigned((quads + 255) / 256)), dim3(256), 0, s, p);
}

template <class T, class S, int G>
void launch_stream(const Int4Params& p, hipStream_t s) {
  const int tiles = p.swiglu ? p.n / 16 : p.splits > 1 ? p.n_pad / 16 : (p.n + 15) / 16;
  const int ahead = ((p.blocks + p.splits - 1) / p.splits + kWaves - 1) / kWaves;
  // two workgroups a CU at most, as the registers allow; the second ones take what is over of an uneven number of tiles
  const dim3 grid(std::min(tiles, std::max(1, (ahead > 4 ? 256 : 512) / p.splits)), p.splits, (p.rows + 15) / 16), block(64 * kWaves);
  switch (ahead) {
    case 1: hipLaunchKernelGGL((int4_stream_kernel<T, S, G, 1>), grid, block, 0, s, p); break;
    case 2: hipLaunchKernelGGL((int4_stream_kernel<T, S, G, 2>), grid, block, 0, s, p); break;
    case 3: hipLaunchKernelGGL((int4_stream_kernel<T, S, G, 3>), grid, block, 0, s, p); break;
    case 4: hipLaunchKernelGGL((int4_stream_kernel<T, S, G, 4>), grid, block, 0, s, p); break;
    case 5: hipLaunchKernelGGL((int4_stream_kernel<T, S, G, 5>), grid, block, 0, s, p); break;
    case 6: hipLaunchKernelGGL((int4_stream_kernel<T, S, G, 6>), grid, block, 0, s, p); break;
    default:
      if constexpr (G > 32) {
        if (ahead == 7) hipLaunchKernelGGL((int4_stream_kernel<T, S, G, 7>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((int4_stream_kernel<T, S, G, 8>), grid, block, 0, s, p);
      }
  }
}

template <class T, class S, int G, int WM, int TM, int TN>
void launch_tile(const Int4Params& p, hipStream_t s) {
  const int cols = 16 * (8 / WM) * TN / (p.swiglu ? 2 : 1), width = p.splits > 1 ? p.n_pad : p.n, rows = 16 * WM * TM;
  const dim3 grid((width + cols - 1) / cols * p.splits, (p.rows + rows - 1) / rows);
  hipLaunchKernelGGL((int4_tile_kernel<T, S, G, WM, TM, TN>), grid, dim3(512), 0, s, p);
}

// Rows and columns of a workgroup's tile, and the splits of k; 0 rows: the stream kernel.
struct Shape {
  int rows, cols, splits;
};

// The stream kernel up to 16 rows, its splits as many blocks as its waves hold. Else the shortest of it (without splits) and
// the tiles and splits by what the kernels' parts measured: 1 us to start, 2.5 us to fill the ring and store and the steps in
// whole rounds of one workgroup a CU, and the slabs' join. The steps' us in the table are of groups of 128; groups of 32 take 1.2
// to 1.4 times as long. The stream kernel takes 2.5 us and in each round 1.25 for a block of each of a workgroup's waves. us it chooses between:
// 64 x 1,024 x 4,096 in stream 8.2, in tiles 11.8; 64 x 2,048 x 1,024 5.2, 9.1; 128 x 2,048 x 2,048 13.3, 14.9;
// 128 x 4,096 x 256 12.0, 7.5; 64 x 4,096 x 4,096 22.1, 15.5; 33 x 4,096 x 12,288 in 128 columns and 1 / 2 / 4 / 8 / 16 splits 89 / 50 / 30 / 20 / 20, in 256
// 100 / 56 / 34 / 23 / 20; 208 x 24,576 x 4,096 in 1 / 2 / 4 / 8 splits of 128 x 128 84 / 87 / 103 / 141, 112 x 256 59 / 77 / 82 / 117, 128 x 256
// 64 / 79 / 85 / 120; 2,048 x 6,144 x 4,096 in 112 x 256 123, 128 x 256 125, 128 x 128 147.
Shape choose(int rows, int n_pad, int blocks, int group, bool swiglu) {
  const int most = most_ahead(blocks, group) * kWaves, mine = (blocks + most - 1) / most;
  if (rows <= 16) return Shape{0, 0, mine};
  static constexpr struct {
    int rows, cols;
    double step;
  } kTile[] = {{32, 128, 0.67}, {32, 256, 0.9},  {48, 128, 0.8},   {48, 256, 1.05},  {64, 128, 0.83},
               {64, 256, 1.14}, {112, 256, 1.58}, {128, 128, 1.18}, {128, 256, 1.77}};
  Shape best{};
  double least = 1e30;
  if (mine == 1 && rows <= 16 * 65535) {  // 16 rows to a workgroup in z
    const int halves = swiglu ? 2 : 1;  // a workgroup takes a gate and its up tile
    const double tiles = std::ceil(rows / 16.0) * (n_pad / 16 / halves);
    best = Shape{0, 0, 1};
    least = 2.5 + std::ceil(tiles / 256) * halves * ((blocks + kWaves - 1) / kWaves) * 1.25;
  }
  for (const auto& tile : kTile) {
    if (rows <= 64 ? rows > tile.rows || tile.rows > (rows + 15) / 16 * 16 : tile.rows < 112) continue;
    // 128 columns are one tile a wave up to 64 rows: gate and up tiles do not pair there, but in the join
    const int from = swiglu && tile.cols == 128 && tile.rows <= 64 ? 2 : 1;
    const double step = tile.step * (group == 32 ? (tile.rows > 64 ? 1.4 : 1.2) : 1.0);
    const double tiles = std::ceil(double(rows) / tile.rows) * ((n_pad + tile.cols - 1) / tile.cols);
    for (int s = from; s <= std::max(from, std::min(16, blocks / 2)); ++s) {
      const double join = s > 1 ? 3.5 + double(s) * rows * n_pad * 8 / 5e6 : 0;
      const double cost = 1 + std::ceil(tiles * s / 256) * (2.5 + std::ceil(double(blocks) / s) * step) + join;
      if (cost < least) {
        least = cost;
        best = Shape{tile.rows, tile.cols, s};
      }
    }
  }
  return best;
}

template <class T, class S, int G>
void pick(const Int4Params& p, const Shape& f, hipStream_t s) {
  if (f.rows == 0) return launch_stream<T, S, G>(p, s);
  const bool wide = f.cols == 256;
  if (f.rows == 32) return wide ? launch_tile<T, S, G, 1, 2, 2>(p, s) : launch_tile<T, S, G, 1, 2, 1>(p, s);
  if (f.rows == 48) return wide ? launch_tile<T, S, G, 1, 3, 2>(p, s) : launch_tile<T, S, G, 1, 3, 1>(p, s);
  if (f.rows == 64) return wide ? launch_tile<T, S, G, 1, 4, 2>(p, s) : launch_tile<T, S, G, 1, 4, 1>(p, s);
  if (f.rows == 112) return launch_tile<T, S, G, 1, 7, 2>(p, s);
  return wide ? launch_tile<T, S, G, 1, 8, 2>(p, s) : launch_tile<T, S, G, 2, 4, 2>(p, s);
}

template <class T, class S>
void pick_group(const Int4Params& p, int group, const Shape& f, hipStream_t s) {
  if (group == 32) pick<T, S, 32>(p, f, s);
  else if (group == 64) pick<T, S, 64>(p, f, s);
  else pick<T, S, 128>(p, f, s);
}

int64_t partial_floats(const Shape& f, int rows, int n_pad) { return f.splits > 1 ? int64_t(f.splits) * rows * n_pad : 0; }

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace
}  // namespace aspire

extern "C" int64_t aspire_linear_int4_workspace(int32_t rows, int32_t n, int32_t k, int32_t group, int32_t swiglu) {
  using namespace aspire;
  if (rows <= 0 || n <= 0 || k <= 0 || n > (1 << 30)) return 0;
  const int n_pad = (n + 15) / 16 * 16;
  return partial_floats(choose(rows, n_pad, (k + 127) / 128, group, swiglu != 0), rows, n_pad);
}

extern "C" void aspire_linear_int4_choice(int32_t rows, int32_t n, int32_t k, int32_t group, int32_t swiglu, int32_t choice[3]) {
  using namespace aspire;
  if (choice == nullptr) return;
  choice[0] = choice[1] = choice[2] = 0;
  if (rows <= 0 || rows > (1 << 22) - 64 || n <= 0 || n > (1 << 30) || k <= 0 || k >= (1 << 22)) return;
  if ((group != 32 && group != 64 && group != 128) || k % group != 0 || (swiglu && n % 32 != 0)) return;
  if ((int64_t(n) + 15) / 16 * ((k + 127) / 128) >= (1 << 23)) return;
  const Shape f = choose(rows, (n + 15) / 16 * 16, (k + 127) / 128, group, swiglu != 0);
  choice[0] = f.rows, choice[1] = f.cols, choice[2] = f.splits;
}

extern "C" int aspire_linear_int4(const aspire_int4_args* a, void* stream) {
  using namespace aspire;
  ASPIRE_CHECK_ARG(a != nullptr, "null arguments");
  ASPIRE_CHECK_ARG(a->rows >= 0 && a->n >= 0 && a->n <= (1 << 30) && a->k > 0 && a->k < (1 << 22), "bad sizes");
  ASPIRE_CHECK_ARG((int64_t(a->n) + 15) / 16 * ((a->k + 127) / 128) < (1 << 23), "weights of 2^34 values or more");
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
  p.scales = static_cast<const uint8_t*>(a->scales);
  p.zeros = static_cast<const uint8_t*>(a->zeros);
  p.out = static_cast<uint16_t*>(a->out);
  p.o_st = a->out_stride;
  p.rows = a->rows;
  p.n = outs;
  p.n_pad = (a->n + 15) / 16 * 16;
  p.k = a->k;
  p.blocks = (a->k + 127) / 128;
  p.swiglu = a->swiglu != 0;
  p.wide_out = aligned(a->out, 8) && a->out_stride % 4 == 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Shape f = choose(p.rows, p.n_pad, p.blocks, a->group, a->swiglu != 0);
  ASPIRE_CHECK_ARG(f.rows == 0 || a->x_stride < (1 << 22), "row strides of 2^22 elements or more past 16 rows");
  p.splits = f.splits;
  p.partials = static_cast<float*>(a->workspace);
  ASPIRE_CHECK_ARG(f.splits == 1 || (a->workspace && aligned(a->workspace, 16) && a->workspace_floats >= partial_floats(f, p.rows, p.n_pad)),
                   "workspace must be 16-byte aligned and hold aspire_linear_int4_workspace floats");
  if (f.splits > 1) p.swiglu = 0;  // slabs hold gate and up columns; the join pairs them
  if (a->fp16 && a->scales_fp16) pick_group<Fp16, Fp16>(p, a->group, f, s);
  else if (a->fp16) pick_group<Fp16, Bf16>(p, a->group, f, s);
  else if (a->scales_fp16) pick_group<Bf16, Fp16>(p, a->group, f, s);
  else pick_group<Bf16, Bf16>(p, a->group, f, s);
  if (f.splits > 1) {
    p.swiglu = a->swiglu != 0;
    if (a->fp16) launch_join<Fp16>(p, s);
    else launch_join<Bf16>(p, s);
  }
  ASPIRE_CHECK_LAUNCH();
  return ASPIRE_OK;
}
