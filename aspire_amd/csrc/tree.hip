// Attention of drafted trees over a paged cache (gfx950): a request's tokens see its cached keys and, of its own last n keys,
// those that their mask bits name.
//
// The n tokens of a request are n * G query rows of each kv head (G = q heads per kv head), cut into tiles of kRows. A tile's keys
// are a stream that every row of it shares, so up to some hundred rows the cache's bytes bound the kernel. A
// workgroup takes a tile's keys in steps of 32, its four waves every fourth step, each through an LDS ring of its own (no
// barrier on the way): K and V rows go from HBM straight into LDS (buffer_load ... lds), K two steps ahead from when its
// fragments are read, V from when its are. Per step and 16 query rows:
//   * S^T = K . Q^T with v_mfma_f32_16x16x32 (K rows from LDS, Q in registers): lane (r, grp) holds keys 4 grp + i of row r;
//   * softmax in fp32 with the scale folded into exp2's argument; the running maximum moves only when a key exceeds it by
//     more than kSlack, so most steps take no maximum across lanes and rescale nothing;
//   * O^T += V^T . P^T: the lane's 8 keys of P^T are those that S^T left it with, V^T comes by transpose reads.
// At the end of its keys the waves join through LDS.
//
// Which workgroup takes which keys is decided on the device: lengths are read there alone, so a captured launch serves any. The
// units (request, tile) of one kv head form a line of steps, each unit preceded by kStartCost steps for its start and end;
// group j of `groups` takes the j-th equal part of the line, for each kv head. A unit that falls to several groups is written as
// fp32 pieces (each normalised by its own sum, with its base-2 LSE) and joined by a second launch in the order of its
// keys: results do not depend on timing. The kv head runs fastest over the workgroups, so with 8 kv heads the
// round-robin spread over the XCDs keeps each head's pages in one L2. (Equal pieces of one key range side by side, a piece a
// workgroup, took 176 us instead of 145 for 5 requests of up to 190 tokens over 12,001, and 134 instead of 106 for 16 of up to 40
// over 8,192; each head's pages on one XCD by hand, 782 instead of 735.)
//
// Measured, both launches: 32 requests of 16 tokens over 32,768 keys (32 / 8 heads of 128, 4.3 GB) 665 us = 6.5 TB/s, and the loads
// alone 733 of 737 when that was the time: the stream into LDS bounds it, whatever the order of pages. 16 uneven trees of up to 40 over
// 8,192 106 us; 5 of up to 190 over 12,001, 40 / 8 heads, 141 us = 480 TFLOP/s: tiles that share keys read them again from L2, and
// softmax and products take turns. One tree of 8 over 2,048: 11 + 4 us, a chain of a few trips to memory in each launch.
#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "common.h"

namespace aspire {
namespace {

constexpr float kNegInfT = -__builtin_huge_valf();
constexpr float kSlack = 8.f;       // log2 units
constexpr int kStepKeys = 32;
constexpr int kWaves = 4;           // of a workgroup
constexpr int kStartCost = 4;       // a piece's start and end, in steps
constexpr int kMinPart = 4;         // the least that a group takes, in steps
constexpr int kTreeGroups = 256;    // workgroups of a launch: one a CU
constexpr uint32_t kTreeBuffer = 0x00020000u;  // gfx9 raw buffer dword 3

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

struct TreeParams {
  aspire_tree_attention_args a;
  float scale_log2;
  int32_t group;       // q heads per kv head
  int32_t groups;      // workgroups per kv head
  int32_t page_shift;  // log2(page_size / 16)
  uint32_t num_entries, num_pages;  // of the list and the pool, below 2^31
  // of workgroup w: pieces[w] = (tile's first row among n * G, row count, first token, number of pieces of the
  // unit that starts in it and ends in a later one, or 0); its partial rows: slot 2 w of a unit that began
  // before it, 2 w + 1 of one that goes on after it
  int4* pieces;
  float* part_lse;     // [2 * workgroups][rows of a tile]
  float* part_o;       // [2 * workgroups][rows of a tile][head_dim]
};

template <bool kF16>
__device__ __forceinline__ f32x4 mfma32(uint4 a, uint4 b, f32x4 c) {
  if (kF16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  return mfma_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
}
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
template <bool kF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {  // to nearest even
  if (kF16) {
    const f16x2 v = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
    return __builtin_bit_cast(uint32_t, v);
  }
  return pack_bf16x2_rne(lo, hi);
}
template <bool kF16>
__device__ __forceinline__ float widen(uint32_t x) {  // of the low half
  return kF16 ? float(__builtin_bit_cast(_Float16, uint16_t(x))) : __uint_as_float(x << 16);
}
// Ones in every half whose value is infinite or NaN.
template <bool kF16>
__device__ __forceinline__ uint32_t special(uint32_t x) {
  constexpr uint32_t e = kF16 ? 0x7c00u : 0x7f80u;
  return ((x & e) == e ? 0xffffu : 0u) | ((x & (e << 16)) == (e << 16) ? 0xffff0000u : 0u);
}

template <typename T>
__device__ __forceinline__ T* tree_uniform(T* ptr) {
  const uint64_t v = reinterpret_cast<uint64_t>(ptr);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(v)), hi = __builtin_amdgcn_readfirstlane(uint32_t(v >> 32));
  return reinterpret_cast<T*>((uint64_t(hi) << 32) | lo);
}

__device__ __forceinline__ int64_t wave_uniform64(int64_t v) {
  return int64_t((uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(v >> 32)))) << 32) | uint32_t(__builtin_amdgcn_readfirstlane(int(v))));
}

// 16 bytes a lane from its offset into the buffer to the lane's place behind dst; once: non-temporal, for keys that are mostly read by
// one tile (choose has both sides).
template <bool kOnce>
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t rs, uint4* dst, int offset);
template <>
__device__ __forceinline__ void load_to_lds<true>(__amdgpu_buffer_rsrc_t rs, uint4* dst, int offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16, offset, 0, 0, 2);
}
template <>
__device__ __forceinline__ void load_to_lds<false>(__amdgpu_buffer_rsrc_t rs, uint4* dst, int offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16, offset, 0, 0, 0);
}

// A request as the arrays have it, its tokens cut to those that there are.
struct Request {
  int q0, n, first, pages, len;
};
__device__ __forceinline__ Request request(const TreeParams& p, int b) {
  const aspire_tree_attention_args& a = p.a;
  Request r;
  const int q0 = a.qo_indptr[b], q1 = a.qo_indptr[b + 1], first = a.kv_indptr[b], end = a.kv_indptr[b + 1];
  const int last = a.kv_last_page_len[b];
  r.q0 = max(q0, 0);
  r.n = max(min(q1, a.tokens) - r.q0, 0);
  r.first = first;
  r.pages = int(min(max(int64_t(end) - first, int64_t(0)), int64_t(0x7fffffff)));
  const int64_t len = r.pages > 0 ? int64_t(r.pages - 1) * a.page_size + min(max(last, 0), a.page_size) : 0;
  r.len = int(min(len, int64_t(0x7fff0000)));
  return r;
}

__device__ __forceinline__ int64_t wave_sum_i64(int64_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
  return v;
}

// Request b's length on the line of steps.
template <int kRows>
__device__ __forceinline__ int64_t cost(const TreeParams& p, int b) {
  const Request r = request(p, b);
  return int64_t((r.n * p.group + kRows - 1) / kRows) * ((r.len + kStepKeys - 1) / kStepKeys + kStartCost);
}

// One wave's query rows and what it does with a step of 32 keys: K rows in kb, V rows in vb, 16 keys after 16.
template <bool kF16, int kD, int kT>
struct TreeWave {
  static constexpr int kChunks = kD / 8, kC = kD / 32, kJ = kD / 16;
  static constexpr int kHalf = 16 * kChunks;           // 16-byte chunks of 16 keys
  static constexpr int kLoads = kHalf / 64;            // 1 KiB loads of them
  static constexpr int kPerLoad = 64 / kChunks;        // rows of one load
  static constexpr float kBias = kF16 ? 7.f : 0.f;     // weights are 2^7 larger in fp16, whose smallest normal number is 2^-14
  static constexpr float kSumLimit = float(1 << (8 + (kF16 ? 7 : 0)));  // 2^(kSlack + kBias)

  int r, grp;
  int kidx[kC], vidx[(kJ + 1) / 2];
  float scale_log2;
  uint4 qf[kT][kC];
  float mx[kT], use[kT], l[kT];
  f32x4 acc[kT][kJ];
  f32x4 sc[kT][2];
  uint4 pf[kT];
  uint32_t vis[kT];  // of the present step, where it is masked (see) or has infinities or NaN to add (see_all)

  // LDS places: chunk c of a K row r is at c ^ swizzle_k(r), so that 16 rows' chunks c lie in different banks, and a V row's
  // where transpose reads of 4 rows do
  static __device__ __forceinline__ int swizzle_k(int row) { return kD == 128 ? row : row >> 1; }
  static __device__ __forceinline__ int swizzle_v(int row) { return kD == 128 ? ((row & 3) << 2) | (row >> 2) : ((row >> 1) & 1) << 2; }

  __device__ __forceinline__ void init(int lane, float scale) {
    r = lane & 15, grp = lane >> 4, scale_log2 = scale;
    const int vt_row = 4 * grp + (r >> 2);
#pragma unroll
    for (int c = 0; c < kC; ++c) kidx[c] = r * kChunks + ((4 * c + grp) ^ swizzle_k(r));
#pragma unroll
    for (int c = 0; c < (kJ + 1) / 2; ++c) vidx[c] = vt_row * kChunks + ((4 * c + (r & 3)) ^ swizzle_v(vt_row));
  }
  // rows row0 .. of a request's (past its last one the last again: they are computed and not written)
  __device__ __forceinline__ void start(const TreeParams& p, int q0, int row0, int last, int g) {
    const aspire_tree_attention_args& a = p.a;
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const int row = min(row0 + t * 16 + r, last), node = row / p.group, head = g * p.group + row - node * p.group;
      const uint16_t* const src = static_cast<const uint16_t*>(a.q) + int64_t(q0 + node) * a.q_stride_t + int64_t(head) * a.q_stride_h;
#pragma unroll
      for (int c = 0; c < kC; ++c) qf[t][c] = *reinterpret_cast<const uint4*>(src + 32 * c + 8 * grp);
      mx[t] = kNegInfT, use[t] = 0.f, l[t] = 0.f;
#pragma unroll
      for (int i = 0; i < kJ; ++i) acc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  // Bits of the 32 keys from key0 on that each row sees, of `there` that are left; off: key0's place among the tree's tokens.
  __device__ __forceinline__ void see(const TreeParams& p, int q0, int row0, int last, int off, int there, bool page0, bool page1) {
    uint32_t limit = there >= 32 ? ~0u : (1u << max(there, 0)) - 1;
    if (!page0) limit &= 0xffff0000u;
    if (!page1) limit &= 0xffffu;
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      uint32_t bits = ~0u;
      if (off > -32) {
        const int64_t* const words = p.a.masks + int64_t(q0 + min(row0 + t * 16 + r, last) / p.group) * p.a.mask_stride;
        const int w = max(off, 0) >> 6, sh = max(off, 0) & 63;
        uint64_t x = w < p.a.mask_words ? uint64_t(words[w]) >> sh : 0;
        if (sh > 32 && w + 1 < p.a.mask_words) x |= uint64_t(words[w + 1]) << (64 - sh);
        bits = off < 0 ? (uint32_t(x) << -off) | ((1u << -off) - 1) : uint32_t(x);
      }
      vis[t] = bits & limit;
    }
  }
  __device__ __forceinline__ void see_all() {
#pragma unroll
    for (int t = 0; t < kT; ++t) vis[t] = ~0u;
  }
  __device__ __forceinline__ void scores(const uint4* kb) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 kr[kC];
#pragma unroll
      for (int c = 0; c < kC; ++c) kr[c] = kb[h * kHalf + kidx[c]];
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        sc[t][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kC; ++c) sc[t][h] = mfma32<kF16>(kr[c], qf[t][c], sc[t][h]);
      }
    }
  }
  __device__ __forceinline__ void softmax(bool masked) {
    float x[kT][8], pv[kT][8], ps[kT];
#pragma unroll
    for (int t = 0; t < kT; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[t][i] = sc[t][0][i], x[t][4 + i] = sc[t][1][i];
    }
    if (masked) {
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        const uint32_t bits = vis[t] >> (4 * grp);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[t][i] = (bits >> i) & 1 ? x[t][i] : kNegInfT;
          x[t][4 + i] = (bits >> (16 + i)) & 1 ? x[t][4 + i] : kNegInfT;
        }
      }
    }
    const auto exponentials = [&]() {
#pragma unroll
      for (int t = 0; t < kT; ++t) {
#pragma unroll
        for (int i = 0; i < 8; ++i) pv[t][i] = __builtin_amdgcn_exp2f(fmaf(x[t][i], scale_log2, -use[t]));
        ps[t] = ((pv[t][0] + pv[t][1]) + (pv[t][2] + pv[t][3])) + ((pv[t][4] + pv[t][5]) + (pv[t][6] + pv[t][7]));
      }
    };
    exponentials();
    // a row that has seen no key yet (on its first step; later if that one was masked) has no offset to go by
    bool over = masked;
#pragma unroll
    for (int t = 0; t < kT; ++t) over |= ps[t] > kSumLimit || mx[t] == kNegInfT;
    if (__builtin_amdgcn_ballot_w64(over) != 0) {
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        float top = fmaxf(fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3])),
                          fmaxf(fmaxf(x[t][4], x[t][5]), fmaxf(x[t][6], x[t][7])));
        top = max_xor32(max_xor16(top)) * scale_log2;
        const float m_new = top > mx[t] + kSlack ? top : mx[t];
        // a row without a key before has zero sums: they stay zero
        const float alpha = __builtin_amdgcn_exp2f(mx[t] - (m_new == kNegInfT ? 0.f : m_new));
        mx[t] = m_new;
        use[t] = m_new == kNegInfT ? 0.f : m_new - kBias;
#pragma unroll
        for (int i = 0; i < kJ; ++i) acc[t][i] *= alpha;
        l[t] *= alpha;
      }
      exponentials();
    }
    // Weights go into the product with V rounded to V's type, as the matrix instruction takes them (their sum is of the fp32 ones).
    // An output is off from 64 bits by 0.0020 of the rms of all (bf16, 16 tokens over 2,048 keys; fp16, heads of 64, 0.00029), its own
    // rounding alone by 0.0017 (0.00021). In two parts, the second of what the first lacks, it is that, but 40 tokens over 8,192 keys take
    // 113 us in place of 107 and 190 over 12,001 159 in place of 142, and an infinite V times a second part of 0 is NaN.
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      pf[t] = make_uint4(pack2<kF16>(pv[t][0], pv[t][1]), pack2<kF16>(pv[t][2], pv[t][3]), pack2<kF16>(pv[t][4], pv[t][5]),
                         pack2<kF16>(pv[t][6], pv[t][7]));
      l[t] += ps[t];
    }
  }
  __device__ __forceinline__ void product(const uint4* vb) {
    const char* const va = reinterpret_cast<const char*>(vb);
#pragma unroll
    for (int i = 0; i < kJ; ++i) {
      const int off = vidx[i >> 1] * 16 + 8 * (i & 1);
      const uint2 wa = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(va + off)));
      const uint2 wb = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                     (__attribute__((address_space(3))) i16x4*)(va + kHalf * 16 + off)));
#pragma unroll
      for (int t = 0; t < kT; ++t) acc[t][i] = mfma32<kF16>(make_uint4(wa.x, wa.y, wb.x, wb.y), pf[t], acc[t][i]);
    }
  }
  // A key that some rows see and others do not may hold infinities or NaN in V, which a product with weight 0 would carry over. Such
  // values are added for the rows that see them and put to 0 in LDS before the product.
  __device__ __forceinline__ bool has_special(const uint4* vb) const {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 2 * kLoads; ++i) {
      const uint4 x = vb[i * 64 + 16 * grp + r];
      bad |= (special<kF16>(x.x) | special<kF16>(x.y) | special<kF16>(x.z) | special<kF16>(x.w)) != 0;
    }
    return bad;
  }
  __device__ __forceinline__ void add_special(const uint4* vb) {
    const char* const va = reinterpret_cast<const char*>(vb);
    for (int key = 0; key < kStepKeys; ++key) {
      const int row = key & 15, e = (key & 3) + 4 * (key >> 4), from = r + 16 * (row >> 2);
      float w[kT];
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        const uint32_t p0 = pf[t].x, p1 = pf[t].y, p2 = pf[t].z, p3 = pf[t].w;
        uint32_t two = p0;
        two = (e >> 1) == 1 ? p1 : two;
        two = (e >> 1) == 2 ? p2 : two;
        two = (e >> 1) == 3 ? p3 : two;
        w[t] = __shfl(widen<kF16>((two >> (16 * (e & 1))) & 0xffffu), from, 64);
      }
#pragma unroll
      for (int i = 0; i < kJ; ++i) {
        const int c = (key >> 4) * kHalf + row * kChunks + ((4 * (i >> 1) + grp) ^ swizzle_v(row));
        const uint2 x = *reinterpret_cast<const uint2*>(va + c * 16 + 8 * (i & 1));
        const uint32_t sx = special<kF16>(x.x), sy = special<kF16>(x.y);
#pragma unroll
        for (int t = 0; t < kT; ++t) {
          if (!((vis[t] >> key) & 1)) continue;
          if (sx & 0xffffu) acc[t][i][0] += w[t] * widen<kF16>(x.x & 0xffffu);
          if (sx >> 16) acc[t][i][1] += w[t] * widen<kF16>(x.x >> 16);
          if (sy & 0xffffu) acc[t][i][2] += w[t] * widen<kF16>(x.y & 0xffffu);
          if (sy >> 16) acc[t][i][3] += w[t] * widen<kF16>(x.y >> 16);
        }
      }
    }
  }
  __device__ __forceinline__ void clear_special(uint4* vb) const {
#pragma unroll
    for (int i = 0; i < 2 * kLoads; ++i) {
      uint4 x = vb[i * 64 + 16 * grp + r];
      x.x &= ~special<kF16>(x.x), x.y &= ~special<kF16>(x.y), x.z &= ~special<kF16>(x.z), x.w &= ~special<kF16>(x.w);
      vb[i * 64 + 16 * grp + r] = x;
    }
  }
};

// A workgroup's four waves are kRW row groups (16 kT query rows each) times kKW = 4 / kRW key groups: a stage is 32 keys for each
// key group.
//   kRW = 1: every wave has all rows and every fourth step in an LDS ring of two of its own. No barrier on the way: K is
//     refilled, two steps ahead, once its fragments have been read, V once its have.
//   kRW = 2, 4: the waves of a key group share its keys; kStages stages in LDS, one barrier a stage, loads kStages - 1 stages
//     ahead, two workgroups a CU. (Tiles of 256 rows on eight waves halve the reads of shared keys but take 165 us where four
//     waves take 146, trees of up to 190 nodes, 40 / 8 heads; half of the eight meeting the barrier half a stage later, 169;
//     three workgroups of three stages at 168 registers 185.)
template <bool kF16, int kD, int kT, int kRW, bool kOnce>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(kRW == 1 ? 1 : 2))) void tree_attention_kernel(
    TreeParams p) {
  typedef TreeWave<kF16, kD, kT> Wave;
  constexpr int kKW = kWaves / kRW, kGroupRows = 16 * kT, kRows = kGroupRows * kRW;
  constexpr int kHalf = Wave::kHalf, kLoads = Wave::kLoads, kJ = Wave::kJ;
  constexpr int kStages = kRW == 4 ? 4 : 2;
  constexpr int kStage = kKW * 4 * kHalf;  // chunks: for each key group K of 32 keys, then V
  // separate objects, so that the compiler can tell a load into one from a read of another
  __shared__ uint4 st0[kRW == 1 ? 8 * kHalf : kStage];   // kRW = 1: K of the rings' first places
  __shared__ uint4 st1[kRW == 1 ? 8 * kHalf : kStage];   // their V
  __shared__ uint4 st2[kRW == 1 ? 8 * kHalf : kStages > 2 ? kStage : 1];
  __shared__ uint4 st3[kRW == 1 ? 8 * kHalf : kStages > 3 ? kStage : 1];
  __shared__ float stat_m[kKW == 1 ? 1 : kWaves][kGroupRows], stat_l[kKW == 1 ? 1 : kWaves][kGroupRows];
  const aspire_tree_attention_args& a = p.a;
  const int lane = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6);
  const int rw = wave % kRW, kw = wave / kRW;
  const int G = p.group, hkv = a.num_kv_heads;
  const int g = wave_uniform(int(blockIdx.x) % hkv), j = wave_uniform(int(blockIdx.x) / hkv);

  // this group's part [line0, line1) of the line, and the row that holds its first step
  int64_t all = 0;
  for (int b = lane; b < a.rows; b += 64) all += cost<kRows>(p, b);
  all = wave_uniform64(wave_sum_i64(all));
  const int groups = wave_uniform(int(min(max(all / kMinPart, int64_t(1)), int64_t(p.groups))));  // each has kMinPart steps at least
  const int64_t line0 = all * j / groups, line1 = all * (j + 1) / groups;
  if (threadIdx.x == 0) p.pieces[blockIdx.x].w = 0;
  if (j >= groups || all == 0) return;
  int64_t at = 0;  // where row b begins
  int b = 0;
  for (int b0 = 0; b0 < a.rows; b0 += 64) {
    const int64_t c = b0 + lane < a.rows ? cost<kRows>(p, b0 + lane) : 0;
    int64_t end = c;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t up = __shfl_up(end, d, 64);
      if (lane >= d) end += up;
    }
    const uint64_t past = __ballot(at + end > line0);
    if (past) {
      const int l = __builtin_ctzll(past);
      b = b0 + l;
      at += __shfl(end - c, l, 64);
      break;
    }
    at += __shfl(end, 63, 64);
  }
  b = wave_uniform(b);
  at = wave_uniform64(at);

  const int row_bytes = int(a.cache_stride_t) * 2;
  const char* const k_base = static_cast<const char*>(a.kv_cache) + int64_t(g) * a.cache_stride_h * 2;
  const char* const v_base = k_base + a.cache_stride_kv * 2;
  const uint32_t page_bytes = uint32_t(a.cache_stride_p) * 2u, sub_bytes = uint32_t(row_bytes) * 16u;  // below 2^32 (checked on the host)
  const int sub_mask = (1 << p.page_shift) - 1;
  const uint32_t num_entries = p.num_entries, num_pages = p.num_pages;
  // This lane's chunks of 16 keys: the ones that belong at its places in LDS. With kRW > 1 a wave loads K or V alone.
  const bool loads_v = kRW > 1 && (wave & 1);
  int voff_k[kLoads], voff_v[kRW == 1 ? kLoads : 1];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = Wave::kPerLoad * i + lane / Wave::kChunks, c = lane % Wave::kChunks;
    voff_k[i] = row * row_bytes + (c ^ (loads_v ? Wave::swizzle_v(row) : Wave::swizzle_k(row))) * 16;
    if (kRW == 1) voff_v[i] = row * row_bytes + (c ^ Wave::swizzle_v(row)) * 16;
  }
  Wave w;
  w.init(lane, p.scale_log2);

  for (; b < a.rows && at < line1; ++b) {
    const Request rq = request(p, b);
    const int q0 = wave_uniform(rq.q0), n = wave_uniform(rq.n), len = wave_uniform(rq.len);
    const int list = wave_uniform(rq.first), pages = wave_uniform(rq.pages);
    const int total_rows = n * G, tiles = (total_rows + kRows - 1) / kRows, steps = (len + kStepKeys - 1) / kStepKeys;
    const int unit = steps + kStartCost, tree_start = len - n;
    // the first tile that reaches into this group's part
    int m = wave_uniform(at >= line0 ? 0 : int(min((line0 - at) / unit, int64_t(tiles))));
    typedef const __attribute__((address_space(4))) int32_t* const_ids_t;
    const const_ids_t ids = (const_ids_t)a.kv_indices;
    for (; m < tiles; ++m) {
      const int64_t unit0 = at + int64_t(m) * unit;
      if (unit0 >= line1) break;
      const int begin = wave_uniform(int(min(max(line0 - unit0 - kStartCost, int64_t(0)), int64_t(steps))));
      const int end = wave_uniform(int(min(max(line1 - unit0 - kStartCost, int64_t(0)), int64_t(steps))));
      const bool starts = line0 <= unit0;  // a unit without keys is written where it starts
      if (begin >= end && !(steps == 0 && starts)) continue;
      const bool whole = begin == 0 && end == steps;
      const int row0 = m * kRows + rw * kGroupRows, last = total_rows - 1;  // this wave's rows
      w.start(p, q0, row0, last, g);

      // The page of 16 keys: half h of a step. raw() only loads it (a scalar load, used a step later), page() is -1 on a page that
      // the pool does not have, or past the end: such halves load nothing. Out-of-range loads write zeros into LDS, and every step issues the same loads.
      const auto raw = [&](int step, int h) -> int {
        const uint32_t entry = uint32_t(list) + uint32_t((2 * step + h) >> p.page_shift);
        return ids[min(entry, num_entries - 1)];
      };
      const auto page = [&](int step, int h, int id) -> int {
        const uint32_t e = uint32_t(2 * step + h) >> p.page_shift;  // 32-bit compares: there are no scalar 64-bit ones
        const bool there = step < end && e < uint32_t(pages) && uint32_t(list) + e < num_entries && uint32_t(id) < num_pages;
        return there ? id : -1;
      };
      const auto issue = [&](uint4* dst, int step, int h, int id, bool v) {
        const int half = 2 * step + h, left = len - half * 16;
        const int span = wave_uniform(id < 0 ? 0 : left >= 16 ? 15 * row_bytes + 2 * kD : left > 0 ? (left - 1) * row_bytes + 2 * kD : 0);
        const char* const at = (v ? v_base : k_base) + uint64_t(uint32_t(max(id, 0))) * page_bytes + uint32_t(half & sub_mask) * sub_bytes;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(tree_uniform(at)), (short)0, span, kTreeBuffer);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load_to_lds<kOnce>(rs, dst + i * 64, kRW == 1 && v ? voff_v[kRW == 1 ? i : 0] : voff_k[i]);
      };
      const auto masked_step = [&](int step, bool page0, bool page1) {
        const bool masked = (step + 1) * kStepKeys > tree_start || !page0 || !page1;
        if (masked) w.see(p, q0, row0, last, step * kStepKeys - tree_start, len - step * kStepKeys, page0, page1);
        return masked;
      };

      if constexpr (kRW == 1) {
        // this wave's steps: begin + wave, and every fourth from there; step s + 8 goes into the ring's place of step s
        const int first = begin + wave;
        if (first < end) {
          uint4* const mk[2] = {st0 + wave * 2 * kHalf, st2 + wave * 2 * kHalf};
          uint4* const mv[2] = {st1 + wave * 2 * kHalf, st3 + wave * 2 * kHalf};
          int id[2][2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int s = first + u * kWaves;
#pragma unroll
            for (int h = 0; h < 2; ++h) issue(mk[u] + h * kHalf, s, h, id[u][h] = page(s, h, raw(s, h)), false);
#pragma unroll
            for (int h = 0; h < 2; ++h) issue(mv[u] + h * kHalf, s, h, id[u][h], true);
          }
          int next0 = raw(first + 2 * kWaves, 0), next1 = raw(first + 2 * kWaves, 1);
          constexpr int kAhead = 6 * kLoads;  // loads behind this step's K, and again behind its V
          constexpr int kWait = 0xf70 | (kAhead & 15) | ((kAhead >> 4) << 14);
          const auto body = [&](int s, uint4* kb, uint4* vb, int& id0, int& id1) {
            bool masked = false;
            __builtin_amdgcn_s_waitcnt(kWait);  // vmcnt: K has landed
            asm volatile("" ::: "memory");
            if (s < end) {
              masked = masked_step(s, id0 >= 0, id1 >= 0);
              w.scores(kb);
            }
            const int far = s + 2 * kWaves, n0 = page(far, 0, next0), n1 = page(far, 1, next1);
            next0 = raw(far + kWaves, 0), next1 = raw(far + kWaves, 1);
            issue(kb, far, 0, n0, false), issue(kb + kHalf, far, 1, n1, false);
            if (s < end) w.softmax(masked);
            __builtin_amdgcn_s_waitcnt(kWait);  // vmcnt: V has landed
            asm volatile("" ::: "memory");
            if (s < end) {
              // (a step in front of the tree has no key that rows see differently)
              if ((s + 1) * kStepKeys > tree_start && __builtin_amdgcn_ballot_w64(w.has_special(vb)) != 0) {
                w.add_special(vb);
                w.clear_special(vb);
              }
              w.product(vb);
            }
            issue(vb, far, 0, n0, true), issue(vb + kHalf, far, 1, n1, true);
            id0 = n0, id1 = n1;
          };
          for (int s = first; s < end; s += 2 * kWaves) {
            body(s, mk[0], mv[0], id[0][0], id[0][1]);
            body(s + kWaves, mk[1], mv[1], id[1][0], id[1][1]);
          }
        }
      } else {
        // Stage t holds the steps begin + kKW t + (0 .. kKW - 1). A wave loads one kind of its key group's: K or V (kKW = 2), or
        // half of them (kKW = 1).
        const int lh = (wave >> 1) & 1, kind = wave & 1;
        constexpr int kMine = kKW == 2 ? 2 * kLoads : kLoads;  // its loads of a stage
        constexpr int kAhead = (kStages - 2) * kMine;          // loads behind the next stage's
        constexpr int kWait = 0x70 | (kAhead & 15) | ((kAhead >> 4) << 14);  // vmcnt, and lgkmcnt(0): its reads of the last stage
        const int stages = (end - begin + kKW - 1) / kKW;
        const auto step_of = [&](int t) { return begin + t * kKW + kw; };
        uint32_t there = 0;  // two bits a stage: whether its halves have pages, the last one that was loaded lowest
        const auto load = [&](uint4* stage, int t, int raw0, int raw1) {
          const int s = step_of(t), id0 = page(s, 0, raw0), id1 = page(s, 1, raw1);
          there = (there << 2) | (id0 >= 0 ? 1u : 0u) | (id1 >= 0 ? 2u : 0u);
          uint4* const dst = stage + kw * 4 * kHalf + kind * 2 * kHalf;
          if (kKW == 2) {
            issue(dst, s, 0, id0, kind), issue(dst + kHalf, s, 1, id1, kind);
          } else {
            issue(dst + lh * kHalf, s, lh, lh ? id1 : id0, kind);
          }
        };
        const auto begin_stage = [&](uint4* stage, int t) { load(stage, t, raw(step_of(t), 0), raw(step_of(t), 1)); };
        begin_stage(st0, 0);
        if constexpr (kStages > 2) begin_stage(st1, 1), begin_stage(st2, 2);
        int next0 = raw(step_of(kStages - 1), 0), next1 = raw(step_of(kStages - 1), 1);
        const bool has_rows = row0 <= last;
        const auto body = [&](int t, uint4* cur, uint4* fill) {
          __builtin_amdgcn_s_waitcnt(kWait);
          asm volatile("" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          load(fill, t + kStages - 1, next0, next1);
          next0 = raw(step_of(t + kStages), 0), next1 = raw(step_of(t + kStages), 1);
          const int s = step_of(t);
          uint4* const kb = cur + kw * 4 * kHalf;
          const bool computes = s < end && has_rows;
          bool bad = false, masked = false;
          if ((begin + (t + 1) * kKW) * kStepKeys > tree_start)  // every wave's: the stage reaches into the tree
            bad = __syncthreads_or(w.has_special(kb + 2 * kHalf)) != 0;
          if (computes) {
            const uint32_t mine = there >> (2 * (kStages - 1));
            masked = masked_step(s, mine & 1, mine & 2);
            w.scores(kb);
            w.softmax(masked);
          }
          if (bad) {
            // with two key groups one's step may lie in front of the tree that the stage reaches into: its rows see all of it
            if (kKW > 1 && !masked) w.see_all();
            if (computes) w.add_special(kb + 2 * kHalf);
            __syncthreads();
            w.clear_special(kb + 2 * kHalf);  // (waves of a key group write the same)
            __syncthreads();
          }
          if (computes) w.product(kb + 2 * kHalf);
        };
        // Stage by stage, and back to the top only from the last place: waits are counted by the order of the loads. (The places
        // are named, not indexed.)
        int t = 0;
        const auto next = [&](uint4* cur, uint4* fill) {
          body(t, cur, fill);
          return ++t < stages;
        };
        if (stages > 0) {
          if constexpr (kStages == 2) {
            while (next(st0, st1) && next(st1, st0)) {}
          } else {
            while (next(st0, st3) && next(st1, st0) && next(st2, st1) && next(st3, st2)) {}
          }
        }
      }

      // the key groups join: each takes its share of the head's values from all
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        w.l[t] = add_xor32(add_xor16(w.l[t]));
        if (kKW > 1 && w.grp == 0) stat_m[wave][t * 16 + w.r] = w.mx[t], stat_l[wave][t * 16 + w.r] = w.l[t];
      }
      constexpr int kShare = kJ / kKW;  // 16-value tiles a wave writes
      f32x4 o[kT][kShare];
      float lse[kT];
      if constexpr (kKW > 1) {
        __builtin_amdgcn_s_waitcnt(0xf70);  // vmcnt(0): the loads past the end have written their zeros
        __syncthreads();
        uint4* const places[4] = {st0, st1, st2, st3};
#pragma unroll
        for (int t = 0; t < kT; ++t) {
          float top = kNegInfT, sum = 0.f;
#pragma unroll
          for (int k = 0; k < kKW; ++k) top = fmaxf(top, stat_m[k * kRW + rw][t * 16 + w.r]);
          const float zero = top == kNegInfT ? 0.f : top;
#pragma unroll
          for (int k = 0; k < kKW; ++k)
            sum += stat_l[k * kRW + rw][t * 16 + w.r] * __builtin_amdgcn_exp2f(stat_m[k * kRW + rw][t * 16 + w.r] - zero);
          const float scale = __builtin_amdgcn_exp2f(w.mx[t] - zero);
          w.l[t] = sum;
          w.use[t] = zero - Wave::kBias;
#pragma unroll
          for (int i = 0; i < kJ; ++i) {
            const f32x4 x = w.acc[t][i] * scale;
            places[i / kShare][((wave * kT + t) * kShare + i % kShare) * 64 + lane] = __builtin_bit_cast(uint4, x);
          }
        }
        __syncthreads();
        const uint4* const mine = kw == 0 ? st0 : kw == 1 ? st1 : kw == 2 ? st2 : st3;
#pragma unroll
        for (int t = 0; t < kT; ++t) {
#pragma unroll
          for (int i = 0; i < kShare; ++i) {
            o[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < kKW; ++k)
              o[t][i] += __builtin_bit_cast(f32x4, mine[(((k * kRW + rw) * kT + t) * kShare + i) * 64 + lane]);
          }
        }
      } else {
#pragma unroll
        for (int t = 0; t < kT; ++t)
#pragma unroll
          for (int i = 0; i < kShare; ++i) o[t][i] = w.acc[t][i];
      }
      const int slot = 2 * blockIdx.x + (begin == 0 ? 1 : 0);
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        const float inv = w.l[t] == 0.f ? 0.f : 1.f / w.l[t];
        lse[t] = w.l[t] == 0.f ? kNegInfT : w.use[t] + __builtin_log2f(w.l[t]);
#pragma unroll
        for (int i = 0; i < kShare; ++i) o[t][i] *= inv;
        const int row = row0 + t * 16 + w.r;
        if (row > last) continue;
        // value e of 16-value tile i: 32 (i / 2) + 8 grp + 4 (i % 2) + e
        const int tile0 = kw * kShare;
        if (whole) {
          const int node = row / G, head = g * G + row - node * G;
          uint16_t* const dst = static_cast<uint16_t*>(a.out) + int64_t(q0 + node) * a.out_stride_t + int64_t(head) * a.out_stride_h;
          if constexpr (kShare > 1) {
#pragma unroll
            for (int i = 0; i < kShare; i += 2)
              *reinterpret_cast<uint4*>(dst + 16 * (tile0 + i) + 8 * w.grp) =
                  make_uint4(pack2<kF16>(o[t][i][0], o[t][i][1]), pack2<kF16>(o[t][i][2], o[t][i][3]),
                             pack2<kF16>(o[t][i + 1][0], o[t][i + 1][1]), pack2<kF16>(o[t][i + 1][2], o[t][i + 1][3]));
          } else {
            *reinterpret_cast<uint2*>(dst + 32 * (tile0 >> 1) + 8 * w.grp + 4 * (tile0 & 1)) =
                make_uint2(pack2<kF16>(o[t][0][0], o[t][0][1]), pack2<kF16>(o[t][0][2], o[t][0][3]));
          }
          if (a.lse != nullptr && kw == 0 && w.grp == 0) a.lse[int64_t(q0 + node) * a.num_qo_heads + head] = lse[t];
        } else {
          const int64_t at_row = int64_t(slot) * kRows + row - m * kRows;
          float* const dst = p.part_o + at_row * kD;
#pragma unroll
          for (int i = 0; i < kShare; ++i)
            *reinterpret_cast<f32x4*>(dst + 32 * ((tile0 + i) >> 1) + 8 * w.grp + 4 * ((tile0 + i) & 1)) = o[t][i];
          if (kw == 0 && w.grp == 0) p.part_lse[at_row] = lse[t];
        }
      }
      if (begin == 0 && end < steps && threadIdx.x == 0) {
        // the groups that hold the unit's other steps: the last one's part holds its last step
        const int64_t last_step = unit0 + unit - 1;
        int jl = int(last_step * groups / all);
        jl = min(max(jl, j), groups - 1);
        while (jl < groups - 1 && all * (jl + 1) / groups <= last_step) ++jl;
        while (jl > j && all * jl / groups > last_step) --jl;
        p.pieces[blockIdx.x] = make_int4(m * kRows, min(kRows, total_rows - m * kRows), q0, jl - j + 1);
      }
      if (kKW == 1) __builtin_amdgcn_s_waitcnt(0xf70);  // vmcnt(0): no load past the end meets the next unit's
      __syncthreads();  // the stages are free again
    }
    at += int64_t(tiles) * unit;
  }
}

// Units cut into pieces: out = sum_i 2^(lse_i - m) o_i / sum_i 2^(lse_i - m), rounded once, in the order of the keys. Workgroup
// (w, y) has rows of the unit that starts in workgroup w of the launch before and ends in another; a wave takes kTake rows at
// once, 64 / (kD / 8) pieces of each at a time, kRound times. Latency bounds it, 3.5 to 11 us: the pieces' list, then their rows.
template <bool kF16, int kD, int kTake>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeParams p, int tile_rows) {
  constexpr int kLanes = kD / 8, kAtOnce = 64 / kLanes, kRound = 2;
  const aspire_tree_attention_args& a = p.a;
  const int hkv = a.num_kv_heads, g = blockIdx.x % hkv;
  const int lane = threadIdx.x & 63, d = (lane % kLanes) * 8, part = lane / kLanes;
  const int row0 = (blockIdx.y * 4 + wave_uniform(threadIdx.x >> 6)) * kTake;
  const int4 u = p.pieces[blockIdx.x];
  const int rows = wave_uniform(u.y), splits = wave_uniform(u.w);
  if (splits == 0 || row0 >= rows) return;
  float top[kTake], sum[kTake], o[kTake][8];
#pragma unroll
  for (int t = 0; t < kTake; ++t) {
    top[t] = kNegInfT, sum[t] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[t][e] = 0.f;
  }
  for (int k = 0; k < splits; k += kAtOnce * kRound) {
    float lse[kTake][kRound];
    float4 x[kTake][kRound], y[kTake][kRound];
#pragma unroll
    for (int t = 0; t < kTake; ++t) {
#pragma unroll
      for (int i = 0; i < kRound; ++i) {
        const int s = k + i * kAtOnce + part;
        const int64_t slot = 2 * (int64_t(blockIdx.x) + int64_t(min(s, splits - 1)) * hkv) + (min(s, splits - 1) == 0 ? 1 : 0);
        const int64_t at = slot * tile_rows + min(row0 + t, rows - 1);
        lse[t][i] = s < splits ? p.part_lse[at] : kNegInfT;
        x[t][i] = *reinterpret_cast<const float4*>(p.part_o + at * kD + d);
        y[t][i] = *reinterpret_cast<const float4*>(p.part_o + at * kD + d + 4);
      }
    }
#pragma unroll
    for (int t = 0; t < kTake; ++t) {
      float next = top[t];
#pragma unroll
      for (int i = 0; i < kRound; ++i) next = fmaxf(next, lse[t][i]);
      const float zero = next == kNegInfT ? 0.f : next, keep = __builtin_amdgcn_exp2f(top[t] - zero);
      sum[t] *= keep;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[t][e] *= keep;
#pragma unroll
      for (int i = 0; i < kRound; ++i) {
        if (k + i * kAtOnce + part >= splits) continue;
        const float f = __builtin_amdgcn_exp2f(lse[t][i] - zero);
        sum[t] += f;
        o[t][0] += f * x[t][i].x, o[t][1] += f * x[t][i].y, o[t][2] += f * x[t][i].z, o[t][3] += f * x[t][i].w;
        o[t][4] += f * y[t][i].x, o[t][5] += f * y[t][i].y, o[t][6] += f * y[t][i].z, o[t][7] += f * y[t][i].w;
      }
      top[t] = next;
    }
  }
#pragma unroll
  for (int t = 0; t < kTake; ++t) {
    // the pieces' lanes, in a fixed order
#pragma unroll
    for (int step = kLanes; step < 64; step <<= 1) {
      const float other = __shfl_xor(top[t], step, 64), next = fmaxf(top[t], other), zero = next == kNegInfT ? 0.f : next;
      const float f = __builtin_amdgcn_exp2f(top[t] - zero), h = __builtin_amdgcn_exp2f(other - zero);
      sum[t] = f * sum[t] + h * __shfl_xor(sum[t], step, 64);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[t][e] = f * o[t][e] + h * __shfl_xor(o[t][e], step, 64);
      top[t] = next;
    }
    if (row0 + t >= rows || part != 0) continue;
    const float inv = sum[t] == 0.f ? 0.f : 1.f / sum[t];
    const int at = u.x + row0 + t, node = at / p.group, token = u.z + node, head = g * p.group + at - node * p.group;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + int64_t(token) * a.out_stride_t + int64_t(head) * a.out_stride_h + d) =
        make_uint4(pack2<kF16>(o[t][0] * inv, o[t][1] * inv), pack2<kF16>(o[t][2] * inv, o[t][3] * inv),
                   pack2<kF16>(o[t][4] * inv, o[t][5] * inv), pack2<kF16>(o[t][6] * inv, o[t][7] * inv));
    if (a.lse != nullptr && d == 0)
      a.lse[int64_t(token) * a.num_qo_heads + head] = sum[t] == 0.f ? kNegInfT : top[t] + __builtin_log2f(sum[t]);
  }
}

// What a launch is made of: 16-row tiles a wave, row groups of a workgroup, workgroups a kv head, and whether keys are mostly read by
// one tile alone.
struct TreeChoice {
  int tiles, row_groups, groups;
  bool once;
  int rows() const { return 16 * tiles * row_groups; }
};
TreeChoice choose(int tokens, int rows, int hq, int hkv) {
  // The smallest tile that holds a mean request's query rows. A larger one computes rows that are not there, a smaller one reads keys
  // again for each tile. us with tiles of 16 / 32 / 64 / 128 rows: one request of 16 rows over 2,048 keys 19.1 / 20.3 / 20.1 / 21.5; 32 of
  // 64 over 32,768: 2,555 / 1,290 / 665 / 688; 16 of about 80 over 8,192: 295 / 184 / 131 / 107; 5 of about 480 over 12,001: 673 / 336 /
  // 226 / 143. Up to 32 rows a wave holds them all and goes by itself, one workgroup a CU; with more, two workgroups a CU.
  // Rows without tokens count in the mean: the call is better made without them (5 of 480 rows with 59 empty ones 296 us in
  // place of 141, 32 of 64 with 32 empty ones 1,286 in place of 663).
  // Non-temporal loads where a mean request is one tile, us with / without: 32 of 64 rows over 32,768 keys 665 / 737, 16 of up to 160 (5
  // of them two tiles) over 8,192 106 / 109; 5 of up to 950 over 12,001 148 / 142, 24 of up to 231 over 5,000, heads of 64, 41.6 / 40.3.
  const int64_t mean = (int64_t(tokens) + rows - 1) / rows * (hq / hkv);
  TreeChoice c{mean <= 16 ? 1 : 2, mean <= 32 ? 1 : mean <= 64 ? 2 : 4, 0, mean <= 128};
  c.groups = std::max(1, (c.row_groups == 1 ? 1 : 2) * kTreeGroups / hkv);
  return c;
}
template <bool kF16, int kD>
void launch(const TreeParams& p, TreeChoice c, hipStream_t s) {
  const int wgs = c.groups * p.a.num_kv_heads;
  if (c.tiles == 1) tree_attention_kernel<kF16, kD, 1, 1, true><<<wgs, 256, 0, s>>>(p);
  else if (c.row_groups == 1) tree_attention_kernel<kF16, kD, 2, 1, true><<<wgs, 256, 0, s>>>(p);
  else if (c.row_groups == 2) tree_attention_kernel<kF16, kD, 2, 2, true><<<wgs, 256, 0, s>>>(p);
  else if (c.once) tree_attention_kernel<kF16, kD, 2, 4, true><<<wgs, 256, 0, s>>>(p);
  else tree_attention_kernel<kF16, kD, 2, 4, false><<<wgs, 256, 0, s>>>(p);
  // two rows a wave where there are many: 16 trees of up to 40 tokens 106.3 us, with one 107.5, with four 108.6
  if (c.rows() <= 32) tree_join_kernel<kF16, kD, 1><<<dim3(wgs, c.rows() / 4), 256, 0, s>>>(p, c.rows());
  else tree_join_kernel<kF16, kD, 2><<<dim3(wgs, c.rows() / 8), 256, 0, s>>>(p, c.rows());
}
int64_t piece_bytes(int64_t workgroups) { return (workgroups * int64_t(sizeof(int4)) + 255) / 256 * 256; }

}  // namespace
}  // namespace aspire

extern "C" int64_t aspire_tree_attention_workspace(int32_t tokens, int32_t rows, int32_t num_qo_heads, int32_t num_kv_heads,
                                                   int32_t head_dim) {
  using namespace aspire;
  if (tokens <= 0 || rows <= 0 || num_kv_heads <= 0 || num_qo_heads <= 0 || num_qo_heads % num_kv_heads != 0 || head_dim <= 0 ||
      num_qo_heads > 1024)
    return 0;
  const TreeChoice c = choose(tokens, rows, num_qo_heads, num_kv_heads);
  const int64_t wgs = int64_t(c.groups) * num_kv_heads;
  return piece_bytes(wgs) / 4 + 2 * wgs * c.rows() * (head_dim + 1);
}

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
  ASPIRE_CHECK_ARG(a->tokens <= (1 << 20) && a->rows <= (1 << 20), "more than 2^20 tokens or rows");
  if (a->tokens == 0 || a->rows == 0) return ASPIRE_OK;
  ASPIRE_CHECK_ARG(a->q && a->out && a->qo_indptr && a->kv_indptr && a->kv_last_page_len && (a->masks || a->mask_words == 0), "null array");
  const bool none = a->num_pages == 0 || a->num_page_indices == 0;  // no page is there: no key is seen
  ASPIRE_CHECK_ARG(none || (a->kv_cache && a->kv_indices), "null cache or list");
  ASPIRE_CHECK_ARG(a->cache_stride_t >= a->head_dim && a->cache_stride_t < (1 << 20), "tokens of a page must lie head_dim to 2^20 - 1 values apart");
  ASPIRE_CHECK_ARG(a->cache_stride_p >= 0 && a->cache_stride_p < (int64_t(1) << 31), "pages must lie less than 2^31 values apart");
  const auto aligned = [](const void* ptr, std::initializer_list<int64_t> strides) {
    int64_t bits = static_cast<int64_t>(reinterpret_cast<uintptr_t>(ptr)) / 2 % 8;
    for (int64_t s : strides) bits |= s;
    return (bits & 7) == 0;
  };
  ASPIRE_CHECK_ARG(aligned(a->q, {a->q_stride_t, a->q_stride_h}) && aligned(a->out, {a->out_stride_t, a->out_stride_h}) &&
                       aligned(a->kv_cache, {a->cache_stride_p, a->cache_stride_kv, a->cache_stride_t, a->cache_stride_h}),
                   "heads must start on 16 bytes");
  const TreeChoice c = choose(a->tokens, a->rows, a->num_qo_heads, a->num_kv_heads);
  const int wgs = c.groups * a->num_kv_heads, tile_rows = c.rows();
  ASPIRE_CHECK_ARG(a->workspace && a->workspace_floats >= aspire_tree_attention_workspace(a->tokens, a->rows, a->num_qo_heads, a->num_kv_heads, a->head_dim),
                   "workspace too small");
  ASPIRE_CHECK_ARG((reinterpret_cast<uintptr_t>(a->workspace) & 15) == 0, "workspace must start on 16 bytes");
  TreeParams p{};
  p.a = *a;
  p.scale_log2 = a->sm_scale * 1.4426950408889634f;
  p.group = a->num_qo_heads / a->num_kv_heads;
  p.groups = c.groups;
  if (none) p.a.kv_indices = a->qo_indptr;  // an entry to load; its value is no page's id
  p.num_entries = none ? 1u : static_cast<uint32_t>(std::min<int64_t>(a->num_page_indices, 0x7fffffff));
  p.num_pages = none ? 0u : static_cast<uint32_t>(std::min<int64_t>(a->num_pages, 0x7fffffff));
  while ((16 << p.page_shift) < a->page_size) ++p.page_shift;
  p.pieces = reinterpret_cast<int4*>(a->workspace);
  p.part_o = a->workspace + piece_bytes(wgs) / 4;
  p.part_lse = p.part_o + int64_t(2) * wgs * tile_rows * a->head_dim;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype == 1) {
    if (a->head_dim == 128) launch<true, 128>(p, c, s);
    else launch<true, 64>(p, c, s);
  } else {
    if (a->head_dim == 128) launch<false, 128>(p, c, s);
    else launch<false, 64>(p, c, s);
  }
  ASPIRE_CHECK_LAUNCH();
  return ASPIRE_OK;
}
