// Rotary positions in the forms that checkpoints have (pairs in halves or interleaved, a part of the
// head, any table of frequencies), alone or with the append of k and v to the paged cache.
//
// Pair i of a token at position p turns by the angle p f_i, times an amplitude A:
//     y_a = A (a cos - b sin),  y_b = A (b cos + a sin);   dims (i, i + R/2) or (2i, 2i + 1) of the first R.
// The transpose, which the gradient needs, turns back by the same angle (`inverse`).
//
// Angles: f_i comes as the nearest 64-bit fixed-point fraction of a turn, so p f_i modulo one turn is one 64-bit
// product that drops its overflow and adds no rounding: off by p 2^-65 turns at most, below 2^-24 radians up to position
// 2^38; the fp32 product of other rotary codes is off by 2^-24 of the whole angle, 0.06 radians at a million tokens. What is left is reduced to an
// eighth of a turn by its top bits, and the series of sin and cos there end below 2^-26.
//
// Bound by HBM at prompt sizes (each value read once and written once: 8,192 tokens of 32 q and 8 kv heads of 128 in
// 32 us, 5.3 TB/s, where a large copy runs at 5.2; with the append 46 us, 4.4 TB/s) and by the chain of loads (position
// or row search, then page) at decode sizes (4 tokens 2.9 us, appended 3.7).
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace aspire {
namespace {

constexpr int kMaxPairs = 128;    // head_dim <= 256
constexpr int kRotWaves = 4;      // waves per workgroup
constexpr int kRotTasks = 2;      // tasks a lane has in flight (4: a fifth slower appends, half as many waves a CU)

struct Rows {
  const char* in;
  int64_t in_st, in_sh;           // bytes
  char* out;
  int64_t out_st, out_sh;
  int32_t heads;
  int32_t tasks;                  // of one head
  uint32_t magic;                 // 2^32 / tasks, up: idx / tasks as a high product while idx * tasks < 2^32; 0: one task
};

struct RotaryParams {
  Rows q, k, v;
  int32_t total_tokens, pairs, rotary_dim, head_dim;
  int32_t turning;                // tasks of a head that turn pairs; the rest copy
  const uint64_t* turns;
  float amplitude, direction;     // direction -1: inverse
  const void* positions;
  int32_t positions_64;
  // append
  char* cache;
  int64_t c_sp, c_skv, c_st, c_sh;  // bytes
  int64_t num_pages, num_page_indices;
  int32_t page_size, num_seq;
  const int32_t* indptr;
  const int32_t* page_indices;
  const int32_t* page_indptr;
  const int32_t* last_page_len;
};

struct Bf16 { uint16_t bits; };
struct Fp16 { uint16_t bits; };

__device__ __forceinline__ float widen(Bf16 x) { return __uint_as_float(uint32_t(x.bits) << 16); }
__device__ __forceinline__ float widen(Fp16 x) { return float(__builtin_bit_cast(_Float16, x.bits)); }
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ void narrow(float f, Bf16& x) { x.bits = __builtin_bit_cast(uint16_t, static_cast<__bf16>(f)); }
__device__ __forceinline__ void narrow(float f, Fp16& x) { x.bits = __builtin_bit_cast(uint16_t, static_cast<_Float16>(f)); }
__device__ __forceinline__ void narrow(float f, float& x) { x = f; }

template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Vec { T e[VEC]; };

// cos and sin of 2 pi t / 2^64.
__device__ __forceinline__ float2 cos_sin_of_turn(uint64_t t) {
  const uint32_t quarter = uint32_t((t + (uint64_t(1) << 61)) >> 62);
  const int64_t r = int64_t(t - (uint64_t(quarter) << 62));  // [-2^61, 2^61): an eighth of a turn either way
  // r to 24 bits, or (a small r below 0, whose low half is near 2^32) to 2^-56 of a turn
  const float turn = fmaf(float(int32_t(r >> 32)), 4294967296.f, float(uint32_t(r)));
  const float x = turn * 3.4061215800304843e-19f;            // 2 pi / 2^64
  const float x2 = x * x;
  float s = fmaf(x2, 2.7557319e-6f, -1.9841270e-4f);         // 1/9!, 1/7!, 1/5!, 1/3!
  s = fmaf(x2, s, 8.3333333e-3f);
  s = fmaf(x2, s, -1.6666667e-1f);
  s = fmaf(x2 * x, s, x);
  float c = fmaf(x2, -2.7557319e-7f, 2.4801587e-5f);         // 1/10!, 1/8!, 1/6!, 1/4!, 1/2!
  c = fmaf(x2, c, -1.3888889e-3f);
  c = fmaf(x2, c, 4.1666667e-2f);
  c = fmaf(x2, c, -0.5f);
  c = fmaf(x2, c, 1.f);
  const float cc = quarter & 1 ? s : c, ss = quarter & 1 ? c : s;
  return make_float2((quarter + 1) & 2 ? -cc : cc, quarter & 2 ? -ss : ss);
}

// 2^wpt_log2 waves take a token; each computes its R/2 angles once, a lane each, and hands them round through its LDS
// slice. A task is two accesses: of VEC values in the halves of the pairs, of neighbouring VEC values of interleaved
// pairs, or of 16 bytes (kWide; else VEC values) of what is only copied. Tasks of all heads are numbered through,
// so every lane works whatever the head's width. The first tasks' loads are on their way before the position is known.
template <class T, int VEC, bool kPairs, bool kAppend, bool kWide>
__global__ __launch_bounds__(64 * kRotWaves) void rotary_kernel(RotaryParams p, int wpt_log2) {
  constexpr int kCopy = kWide ? 16 / int(sizeof(T)) : VEC;
  constexpr bool kSingle = kPairs && VEC == 1;   // interleaved pairs that are not aligned: two single accesses
  using V = Vec<T, VEC>;
  using C = Vec<T, kCopy>;
  __shared__ float2 rot[kRotWaves][kMaxPairs];
  const int lane = threadIdx.x & 63;
  const int wave = wave_uniform(threadIdx.x >> 6);
  const int64_t unit = int64_t(blockIdx.x) * kRotWaves + wave;
  const int tok = wave_uniform(int(unit >> wpt_log2));
  const int part = wave_uniform(int(unit) & ((1 << wpt_log2) - 1));
  if (tok >= p.total_tokens) return;

  struct Task {
    int head;                     // numbered over q, k and v; -1: none
    int at, second;               // first value, and how far the second access is from it (0: none)
    bool turning;
    union { V v; C c; } a, b;
  } task[kRotTasks];
  const int nq = p.q.heads * p.q.tasks, nk = p.k.heads * p.k.tasks;
  const int n = nq + nk + (kAppend ? p.v.heads * p.v.tasks : 0);
  const auto rows_of = [&](int head) -> const Rows& {
    return head < p.q.heads ? p.q : kAppend && head >= p.q.heads + p.k.heads ? p.v : p.k;
  };
  const auto load = [&](int base) {
#pragma unroll
    for (int u = 0; u < kRotTasks; ++u) {
      Task& f = task[u];
      int idx = base + ((u * 64) << wpt_log2) + lane;
      f.head = -1;
      if (idx >= n) continue;
      const bool is_q = idx < nq, is_v = kAppend && idx >= nq + nk;
      const Rows& r = is_q ? p.q : is_v ? p.v : p.k;
      idx -= is_q ? 0 : is_v ? nq + nk : nq;
      const int h = r.magic ? int(__umulhi(uint32_t(idx), r.magic)) : idx;
      const int t = idx - h * r.tasks;
      f.head = h + (is_q ? 0 : is_v ? p.q.heads + p.k.heads : p.q.heads);
      f.turning = !is_v && t < p.turning;
      if (f.turning) {
        f.at = t * (kSingle ? 2 : kPairs ? 2 * VEC : VEC);
        f.second = kSingle ? 1 : !kPairs ? p.pairs : f.at + VEC < p.rotary_dim ? VEC : 0;
      } else {
        f.at = is_v ? t * 2 * kCopy : p.rotary_dim + (t - p.turning) * 2 * kCopy;
        f.second = f.at + kCopy < p.head_dim ? kCopy : 0;
      }
      const T* src = reinterpret_cast<const T*>(r.in + tok * r.in_st + h * r.in_sh) + f.at;
      if (f.turning) {
        f.a.v = *reinterpret_cast<const V*>(src);
        if (f.second) f.b.v = *reinterpret_cast<const V*>(src + f.second);
      } else {
        f.a.c = *reinterpret_cast<const C*>(src);
        if (f.second) f.b.c = *reinterpret_cast<const C*>(src + f.second);
      }
    }
  };
  load(part * 64);

  int64_t pos = -1;
  char* page = nullptr;           // the token's place in the cache
  if (kAppend) {
    const int b = wave_last_le(p.indptr, p.num_seq, tok);
    if (b >= 0) {
      const int end = p.indptr[b + 1], first = p.page_indptr[b], pages = p.page_indptr[b + 1] - first;
      const int64_t length = int64_t(max(pages - 1, 0)) * p.page_size + p.last_page_len[b];
      const int64_t place = tok + length - end;
      if (tok < end && pages > 0 && place >= 0 && place < length) {
        const int64_t entry = first + place / p.page_size;
        pos = place;
        if (entry >= 0 && entry < p.num_page_indices) {
          const int id = p.page_indices[entry];
          if (id >= 0 && id < p.num_pages) page = p.cache + id * p.c_sp + (place % p.page_size) * p.c_st;
        }
      }
    }
    if (p.positions != nullptr && pos >= 0)
      pos = p.positions_64 ? static_cast<const int64_t*>(p.positions)[tok] : static_cast<const int32_t*>(p.positions)[tok];
  } else {
    pos = p.positions_64 ? static_cast<const int64_t*>(p.positions)[tok] : static_cast<const int32_t*>(p.positions)[tok];
  }
  for (int i = lane; i < p.pairs; i += 64) {
    float2 r = make_float2(1.f, 0.f);
    if (pos >= 0) {
      r = cos_sin_of_turn(uint64_t(pos) * p.turns[i]);
      r.x *= p.amplitude;
      r.y *= p.amplitude * p.direction;
    }
    rot[wave][i] = r;
  }
  __builtin_amdgcn_wave_barrier();  // the slice is the wave's own, whose LDS accesses keep their order

  const auto turn = [&](int pair, T& x, T& y) {
    const float2 r = rot[wave][pair];
    const float xf = widen(x), yf = widen(y);
    narrow(xf * r.x - yf * r.y, x);
    narrow(yf * r.x + xf * r.y, y);
  };
  for (int base = part * 64; base < n; base += (64 * kRotTasks) << wpt_log2) {
    if (base != part * 64) load(base);
#pragma unroll
    for (int u = 0; u < kRotTasks; ++u) {
      Task& f = task[u];
      if (f.head < 0) continue;
      const bool is_q = f.head < p.q.heads;
      if (kAppend && !is_q && page == nullptr) continue;
      const Rows& r = rows_of(f.head);
      const int h = f.head - (is_q ? 0 : kAppend && f.head >= p.q.heads + p.k.heads ? p.q.heads + p.k.heads : p.q.heads);
      char* out = kAppend && !is_q ? page + (f.head >= p.q.heads + p.k.heads ? p.c_skv : 0) + h * p.c_sh
                                   : r.out + tok * r.out_st + h * r.out_sh;
      T* dst = reinterpret_cast<T*>(out) + f.at;
      if (!f.turning) {
        *reinterpret_cast<C*>(dst) = f.a.c;
        if (f.second) *reinterpret_cast<C*>(dst + f.second) = f.b.c;
        continue;
      }
      if (pos >= 0) {
        if (!kPairs || kSingle) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) turn((kSingle ? f.at / 2 : f.at) + e, f.a.v.e[e], f.b.v.e[e]);
        } else {
#pragma unroll
          for (int e = 0; e + 1 < VEC; e += 2) turn((f.at + e) / 2, f.a.v.e[e], f.a.v.e[e + 1]);
          if (f.second)
#pragma unroll
            for (int e = 0; e + 1 < VEC; e += 2) turn((f.at + VEC + e) / 2, f.b.v.e[e], f.b.v.e[e + 1]);
        }
      }
      *reinterpret_cast<V*>(dst) = f.a.v;
      if (f.second) *reinterpret_cast<V*>(dst + f.second) = f.b.v;
    }
  }
}

template <class T, int VEC, bool kAppend, bool kWide>
void launch(const RotaryParams& p, bool interleaved, int wpt_log2, hipStream_t s) {
  const int64_t units = int64_t(p.total_tokens) << wpt_log2;
  const dim3 grid(unsigned((units + kRotWaves - 1) / kRotWaves)), block(64 * kRotWaves);
  if (interleaved)
    hipLaunchKernelGGL((rotary_kernel<T, VEC, true, kAppend, kWide>), grid, block, 0, s, p, wpt_log2);
  else
    hipLaunchKernelGGL((rotary_kernel<T, VEC, false, kAppend, kWide>), grid, block, 0, s, p, wpt_log2);
}

// vec: values of a turning access; wide: what is copied is 16-byte aligned.
template <class T, bool kAppend>
void dispatch(const RotaryParams& p, int vec, bool wide, bool interleaved, int wpt_log2, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return launch<T, 8, kAppend, true>(p, interleaved, wpt_log2, s);
  if constexpr (sizeof(T) == 4) {
    if (vec == 4) return launch<T, 4, kAppend, true>(p, interleaved, wpt_log2, s);
  } else if (vec == 4) {
    return wide ? launch<T, 4, kAppend, true>(p, interleaved, wpt_log2, s) : launch<T, 4, kAppend, false>(p, interleaved, wpt_log2, s);
  }
  if (vec == 2) return wide ? launch<T, 2, kAppend, true>(p, interleaved, wpt_log2, s) : launch<T, 2, kAppend, false>(p, interleaved, wpt_log2, s);
  return wide ? launch<T, 1, kAppend, true>(p, interleaved, wpt_log2, s) : launch<T, 1, kAppend, false>(p, interleaved, wpt_log2, s);
}

int rotary(const aspire_rotary_args* a, bool append, const char* what, hipStream_t stream) {
#define ROTARY_CHECK(cond, msg)                                   \
  do {                                                            \
    if (!(cond)) {                                                \
      set_error("%s: %s", what, msg);                             \
      return ASPIRE_ERR_INVALID;                                  \
    }                                                             \
  } while (0)
  ROTARY_CHECK(a != nullptr, "null arguments");
  ROTARY_CHECK(a->dtype >= ASPIRE_ROTARY_BF16 && a->dtype <= ASPIRE_ROTARY_FP32, "dtype must be bf16, fp16 or fp32");
  ROTARY_CHECK(!append || a->dtype != ASPIRE_ROTARY_FP32, "the cache holds bf16 or fp16");
  ROTARY_CHECK(a->head_dim > 0 && a->head_dim <= 2 * kMaxPairs, "head_dim must be 1 to 256");
  ROTARY_CHECK(a->rotary_dim > 0 && a->rotary_dim % 2 == 0 && a->rotary_dim <= a->head_dim,
               "rotary_dim must be even and within head_dim");
  ROTARY_CHECK(a->total_tokens >= 0 && a->num_qo_heads >= 0 && a->num_kv_heads >= 0, "bad sizes");
  ROTARY_CHECK(a->num_qo_heads <= 1024 && a->num_kv_heads <= 1024, "at most 1024 heads");
  if (a->total_tokens == 0 || a->num_qo_heads + a->num_kv_heads == 0) return ASPIRE_OK;
  ROTARY_CHECK(a->turns, "null turns");
  ROTARY_CHECK(a->num_qo_heads == 0 || (a->q && a->q_out), "null q");
  ROTARY_CHECK(a->num_kv_heads == 0 || (a->k && (append ? a->v : a->k_out)), append ? "null k / v" : "null k");
  ROTARY_CHECK(append || a->positions, "null positions");

  const int64_t size = a->dtype == ASPIRE_ROTARY_FP32 ? 4 : 2;
  const int whole = int(16 / size);
  int vec = whole;                 // values that every address and stride allows in one access
  const auto fits = [&](const void* ptr, int64_t st, int64_t sh) {
    while (vec > 1 && (reinterpret_cast<uintptr_t>(ptr) % (vec * size) != 0 || st % vec != 0 || sh % vec != 0)) vec /= 2;
  };
  if (a->num_qo_heads > 0) {
    fits(a->q, a->q_stride_t, a->q_stride_h);
    fits(a->q_out, a->q_out_stride_t, a->q_out_stride_h);
  }
  if (a->num_kv_heads > 0) {
    fits(a->k, a->k_stride_t, a->k_stride_h);
    if (!append) {
      fits(a->k_out, a->k_out_stride_t, a->k_out_stride_h);
    } else {
      fits(a->v, a->v_stride_t, a->v_stride_h);
      fits(a->kv_cache, a->cache_stride_p, a->cache_stride_kv);
      fits(a->kv_cache, a->cache_stride_t, a->cache_stride_h);
    }
  }
  const bool wide = vec == whole && a->rotary_dim % whole == 0 && a->head_dim % whole == 0;
  const int span = a->interleaved ? a->rotary_dim : a->rotary_dim / 2;
  while (vec > 1 && (span % vec != 0 || (!wide && a->head_dim % vec != 0))) vec /= 2;
  const int copy = wide ? whole : vec;
  RotaryParams p{};
  const int turning = !a->interleaved ? span / vec : vec == 1 ? span / 2 : (span / vec + 1) / 2;
  const auto rows = [&](const void* in, int64_t st, int64_t sh, void* out, int64_t ost, int64_t osh, int heads, int tasks) {
    return Rows{static_cast<const char*>(in), st * size, sh * size, static_cast<char*>(out), ost * size, osh * size,
                heads, tasks, tasks > 1 ? uint32_t((uint64_t(1) << 32) / tasks + 1) : 0u};
  };
  const auto per_head = [&](bool copies) { return turning + (copies ? ((a->head_dim - a->rotary_dim) / copy + 1) / 2 : 0); };
  p.q = rows(a->q, a->q_stride_t, a->q_stride_h, a->q_out, a->q_out_stride_t, a->q_out_stride_h, a->num_qo_heads,
             per_head(a->q_out != a->q));
  p.k = rows(a->k, a->k_stride_t, a->k_stride_h, a->k_out, a->k_out_stride_t, a->k_out_stride_h, a->num_kv_heads,
             per_head(append || a->k_out != a->k));
  p.v = rows(a->v, a->v_stride_t, a->v_stride_h, nullptr, 0, 0, a->num_kv_heads, (a->head_dim / copy + 1) / 2);
  p.total_tokens = a->total_tokens;
  p.pairs = a->rotary_dim / 2;
  p.rotary_dim = a->rotary_dim;
  p.head_dim = a->head_dim;
  p.turning = turning;
  p.turns = a->turns;
  p.amplitude = a->amplitude;
  p.direction = a->inverse ? -1.f : 1.f;
  p.positions = a->positions;
  p.positions_64 = a->positions_64;
  if (append) {
    ROTARY_CHECK(a->kv_cache && a->num_pages >= 0 && a->page_size > 0, "bad cache");
    ROTARY_CHECK(a->num_seq >= 0 && (a->num_seq == 0 || (a->append_indptr && a->kv_page_indptr && a->kv_last_page_len)),
                 "null page table");
    ROTARY_CHECK(a->num_page_indices >= 0 && (a->num_page_indices == 0 || a->kv_page_indices), "null page indices");
    p.cache = static_cast<char*>(a->kv_cache);
    p.c_sp = a->cache_stride_p * size;
    p.c_skv = a->cache_stride_kv * size;
    p.c_st = a->cache_stride_t * size;
    p.c_sh = a->cache_stride_h * size;
    p.num_pages = a->num_pages;
    p.num_page_indices = a->num_page_indices;
    p.page_size = a->page_size;
    p.num_seq = a->num_seq;
    p.indptr = a->append_indptr;
    p.page_indices = a->kv_page_indices;
    p.page_indptr = a->kv_page_indptr;
    p.last_page_len = a->kv_last_page_len;
  }
  // Waves a token: 4 share its look-ups and angles at prompt sizes, more while the launch stays within kRotMaxWaves. us at
  // 1 / 2 / 4 / 8 / 16 / 32 waves, 32 q and 8 kv heads of 128: 8,192 tokens turned 32 / 34 / 31 / 41 / 73 / 133, appended 47 / 45 / 46 /
  // 56 / 100 / 177; 64 tokens 6.1 / 4.7 / 3.9 / 3.5 / 3.7 / 4.5 and 8.7 / 6.3 / 5.0 / 4.5 / 4.5 / 5.8.
  constexpr int64_t kRotMaxWaves = 1024;
  const int tasks = p.q.heads * p.q.tasks + p.k.heads * p.k.tasks + (append ? p.v.heads * p.v.tasks : 0);
  int wpt_log2 = 0;
  // threads of a launch stay below 2^32, those of the last, partly filled workgroup among them
  ROTARY_CHECK(a->total_tokens <= (1 << 26) - kRotWaves, "more than 2^26 - 4 tokens");
  while (wpt_log2 < 6 && a->total_tokens < (1 << 23) && (64 << wpt_log2) < tasks && (wpt_log2 < 2 || (int64_t(p.total_tokens) << (wpt_log2 + 1)) <= kRotMaxWaves)) ++wpt_log2;
  if (a->dtype == ASPIRE_ROTARY_FP32) {
    dispatch<float, false>(p, vec, wide, a->interleaved != 0, wpt_log2, stream);
  } else if (a->dtype == ASPIRE_ROTARY_FP16) {
    if (append) dispatch<Fp16, true>(p, vec, wide, a->interleaved != 0, wpt_log2, stream);
    else dispatch<Fp16, false>(p, vec, wide, a->interleaved != 0, wpt_log2, stream);
  } else {
    if (append) dispatch<Bf16, true>(p, vec, wide, a->interleaved != 0, wpt_log2, stream);
    else dispatch<Bf16, false>(p, vec, wide, a->interleaved != 0, wpt_log2, stream);
  }
#undef ROTARY_CHECK
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error("%s: kernel launch failed: %s", what, hipGetErrorString(e));
    return ASPIRE_ERR_HIP;
  }
  return ASPIRE_OK;
}

}  // namespace
}  // namespace aspire

extern "C" int aspire_rotary(const aspire_rotary_args* args, void* stream) {
  return aspire::rotary(args, false, __func__, static_cast<hipStream_t>(stream));
}

extern "C" int aspire_rotary_append(const aspire_rotary_args* args, void* stream) {
  return aspire::rotary(args, true, __func__, static_cast<hipStream_t>(stream));
}
