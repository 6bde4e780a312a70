// Pages and tables of a step from request lengths, on the device (gfx950).
//
// Both kernels are chains of a few memory round trips over some hundred to some hundred thousand bytes, so latency bounds
// them: rows' counts are read once, prefix sums are taken by wave shuffles and held in LDS, and every page, entry
// or token then finds its row there by a binary search (LDS reads, no further trip to memory). Measured, 4 / 64 rows of
// long contexts: the pool 2.6 / 3.1 us, the tables 3.5 / 5.7.
#include <algorithm>

#include "common.h"

namespace aspire {
namespace {

constexpr int kMaxPageRows = 4096;  // running counts of all rows fit in LDS

// Inclusive prefix sums of two values over the workgroup (kThreads a multiple of 64); the totals are everyone's. sums holds
// kThreads / 64 pairs, not in use elsewhere.
struct Pair {
  int64_t a, b;
};
template <int kThreads>
__device__ __forceinline__ Pair block_scan(Pair v, Pair* sums, Pair& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t up_a = __shfl_up(v.a, d, 64), up_b = __shfl_up(v.b, d, 64);
    if (lane >= d) v.a += up_a, v.b += up_b;
  }
  if (lane == 63) sums[wave] = v;
  __syncthreads();
  Pair before{0, 0};
  total = Pair{0, 0};
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    const Pair s = sums[w];
    if (w < wave) before.a += s.a, before.b += s.b;
    total.a += s.a, total.b += s.b;
  }
  return {v.a + before.a, v.b + before.b};
}

// The row of item i: the last one in [0, rows) whose first item offsets[row] is at most i.
__device__ __forceinline__ int row_of(const int32_t* offsets, int rows, int i) {
  int lo = 0, hi = rows;  // offsets[lo] <= i < offsets[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// ------------------------------------------------------------------------------------------- the pool
// One workgroup: the stack is one object, and what a step moves is a page a row. Thread t owns rows t * per .. t * per
// + per - 1. First all pages that are given back go onto the stack, then, behind a barrier, pages are taken from it.
constexpr int kResizeThreads = 512;

__global__ __launch_bounds__(kResizeThreads) void page_resize_kernel(aspire_page_resize_args a) {
  extern __shared__ int32_t resize_lds[];
  __shared__ Pair sums[kResizeThreads / 64];
  __shared__ int32_t first_short, took;
  int32_t* const given_at = resize_lds;                // the row's first page among those given back
  int32_t* const taken_at = resize_lds + a.rows;       // and among those taken
  int32_t* const start = resize_lds + 2 * a.rows;      // the row's first entry that is moved
  const int per = (a.rows + kResizeThreads - 1) / kResizeThreads;
  const int row0 = min(int(threadIdx.x) * per, a.rows), row1 = min(row0 + per, a.rows);
  const auto held_of = [&](int b) { return min(max(a.held[b], 0), a.width); };
  const auto want_of = [&](int b, int held) {
    const int len = a.lengths[b];
    return len < 0 ? held : int((int64_t(len) + a.page_size - 1) / a.page_size);
  };
  const int count = min(max(*a.free_count, 0), a.num_pages);
  if (threadIdx.x == 0) first_short = a.rows;

  Pair sum{0, 0}, total;
  for (int b = row0; b < row1; ++b) {
    const int held = held_of(b), want = want_of(b, held);
    sum.a += max(held - want, 0);
    sum.b += max(want - held, 0);
  }
  Pair at = block_scan<kResizeThreads>(sum, sums, total);
  at.a -= sum.a, at.b -= sum.b;
  const int given = int(total.a);  // at most rows * width, which the host holds under 2^31
  const int64_t free_now = min(int64_t(count) + given, int64_t(a.num_pages));
  if (threadIdx.x == 0) took = int(min(total.b, int64_t(0x7fffffff)));
  // rows that cannot be served: from the first one on
  int64_t after = at.b;
  for (int b = row0; b < row1; ++b) {
    const int held = held_of(b), want = want_of(b, held);
    given_at[b] = int(at.a);
    at.a += max(held - want, 0);
    taken_at[b] = int(min(after, int64_t(0x7fffffff)));  // (where it is cut no row is served)
    after += max(want - held, 0);
    start[b] = min(held, want);
    if (want > held && (want > a.width || after > free_now)) atomicMin(&first_short, b);
  }
  __syncthreads();
  const int served = first_short;
  for (int b = row0; b < row1; ++b) {
    const int held = held_of(b), want = want_of(b, held);
    if (b == served) took = taken_at[b];
    a.shortage[b] = b < served ? 0 : max(want - held, 0);
    if (want < held || b < served) a.held[b] = want;
  }
  if (given > 0) {
    for (int k = threadIdx.x; k < given; k += kResizeThreads) {
      const int b = row_of(given_at, a.rows, k);
      int32_t* const entry = a.block_table + int64_t(b) * a.width + start[b] + (k - given_at[b]);
      const int64_t place = int64_t(count) + given - 1 - k;
      if (place < a.num_pages) a.free_pages[place] = *entry;
      *entry = -1;
    }
  }
  __syncthreads();
  const int taken = took;
  for (int k = threadIdx.x; k < taken; k += kResizeThreads) {
    const int b = row_of(taken_at, served, k);
    const int64_t place = free_now - 1 - k;
    a.block_table[int64_t(b) * a.width + start[b] + (k - taken_at[b])] = a.free_pages[place];
    a.free_pages[place] = -1;
  }
  if (threadIdx.x == 0) *a.free_count = int(free_now) - taken;
}

// -------------------------------------------------------------------------------------------- the tables
// Every workgroup takes the prefix sums of all rows for itself (a few thousand bytes from L2) instead of waiting for another
// launch, then its share of the page entries and of the tokens.
constexpr int kTableThreads = 256;
constexpr int kLongestTree = 4096;
constexpr int kParentWindow = 1024;  // parents before a workgroup's own tokens that are held in LDS

__global__ __launch_bounds__(kTableThreads) void step_tables_kernel(aspire_step_tables_args a) {
  extern __shared__ int32_t tables_lds[];
  __shared__ Pair sums[kTableThreads / 64];
  __shared__ int32_t first_out;
  __shared__ int32_t window[kParentWindow + kTableThreads];
  int32_t* const tok = tables_lds;               // rows + 1
  int32_t* const pag = tables_lds + a.rows + 1;  // rows + 1
  const int per = (a.rows + kTableThreads - 1) / kTableThreads;
  const int row0 = min(int(threadIdx.x) * per, a.rows), row1 = min(row0 + per, a.rows);
  const auto fresh_of = [&](int b) {
    const int cached = a.cached[b], fresh = a.fresh[b];
    return cached < 0 || fresh < 0 || fresh > 0x7fffffff - cached ? 0 : fresh;
  };
  const auto pages_of = [&](int b, int fresh) {
    return fresh == 0 ? int64_t(0) : (int64_t(a.cached[b]) + fresh + a.page_size - 1) / a.page_size;
  };
  Pair sum{0, 0}, all;  // tokens and pages
  for (int b = row0; b < row1; ++b) {
    const int fresh = fresh_of(b);
    sum.a += fresh;
    sum.b += pages_of(b, fresh);
  }
  // a token walks up all its ancestors: without a mask's bound a tree's has one of its own
  const int most = a.tree_words > 0 ? 64 * a.tree_words : a.parents != nullptr ? kLongestTree : 0x7fffffff;
  if (threadIdx.x == 0) first_out = a.rows;
  const Pair upto = block_scan<kTableThreads>(sum, sums, all);
  int64_t t = upto.a - sum.a, e = upto.b - sum.b;
  for (int b = row0; b < row1; ++b) {
    const int fresh = fresh_of(b);
    // counts behind a row that is left out are never used: what they are cut to does not matter
    tok[b] = int(min(t, int64_t(0x7fffffff)));
    pag[b] = int(min(e, int64_t(0x7fffffff)));
    t += fresh;
    e += pages_of(b, fresh);
    if (t > a.max_tokens || e > a.max_entries || fresh > most) {
      atomicMin(&first_out, b);
      for (int c = b + 1; c < row1; ++c) tok[c] = tok[b], pag[c] = pag[b];
      break;
    }
  }
  if (threadIdx.x == kTableThreads - 1) {
    tok[a.rows] = int(min(all.a, int64_t(0x7fffffff)));
    pag[a.rows] = int(min(all.b, int64_t(0x7fffffff)));
  }
  __syncthreads();
  const int served = first_out;
  const int num_tokens = tok[served], num_entries = pag[served];

  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b <= a.max_rows; b += kTableThreads) {
      a.qo_indptr[b] = b <= served ? tok[b] : num_tokens;
      a.kv_indptr[b] = b <= served ? pag[b] : num_entries;
      if (b == a.max_rows) break;
      const int n = b < served ? pag[b + 1] - pag[b] : 0;
      a.last_page_len[b] = n > 0 ? int(int64_t(a.cached[b]) + a.fresh[b] - int64_t(n - 1) * a.page_size) : 0;
    }
    if (threadIdx.x == 0) {
      a.totals[0] = all.a;
      a.totals[1] = all.b;
      a.totals[2] = served;
    }
  }
  const int stride = gridDim.x * kTableThreads;
  for (int i = blockIdx.x * kTableThreads + threadIdx.x; i < num_entries; i += stride) {
    const int b = row_of(pag, served, i), p = i - pag[b];
    a.kv_indices[i] = p < a.width ? a.block_table[int64_t(b) * a.table_stride + p] : -1;
  }
  for (int base = blockIdx.x * kTableThreads; base < a.max_tokens; base += stride) {
    const int i = base + threadIdx.x;
    int first = 0;  // the parents from here to this workgroup's last token are in the window, if they fit
    bool near = false;
    if (a.parents != nullptr && base < num_tokens) {
      first = tok[row_of(tok, served, base)];
      near = base - first <= kParentWindow;
      if (near) {
        __syncthreads();
        const int end = min(base + kTableThreads, num_tokens);
        for (int j = first + threadIdx.x; j < end; j += kTableThreads) window[j - first] = a.parents[j];
        __syncthreads();
      }
    }
    if (i >= a.max_tokens) continue;
    if (i >= num_tokens) {
      a.positions[i] = -1;
      a.slots[i] = -1;
      for (int w = 0; w < a.tree_words; ++w) a.masks[int64_t(i) * a.tree_words + w] = 0;
      continue;
    }
    const int b = row_of(tok, served, i), node = i - tok[b], place = a.cached[b] + node;
    const int p = place / a.page_size;
    const int page = p < a.width ? a.block_table[int64_t(b) * a.table_stride + p] : -1;
    a.slots[i] = page < 0 ? -1 : int64_t(page) * a.page_size + (place - p * a.page_size);
    int depth = node;
    if (a.parents == nullptr) {
      for (int w = 0; w < a.tree_words; ++w) {
        const int bits = min(max(node + 1 - 64 * w, 0), 64);
        a.masks[int64_t(i) * a.tree_words + w] = bits == 64 ? ~int64_t(0) : (int64_t(1) << bits) - 1;
      }
    } else {
      // Up the ancestors; an index that is not below its node's ends the walk. Indices fall on the way, so each word of the mask is
      // written as the walk leaves it, zeros where it passes over one.
      int64_t* const mask = a.tree_words > 0 ? a.masks + int64_t(i) * a.tree_words : nullptr;
      int w = a.tree_words;  // words from here on are written, but for bits
      uint64_t bits = 0;
      const auto leave = [&](int to) {  // for word `to` (-1: the walk is over)
        if (mask == nullptr) return;
        if (w < a.tree_words) mask[w] = int64_t(bits);
        for (int k = w - 1; k > to; --k) mask[k] = 0;
        w = to, bits = 0;
      };
      depth = -1;
      for (int up = node; up >= 0;) {
        ++depth;
        if ((up >> 6) != w) leave(up >> 6);
        bits |= uint64_t(1) << (up & 63);
        const int j = tok[b] + up;
        const int above = near ? window[j - first] : a.parents[j];
        up = above < up ? above : -1;
      }
      leave(-1);
    }
    a.positions[i] = a.cached[b] + depth;
  }
}

}  // namespace
}  // namespace aspire

extern "C" int aspire_page_resize(const aspire_page_resize_args* a, void* stream) {
  using namespace aspire;
  ASPIRE_CHECK_ARG(a != nullptr, "null arguments");
  ASPIRE_CHECK_ARG(a->rows >= 0 && a->rows <= kMaxPageRows, "rows must be 0 to 4096");
  ASPIRE_CHECK_ARG(a->width >= 0 && a->num_pages >= 0 && a->page_size > 0, "bad sizes");
  ASPIRE_CHECK_ARG(int64_t(a->rows) * a->width < (int64_t(1) << 31), "rows * width must be below 2^31");
  if (a->rows == 0) return ASPIRE_OK;
  ASPIRE_CHECK_ARG(a->held && a->free_count && a->shortage && a->lengths && (a->block_table || a->width == 0) &&
                       (a->free_pages || a->num_pages == 0), "null array");
  page_resize_kernel<<<1, kResizeThreads, 12 * a->rows, static_cast<hipStream_t>(stream)>>>(*a);
  ASPIRE_CHECK_LAUNCH();
  return ASPIRE_OK;
}

extern "C" int aspire_step_tables(const aspire_step_tables_args* a, void* stream) {
  using namespace aspire;
  ASPIRE_CHECK_ARG(a != nullptr, "null arguments");
  ASPIRE_CHECK_ARG(a->rows >= 0 && a->rows <= a->max_rows && a->max_rows <= kMaxPageRows, "rows must be 0 to max_rows, max_rows at most 4096");
  ASPIRE_CHECK_ARG(a->width >= 0 && a->max_tokens >= 0 && a->max_entries >= 0 && a->page_size > 0, "bad sizes");
  ASPIRE_CHECK_ARG(a->max_tokens <= (1 << 30) && a->max_entries <= (1 << 30), "more than 2^30 tokens or entries");
  ASPIRE_CHECK_ARG(a->tree_words >= 0 && a->tree_words <= 64, "tree_words must be 0 to 64");
  ASPIRE_CHECK_ARG(a->rows == 0 || (a->cached && a->fresh && (a->block_table || a->width == 0)), "null input");
  ASPIRE_CHECK_ARG(a->qo_indptr && a->kv_indptr && a->totals && (a->max_rows == 0 || a->last_page_len) &&
                       (a->max_entries == 0 || a->kv_indices) && (a->max_tokens == 0 || (a->positions && a->slots)) &&
                       (a->max_tokens == 0 || a->tree_words == 0 || a->masks), "null output");
  const int64_t most = std::max<int64_t>(a->max_entries, a->max_tokens);
  const int grid = static_cast<int>(std::min<int64_t>(std::max<int64_t>((most + kTableThreads - 1) / kTableThreads, 1), 512));
  step_tables_kernel<<<grid, kTableThreads, 8 * (a->rows + 1), static_cast<hipStream_t>(stream)>>>(*a);
  ASPIRE_CHECK_LAUNCH();
  return ASPIRE_OK;
}
