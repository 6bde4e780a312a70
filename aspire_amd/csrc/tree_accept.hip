// What a step keeps of its drafted trees (gfx950): the accepted path of each, and its rows of every layer's cache moved to
// where they stay.
#include <algorithm>
#include <initializer_list>

#include "common.h"

namespace aspire {
namespace {

// ------------------------------------------------------------------------------------------ the path
// A node matches when its token is its parent's target. next[p] = the lowest matching child of p, found by all nodes at
// once (an LDS minimum, whose order does not matter); the path is then a chain of LDS reads, which bound the kernel together with
// two trips to memory. A child stands behind its parent, so a path rises and ends. One wave a row; trees past
// kVerifyNodes tokens look each node's children up in memory instead. Measured: 4 trees of 12 tokens 2.3 us, 64 of up to 48 3.3.
constexpr int kVerifyNodes = 2048;
constexpr int kNone = 0x7fffffff;

__global__ __launch_bounds__(64) void verify_tree_kernel(const int32_t* tree_tokens, const int32_t* parents,
                                                         const int32_t* targets, const int32_t* qo_indptr, int tokens,
                                                         int max_path, int32_t* output, int32_t* path, int32_t* kept) {
  __shared__ int32_t next[kVerifyNodes];
  const int b = blockIdx.x, lane = threadIdx.x;
  const int first = max(qo_indptr[b], 0);
  const int n = max(min(qo_indptr[b + 1], tokens) - first, 0);
  const bool small = n <= kVerifyNodes;
  if (small) {
    for (int i = lane; i < n; i += 64) next[i] = kNone;
    __syncthreads();
    for (int i = lane; i < n; i += 64) {
      const int p = parents[first + i];
      if (p >= 0 && p < i && tree_tokens[first + i] == targets[first + p]) atomicMin(&next[p], i);
    }
    __syncthreads();
  }
  const int64_t row = int64_t(b) * max_path;
  int cur = n > 0 ? 0 : kNone, count = 0;
  for (int j0 = 0; j0 < max_path; j0 += 64) {
    int mine = -1;
    for (int k = 0; k < 64 && cur != kNone && count < max_path; ++k) {
      if (lane == k) mine = cur;
      ++count;
      if (small) {
        cur = next[cur];
      } else {
        const int target = targets[first + cur], up = cur;
        cur = kNone;
        for (int i0 = up + 1; i0 < n && cur == kNone; i0 += 64) {
          const int i = i0 + lane;
          const uint64_t hit = __ballot(i < n && parents[first + i] == up && tree_tokens[first + i] == target);
          if (hit) cur = i0 + __builtin_ctzll(hit);
        }
      }
    }
    if (j0 + lane < max_path) {
      path[row + j0 + lane] = mine;
      output[row + j0 + lane] = mine < 0 ? -1 : targets[first + mine];
    }
  }
  if (lane == 0) kept[b] = count;
}

// ------------------------------------------------------------------------------------------ the move
// A workgroup takes one row of one layer; thread t the vectors t, t + kMoveThreads, ... of a token's K and V. The path rises,
// so no place is written before it has been read as long as each vector's moves are done in order: no wait between
// threads. Moves go in rounds whose loads are in flight together (places written in a round lie below every later
// source). Measured: 36 layers, 64 trees of up to 48 tokens, 8 heads of 128 bf16 7.7 us (17 MB), 28 layers and 4 trees 3.9: the chain
// kept, path, slots, rows.
constexpr int kMoveThreads = 256;
constexpr int kMoveLayers = 64;  // addresses in a launch's arguments
constexpr int kMoveRound = 8;

struct CompactParams {
  char* caches[kMoveLayers];
  int64_t s_p, s_kv, s_t, s_h, num_pages;
  const int32_t* path;
  const int32_t* kept;
  const int32_t* qo_indptr;
  const int64_t* slots;
  int32_t heads, per_head, page_size, tokens, max_path;  // per_head: vectors of a head
};

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4m;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2m;

template <typename V>
__global__ __launch_bounds__(kMoveThreads) void compact_kernel(CompactParams p) {
  __shared__ int64_t from[kMoveThreads], to[kMoveThreads];
  const int b = blockIdx.x;
  char* const cache = p.caches[blockIdx.y];
  const int count = min(p.kept[b], p.max_path);
  if (count < 2) return;
  const int first = p.qo_indptr[b], end = min(p.qo_indptr[b + 1], p.tokens);
  if (first < 0) return;
  const int vectors = 2 * p.heads * p.per_head;
  const auto offset = [&](int i) -> int64_t {  // of token i's slot, or -1
    const int64_t slot = p.slots[i], page = slot / p.page_size;
    return slot < 0 || page >= p.num_pages ? -1 : page * p.s_p + (slot - page * p.page_size) * p.s_t;
  };
  for (int j0 = 1; j0 < count; j0 += kMoveThreads) {
    const int part = min(count - j0, kMoveThreads);
    __syncthreads();
    if (int(threadIdx.x) < part) {
      const int j = j0 + threadIdx.x, node = p.path[int64_t(b) * p.max_path + j];
      const bool moves = node > j && node < end - first;
      const int64_t src = moves ? offset(first + node) : -1, dst = moves ? offset(first + j) : -1;
      from[threadIdx.x] = src < 0 || dst < 0 ? -1 : src;
      to[threadIdx.x] = dst;
    }
    __syncthreads();
    for (int v = threadIdx.x; v < vectors; v += kMoveThreads) {
      const int kv = v >= vectors / 2, w = v - kv * (vectors / 2), h = w / p.per_head;
      char* const base = cache + kv * p.s_kv + h * p.s_h + (w - h * p.per_head) * int64_t(sizeof(V));
      for (int k = 0; k < part; k += kMoveRound) {
        V x[kMoveRound];
        int64_t src[kMoveRound], dst[kMoveRound];
#pragma unroll
        for (int i = 0; i < kMoveRound; ++i) {
          src[i] = k + i < part ? from[k + i] : -1;
          dst[i] = to[min(k + i, part - 1)];
          x[i] = V(0);
          if (src[i] >= 0) x[i] = *reinterpret_cast<const V*>(base + src[i]);
        }
#pragma unroll
        for (int i = 0; i < kMoveRound; ++i)
          if (src[i] >= 0) *reinterpret_cast<V*>(base + dst[i]) = x[i];
      }
    }
  }
}

}  // namespace
}  // namespace aspire

extern "C" int aspire_verify_tree(const int32_t* tree_tokens, const int32_t* parents, const int32_t* targets,
                                  const int32_t* qo_indptr, int32_t tokens, int32_t rows, int32_t max_path, int32_t* output,
                                  int32_t* path, int32_t* kept, void* stream) {
  using namespace aspire;
  ASPIRE_CHECK_ARG(tokens >= 0 && rows >= 0 && max_path >= 1 && max_path <= (1 << 30), "bad sizes");
  ASPIRE_CHECK_ARG(rows <= (1 << 24), "more than 2^24 rows");
  if (rows == 0) return ASPIRE_OK;
  ASPIRE_CHECK_ARG(qo_indptr && output && path && kept && (tokens == 0 || (tree_tokens && parents && targets)), "null array");
  verify_tree_kernel<<<rows, 64, 0, static_cast<hipStream_t>(stream)>>>(tree_tokens, parents, targets, qo_indptr, tokens,
                                                                        max_path, output, path, kept);
  ASPIRE_CHECK_LAUNCH();
  return ASPIRE_OK;
}

extern "C" int aspire_compact_accepted(const aspire_compact_args* a, void* stream) {
  using namespace aspire;
  ASPIRE_CHECK_ARG(a != nullptr, "null arguments");
  ASPIRE_CHECK_ARG(a->layers >= 0 && a->heads >= 0 && a->head_bytes >= 0 && a->page_size > 0 && a->rows >= 0 &&
                       a->tokens >= 0 && a->max_path >= 0 && a->max_path <= (1 << 30) && a->num_pages >= 0, "bad sizes");
  ASPIRE_CHECK_ARG(a->rows <= (1 << 22), "more than 2^22 rows");
  if (a->layers == 0 || a->heads == 0 || a->head_bytes == 0 || a->rows == 0 || a->max_path < 2 || a->tokens == 0 || a->num_pages == 0)
    return ASPIRE_OK;
  ASPIRE_CHECK_ARG(int64_t(a->heads) * a->head_bytes <= (1 << 28), "more than 2^28 bytes a token");
  ASPIRE_CHECK_ARG((a->caches || a->first_cache) && a->path && a->kept && a->qo_indptr && a->slots, "null array");
  // the widest vectors that every row starts and ends on
  uint64_t bits = static_cast<uint64_t>(a->head_bytes);
  for (int64_t s : {a->stride_p, a->stride_kv, a->stride_t, a->stride_h}) bits |= static_cast<uint64_t>(s);
  const auto address = [&](int l) {
    return a->caches ? a->caches[l] : reinterpret_cast<uintptr_t>(a->first_cache) + uint64_t(l) * static_cast<uint64_t>(a->stride_l);
  };
  for (int l = 0; l < a->layers; ++l) {
    ASPIRE_CHECK_ARG(address(l) != 0, "null cache");
    bits |= address(l);
  }
  int vec = 16;
  while (bits & static_cast<uint64_t>(vec - 1)) vec /= 2;
  CompactParams p{};
  p.s_p = a->stride_p, p.s_kv = a->stride_kv, p.s_t = a->stride_t, p.s_h = a->stride_h;
  p.num_pages = a->num_pages;
  p.path = a->path, p.kept = a->kept, p.qo_indptr = a->qo_indptr, p.slots = a->slots;
  p.heads = a->heads, p.per_head = a->head_bytes / vec, p.page_size = a->page_size, p.tokens = a->tokens, p.max_path = a->max_path;
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int l0 = 0; l0 < a->layers; l0 += kMoveLayers) {
    const int layers = std::min(a->layers - l0, kMoveLayers);
    for (int l = 0; l < layers; ++l) p.caches[l] = reinterpret_cast<char*>(address(l0 + l));
    const dim3 grid(a->rows, layers);
    if (vec == 16) compact_kernel<u32x4m><<<grid, kMoveThreads, 0, s>>>(p);
    else if (vec == 8) compact_kernel<u32x2m><<<grid, kMoveThreads, 0, s>>>(p);
    else if (vec == 4) compact_kernel<uint32_t><<<grid, kMoveThreads, 0, s>>>(p);
    else if (vec == 2) compact_kernel<uint16_t><<<grid, kMoveThreads, 0, s>>>(p);
    else compact_kernel<uint8_t><<<grid, kMoveThreads, 0, s>>>(p);
  }
  ASPIRE_CHECK_LAUNCH();
  return ASPIRE_OK;
}
