// The paged key-value cache: new tokens go to their slots, pages are copied.  Both are bound by memory: each value is
// read once and written once, in 16-byte pieces.  16384 tokens of 8 heads of 128: 23 us, 5.9 TB/s; 40 pages of 256 positions in 28
// layers: 353 us, 6.7 TB/s.
#include <cuda_runtime.h>

#include <climits>
#include <cstring>
#include <new>

#include "attn.h"
#include "common.h"
#include "ptx_sm100.cuh"

namespace b200q {
namespace {

// ------------------------------------------------------------------------------- store
struct StoreParams {
  const uint4 *k, *v;
  uint4 *k_cache, *v_cache;
  int64_t k_token, k_head, v_token, v_head;                 // all strides in 16-byte pieces
  int64_t kc_page, kc_token, kc_head, vc_page, vc_token, vc_head;
  const int32_t* slots;
  int tokens, row, per_head;                                 // pieces of a token's keys, of a head
  int pages, page_size;
  int* status;
};

// A block takes kStoreTokens tokens; a thread moves the same piece of each, keys and values: 2 x kStoreTokens loads in
// flight.
constexpr int kStoreTokens = 4;

__global__ void __launch_bounds__(256) kv_store_kernel(const StoreParams p) {
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int t0 = blockIdx.x * kStoreTokens;
  for (int c = threadIdx.x; c < p.row; c += blockDim.x) {
    const int head = c / p.per_head, d = c - head * p.per_head;
    uint4 k[kStoreTokens], v[kStoreTokens];
    int slot[kStoreTokens];
#pragma unroll
    for (int i = 0; i < kStoreTokens; ++i) {
      slot[i] = t0 + i < p.tokens ? p.slots[t0 + i] : -1;
      if (t0 + i >= p.tokens) continue;
      k[i] = p.k[(t0 + i) * p.k_token + head * p.k_head + d];
      v[i] = p.v[(t0 + i) * p.v_token + head * p.v_head + d];
    }
#pragma unroll
    for (int i = 0; i < kStoreTokens; ++i) {
      if (slot[i] < 0) continue;
      const int page = slot[i] / p.page_size, at = slot[i] - page * p.page_size;
      if (page >= p.pages) {
        if (c == 0) atomicCAS(p.status, 0, 0xa02);
        continue;
      }
      p.k_cache[page * p.kc_page + at * p.kc_token + head * p.kc_head + d] = k[i];
      p.v_cache[page * p.vc_page + at * p.vc_token + head * p.vc_head + d] = v[i];
    }
  }
}

// -------------------------------------------------------------------------------- copy
// The pairs travel as a kernel argument: no copy from the host, and a captured call keeps them.
constexpr int kPairs = 480;
struct PagePairs {
  int32_t src[kPairs], dst[kPairs];
};
constexpr int kCopyThreads = 256, kCopyPieces = 8;           // 32 KB a block

__global__ void __launch_bounds__(kCopyThreads)
kv_copy_pages_kernel(uint4* cache, int64_t outer_stride, int64_t page_stride, int64_t page_pieces,
                     const __grid_constant__ PagePairs pairs) {
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  uint4* base = cache + blockIdx.z * outer_stride;
  const uint4* src = base + pairs.src[blockIdx.y] * page_stride;
  uint4* dst = base + pairs.dst[blockIdx.y] * page_stride;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kCopyThreads * kCopyPieces) + threadIdx.x;
  uint4 x[kCopyPieces];
#pragma unroll
  for (int i = 0; i < kCopyPieces; ++i)
    if (first + i * kCopyThreads < page_pieces) x[i] = src[first + i * kCopyThreads];
#pragma unroll
  for (int i = 0; i < kCopyPieces; ++i)
    if (first + i * kCopyThreads < page_pieces) dst[first + i * kCopyThreads] = x[i];
}

int finish(cudaError_t e, int launches = 1) {
  if (e != cudaSuccess) {
    note_cuda_error(e);
    return B200Q_ERR_LAUNCH;
  }
  count_launch(launches);
  return B200Q_OK;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int b200q_kv_store(const b200q_view* k, const b200q_view* v, const b200q_view* k_cache,
                              const b200q_view* v_cache, const int32_t* slots, int tokens, int kv_heads, int dim,
                              int pages, int page_size, void* stream) {
  if (k == nullptr || v == nullptr || k_cache == nullptr || v_cache == nullptr || slots == nullptr)
    return B200Q_ERR_NULL_POINTER;
  if (tokens <= 0 || kv_heads <= 0 || dim <= 0 || pages <= 0 || page_size <= 0 || tokens > kMostTokens)
    return B200Q_ERR_BAD_SHAPE;
  if (static_cast<int64_t>(kv_heads) * dim > INT_MAX) return B200Q_ERR_BAD_SHAPE;
  if ((dim % 8) != 0) return B200Q_ERR_UNSUPPORTED_SHAPE;
  for (const b200q_view* x : {k, v, k_cache, v_cache})
    if (int rc = check_view(*x)) return rc;
  if ((reinterpret_cast<uintptr_t>(slots) & 3u) != 0) return B200Q_ERR_MISALIGNED;
  StoreParams p{};
  p.status = device_status_ptr();
  if (p.status == nullptr) return B200Q_ERR_LAUNCH;
  if (device_cc_major() != 10) return B200Q_ERR_UNSUPPORTED_ARCH;
  p.k = static_cast<const uint4*>(k->data);
  p.v = static_cast<const uint4*>(v->data);
  p.k_cache = static_cast<uint4*>(k_cache->data);
  p.v_cache = static_cast<uint4*>(v_cache->data);
  p.k_token = k->token / 8, p.k_head = k->head / 8;
  p.v_token = v->token / 8, p.v_head = v->head / 8;
  p.kc_page = k_cache->page / 8, p.kc_token = k_cache->token / 8, p.kc_head = k_cache->head / 8;
  p.vc_page = v_cache->page / 8, p.vc_token = v_cache->token / 8, p.vc_head = v_cache->head / 8;
  p.slots = slots;
  p.tokens = tokens, p.per_head = dim / 8, p.row = kv_heads * p.per_head;
  p.pages = pages, p.page_size = page_size;
  int threads = 32;
  while (threads < 256 && threads < p.row) threads *= 2;
  return finish(launch_overlapped(DEFAULT_SPLIT, kv_store_kernel, dim3((tokens + kStoreTokens - 1) / kStoreTokens),
                                  dim3(threads), 0, static_cast<cudaStream_t>(stream), p));
}

extern "C" int b200q_kv_copy_pages(void* cache, int64_t outer, int64_t outer_stride, int64_t page_stride,
                                   int64_t page_bytes, int pages, const int32_t* src, const int32_t* dst, int count,
                                   void* stream) {
  if (cache == nullptr || src == nullptr || dst == nullptr) return B200Q_ERR_NULL_POINTER;
  if (outer <= 0 || outer > 65535 || page_bytes <= 0 || pages <= 0 || count <= 0) return B200Q_ERR_BAD_SHAPE;
  if (page_bytes / 16 > static_cast<int64_t>(INT_MAX) * kCopyThreads) return B200Q_ERR_BAD_SHAPE;
  if ((page_bytes % 16) != 0 || (page_stride % 16) != 0 || (outer_stride % 16) != 0 || page_stride < 0 ||
      outer_stride < 0 || (pages > 1 && page_stride < page_bytes) || (outer > 1 && outer_stride < page_bytes))
    return B200Q_ERR_UNSUPPORTED_SHAPE;
  if ((reinterpret_cast<uintptr_t>(cache) & 15u) != 0) return B200Q_ERR_MISALIGNED;
  // bit 0: a source, bit 1: a destination
  uint8_t* seen = new (std::nothrow) uint8_t[pages];
  if (seen == nullptr) return B200Q_ERR_BAD_SHAPE;
  memset(seen, 0, pages);
  bool ok = true;
  for (int i = 0; ok && i < count; ++i) {
    ok = src[i] >= 0 && src[i] < pages && dst[i] >= 0 && dst[i] < pages;
    if (!ok) break;
    seen[src[i]] |= 1;
    ok = (seen[dst[i]] & 2) == 0;
    seen[dst[i]] |= 2;
  }
  for (int i = 0; ok && i < count; ++i) ok = seen[dst[i]] == 2;
  delete[] seen;
  if (!ok) return B200Q_ERR_BAD_ARGUMENT;
  if (device_status_ptr() == nullptr) return B200Q_ERR_LAUNCH;
  if (device_cc_major() != 10) return B200Q_ERR_UNSUPPORTED_ARCH;
  const int64_t pieces = page_bytes / 16, per_block = kCopyThreads * kCopyPieces;
  for (int at = 0; at < count; at += kPairs) {
    const int n = count - at < kPairs ? count - at : kPairs;
    PagePairs pairs{};
    memcpy(pairs.src, src + at, n * sizeof(int32_t));
    memcpy(pairs.dst, dst + at, n * sizeof(int32_t));
    const dim3 grid(static_cast<unsigned>((pieces + per_block - 1) / per_block), n, static_cast<unsigned>(outer));
    if (int rc = finish(launch_overlapped(DEFAULT_SPLIT, kv_copy_pages_kernel, grid, dim3(kCopyThreads), 0,
                                          static_cast<cudaStream_t>(stream), static_cast<uint4*>(cache), outer_stride / 16,
                                          page_stride / 16, pieces, pairs)))
      return rc;
  }
  return B200Q_OK;
}
