// Attention: the C entry points, and a simple kernel that takes every case.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cmath>

#include "attn.h"
#include "common.h"
#include "mma_device.cuh"
#include "ptx_sm100.cuh"

namespace b200q {
namespace {

// One warp per query token and head; a lane takes a key of 32 for the scores, and dimensions lane, lane + 32, ... of the sum.
template <typename T>
__global__ void __launch_bounds__(128) attn_rows_kernel(const b200q_attention a, int* status) {
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  __shared__ float qs[4][128];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int token = blockIdx.x, head = blockIdx.y * 4 + w;
  if (head >= a.heads) return;
  int b = token, last, m;
  int64_t k0 = 0;
  if (a.cu_q != nullptr) {
    b = -1;
    for (int i = 0; i < a.sequences; ++i)
      if (token >= a.cu_q[i] && token < a.cu_q[i + 1]) b = i;
    if (b < 0) return;
    k0 = a.cu_k[b];
    m = a.cu_k[b + 1] - a.cu_k[b];
    if (a.page_size == 0) m = k0 < 0 ? 0 : min(m, a.key_tokens - a.cu_k[b]);
  } else {
    m = a.lengths[b];
  }
  if (a.page_size > 0) m = static_cast<int>(min(static_cast<int64_t>(m), static_cast<int64_t>(a.table_width) * a.page_size));
  m = max(m, 0);
  last = m - 1;
  if (a.causal && a.cu_q != nullptr) last = token - a.cu_q[b] + m - (a.cu_q[b + 1] - a.cu_q[b]);
  const int kv = head / (a.heads / a.kv_heads);
  const T* q = static_cast<const T*>(a.q.data) + token * a.q.token + head * a.q.head;
  for (int d = lane; d < a.dim; d += 32) qs[w][d] = to_float<T>(q[d]);
  __syncwarp();
  const int seen = min(m, last + 1);
  float top = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0; j0 < seen; j0 += 32) {
    const int j = j0 + lane;
    int64_t at_k = -1, at_v = -1;
    float s = -INFINITY;
    if (j < seen) {
      int64_t page = 0, pos = k0 + j;
      if (a.page_size > 0) {
        page = a.tables[b * a.table_stride + j / a.page_size];
        pos = j % a.page_size;
      }
      s = 0.f;
      if (page >= 0 && (a.page_size == 0 || page < a.pages)) {
        at_k = page * a.k.page + pos * a.k.token + kv * a.k.head;
        at_v = page * a.v.page + pos * a.v.token + kv * a.v.head;
        const T* k = static_cast<const T*>(a.k.data) + at_k;
        for (int d = 0; d < a.dim; ++d) s += qs[w][d] * to_float<T>(k[d]);
        s *= a.scale;
      } else {
        atomicCAS(status, 0, 0xa01);
      }
    }
    float t = s;
    for (int x = 16; x > 0; x >>= 1) t = fmaxf(t, __shfl_xor_sync(~0u, t, x));
    t = fmaxf(t, top);
    const float base = t == -INFINITY ? 0.f : t, keep = expf(top - base);
    const float p = expf(s - base);
    top = t;
    sum = sum * keep + p;
    for (int i = 0; i < 4; ++i) o[i] *= keep;
    for (int l = 0; l < 32; ++l) {
      const float pl = __shfl_sync(~0u, p, l);
      const int64_t v = __shfl_sync(~0u, at_v, l);
      if (v < 0) continue;
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < a.dim) o[i] += pl * to_float<T>(static_cast<const T*>(a.v.data)[v + lane + 32 * i]);
    }
  }
  for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(~0u, sum, x);
  T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(token) * a.heads + head) * a.dim;
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < a.dim) out[lane + 32 * i] = from_float<T>(seen > 0 ? o[i] / sum : 0.f);
}

int check(const b200q_attention* a, bool decode) {
  if (a == nullptr) return B200Q_ERR_NULL_POINTER;
  const bool paged = a->page_size != 0;
  if (a->out == nullptr || (decode ? a->lengths == nullptr : a->cu_q == nullptr || a->cu_k == nullptr) ||
      (paged && a->tables == nullptr))
    return B200Q_ERR_NULL_POINTER;
  if (a->dtype != B200Q_DTYPE_F16 && a->dtype != B200Q_DTYPE_BF16) return B200Q_ERR_BAD_ARGUMENT;
  if (!std::isfinite(a->scale)) return B200Q_ERR_BAD_ARGUMENT;
  if (a->tokens <= 0 || a->sequences <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->dim <= 0 || a->max_q < 0 || a->max_k < 0)
    return B200Q_ERR_BAD_SHAPE;
  if (decode && (!paged || a->tokens != a->sequences)) return B200Q_ERR_BAD_SHAPE;
  if (paged ? a->pages <= 0 || a->page_size < 0 || a->table_width <= 0 || a->table_stride < 0 : a->key_tokens < 0)
    return B200Q_ERR_BAD_SHAPE;
  if (a->heads % a->kv_heads != 0) return B200Q_ERR_BAD_SHAPE;
  if (a->dim % 8 != 0 || a->dim > 128 || a->heads / a->kv_heads > 128 || a->page_size % 16 != 0)
    return B200Q_ERR_UNSUPPORTED_SHAPE;
  for (const b200q_view* x : {&a->q, &a->k, &a->v})
    if (int rc = check_view(*x)) return rc;
  for (const void* x : {static_cast<const void*>(a->cu_q), static_cast<const void*>(a->cu_k),
                        static_cast<const void*>(a->lengths), static_cast<const void*>(a->tables)})
    if ((reinterpret_cast<uintptr_t>(x) & 3u) != 0) return B200Q_ERR_MISALIGNED;
  if ((reinterpret_cast<uintptr_t>(a->out) & 15u) != 0) return B200Q_ERR_MISALIGNED;
  return B200Q_OK;
}

int run(const b200q_attention* a, bool decode, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check(a, decode)) return rc;
  const size_t need = decode ? attn_decode_workspace(*a) : 0;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return B200Q_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return B200Q_ERR_MISALIGNED;
  int* status = device_status_ptr();
  if (status == nullptr) return B200Q_ERR_LAUNCH;
  if (device_cc_major() != 10) return B200Q_ERR_UNSUPPORTED_ARCH;
  if (decode) return launch_attn_decode(*a, workspace, status, static_cast<cudaStream_t>(stream));
  b200q_attention c = *a;
  auto kernel = c.dtype == B200Q_DTYPE_BF16 ? attn_rows_kernel<__nv_bfloat16> : attn_rows_kernel<__half>;
  cudaError_t e = launch_overlapped(DEFAULT_SPLIT, kernel, dim3(c.tokens, (c.heads + 3) / 4), dim3(128), 0,
                                    static_cast<cudaStream_t>(stream), c, status);
  if (e != cudaSuccess) {
    note_cuda_error(e);
    return B200Q_ERR_LAUNCH;
  }
  count_launch();
  return B200Q_OK;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_attn_prefill(const b200q_attention* a, void* workspace, size_t workspace_bytes, void* stream) {
  return run(a, false, workspace, workspace_bytes, stream);
}

int b200q_attn_decode(const b200q_attention* a, void* workspace, size_t workspace_bytes, void* stream) {
  return run(a, true, workspace, workspace_bytes, stream);
}

size_t b200q_attn_prefill_workspace_bytes(const b200q_attention* a) { return check(a, false) == B200Q_OK ? 0 : 0; }
size_t b200q_attn_decode_workspace_bytes(const b200q_attention* a) {
  return check(a, true) == B200Q_OK ? attn_decode_workspace(*a) : 0;
}

}  // extern "C"
