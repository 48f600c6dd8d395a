// Attention: the C entry points and what they refuse.
#include <cuda_runtime.h>

#include "attn.h"
#include "common.h"

namespace b200q {
namespace {

int check(const b200q_attention* a, bool decode) {
  if (a == nullptr) return B200Q_ERR_NULL_POINTER;
  const bool paged = a->page_size != 0;
  if (a->out == nullptr || (decode ? a->lengths == nullptr : a->cu_q == nullptr || a->cu_k == nullptr) ||
      (paged && a->tables == nullptr))
    return B200Q_ERR_NULL_POINTER;
  if (a->dtype != B200Q_DTYPE_F16 && a->dtype != B200Q_DTYPE_BF16) return B200Q_ERR_BAD_ARGUMENT;
  if (!(a->scale > 0) || !(a->scale < 1e38f)) return B200Q_ERR_BAD_ARGUMENT;
  if (a->tokens <= 0 || a->sequences <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->dim <= 0 || a->max_q < 0 || a->max_k < 0)
    return B200Q_ERR_BAD_SHAPE;
  if (a->tokens > kMostTokens || a->key_tokens > kMostTokens) return B200Q_ERR_BAD_SHAPE;
  if (decode && (!paged || a->tokens != a->sequences)) return B200Q_ERR_BAD_SHAPE;
  if (paged ? a->pages <= 0 || a->page_size < 0 || a->table_width <= 0 || a->table_stride < 0 : a->key_tokens < 0)
    return B200Q_ERR_BAD_SHAPE;
  if (a->heads % a->kv_heads != 0 || a->heads > (1 << 15)) return B200Q_ERR_BAD_SHAPE;
  if (a->dim % 8 != 0 || a->dim > 128 || a->heads / a->kv_heads > 128 || a->page_size % 16 != 0)
    return B200Q_ERR_UNSUPPORTED_SHAPE;
  for (const b200q_view* x : {&a->q, &a->k, &a->v})
    if (int rc = check_view(*x)) return rc;
  // a stride of zero would make rows of the same memory, which no TMA descriptor describes
  if ((a->tokens > 1 && a->q.token == 0) || (a->heads > 1 && a->q.head == 0)) return B200Q_ERR_UNSUPPORTED_SHAPE;
  for (const b200q_view* x : {&a->k, &a->v})
    if (((paged ? a->page_size : a->key_tokens) > 1 && x->token == 0) || (a->kv_heads > 1 && x->head == 0) ||
        (paged && a->pages > 1 && x->page == 0))
      return B200Q_ERR_UNSUPPORTED_SHAPE;
  for (const void* x : {static_cast<const void*>(a->cu_q), static_cast<const void*>(a->cu_k),
                        static_cast<const void*>(a->lengths), static_cast<const void*>(a->tables)})
    if ((reinterpret_cast<uintptr_t>(x) & 3u) != 0) return B200Q_ERR_MISALIGNED;
  if ((reinterpret_cast<uintptr_t>(a->out) & 15u) != 0) return B200Q_ERR_MISALIGNED;
  return B200Q_OK;
}

int run(const b200q_attention* a, bool decode, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check(a, decode)) return rc;
  const size_t need = decode ? attn_decode_workspace(*a) : attn_prefill_workspace(*a);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return B200Q_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return B200Q_ERR_MISALIGNED;
  int* status = device_status_ptr();
  if (status == nullptr) return B200Q_ERR_LAUNCH;
  if (device_cc_major() != 10) return B200Q_ERR_UNSUPPORTED_ARCH;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return decode ? launch_attn_decode(*a, workspace, status, st) : launch_attn_prefill(*a, workspace, status, st);
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

size_t b200q_attn_prefill_workspace_bytes(const b200q_attention* a) {
  return check(a, false) == B200Q_OK ? attn_prefill_workspace(*a) : 0;
}
size_t b200q_attn_decode_workspace_bytes(const b200q_attention* a) {
  return check(a, true) == B200Q_OK ? attn_decode_workspace(*a) : 0;
}

}  // extern "C"
