// Shared by the attention kernels' translation units.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/b200q.h"

namespace b200q {

// b200q_view's rules.
inline int check_view(const b200q_view& x) {
  if (x.data == nullptr) return B200Q_ERR_NULL_POINTER;
  for (int64_t s : {x.page, x.token, x.head})
    if (s % 8 != 0 || s < 0 || s >= (int64_t{1} << 39)) return B200Q_ERR_UNSUPPORTED_SHAPE;
  return (reinterpret_cast<uintptr_t>(x.data) & 15u) != 0 ? B200Q_ERR_MISALIGNED : B200Q_OK;
}

}  // namespace b200q
