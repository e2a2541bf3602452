// Host-side internals of the vmoe_ops context, shared by dense.cu and grad_norm.cu.
#pragma once

#include <stdarg.h>

#include <string>

#include "moe_host.h"

struct vmoe_ops {
  int device = 0;
  int num_sms = 148;
  bool sm100 = false;
  int* status = nullptr;
  char err[512] = "";
};

namespace vmoe_host {

inline int ops_fail(vmoe_ops* o, int code, const char* fmt, ...) {
  if (o) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(o->err, sizeof(o->err), fmt, ap);
    va_end(ap);
  }
  return code;
}

inline int ops_cuda_fail(vmoe_ops* o, cudaError_t e, const char* what) {
  return ops_fail(o, VMOE_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// Carves a workspace into 256-byte aligned parts.  Without a base it only counts, so the
// size functions and the calls lay a workspace out by the same code.
struct Arena {
  char* base = nullptr;
  size_t off = 0;
  template <typename T = void>
  T* take(size_t bytes) {
    char* p = base ? base + off : nullptr;
    off += (bytes + 255) & ~static_cast<size_t>(255);
    return reinterpret_cast<T*>(p);
  }
};

}  // namespace vmoe_host
