// Host helpers of the C ABI entry points: errors and checks of arguments.
#pragma once

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/cascade_b200.h"
#include "kernels.h"

namespace cascade {
namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_error(code, buf);
}

int finish(const char* op, cudaError_t e) {
  if (e == cudaSuccess) return CASCADE_OK;
  return fail(CASCADE_ERR_CUDA, "%s: CUDA error %d (%s)", op, static_cast<int>(e), cudaGetErrorString(e));
}

bool misaligned(const void* p, uintptr_t bytes = 16) { return reinterpret_cast<uintptr_t>(p) & (bytes - 1); }
bool half_type(int32_t t) { return t == CASCADE_BF16 || t == CASCADE_FP16; }
constexpr int64_t kI32 = INT32_MAX;

int check_workspace(const char* op, const void* ws, size_t have, size_t need) {
  if (need && (!ws || have < need))
    return fail(CASCADE_ERR_WORKSPACE, "%s: workspace too small (%zu bytes, need %zu)", op, have, need);
  if (need && misaligned(ws)) return fail(CASCADE_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned", op);
  return CASCADE_OK;
}

}  // namespace
}  // namespace cascade
