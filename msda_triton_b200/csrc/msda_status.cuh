// msda_status.cuh -- argument checks and error reports shared by the entry
// points outside msda_capi.cu.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/msda_b200.h"

namespace msda {

int set_last_error(int code, const char* msg);  // msda_capi.cu: feeds msda_last_error()

inline int report(int code, const char* fmt, ...) {
  char msg[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  return set_last_error(code, msg);
}

inline int report_ok() { return set_last_error(MSDA_SUCCESS, ""); }

inline int report_cuda(cudaError_t err, const char* what) {
  return err == cudaSuccess
             ? report_ok()
             : report(MSDA_ERROR_CUDA, "%s: %s", what, cudaGetErrorString(err));
}

inline int64_t elem_bytes(int dtype) {
  return dtype == MSDA_FLOAT32 ? 4 : dtype == MSDA_FLOAT16 || dtype == MSDA_BFLOAT16 ? 2 : 0;
}

inline bool is_aligned(const void* p, int64_t a) {
  return (reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(a)) == 0;
}

}  // namespace msda
