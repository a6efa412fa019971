// Shared by the C entry points of the vocabulary operators: return codes, type
// dispatch, and the checks of their arguments.
#pragma once
#include <moderngpu_b200.h>
#include <moderngpu/b200/real_types.hxx>

using namespace mgpu;

namespace {

// Runs f and turns what the templates throw into a return code.
template<typename func_t>
int guarded(func_t f) {
  try {
    f();
  } catch(cuda_exception_t& e) {
    cudaGetLastError();
    return MGPU_B200_E_CUDA + (int)e.result;
  } catch(...) {
    return MGPU_B200_E_CUDA + (int)cudaErrorUnknown;
  }
  return MGPU_B200_OK;
}

template<typename func_t>
int with_real(int dtype, func_t f) {
  switch(dtype) {
    case MGPU_B200_F32: return f((float*)nullptr);
    case MGPU_B200_F16: return f((__half*)nullptr);
    case MGPU_B200_BF16: return f((__nv_bfloat16*)nullptr);
  }
  return MGPU_B200_E_UNSUPPORTED;
}

template<typename func_t>
int with_token(int dtype, func_t f) {
  switch(dtype) {
    case MGPU_B200_I32: return f((int32_t*)nullptr);
    case MGPU_B200_I64: return f((int64_t*)nullptr);
  }
  return MGPU_B200_E_UNSUPPORTED;
}

int real_size(int dtype) {
  switch(dtype) {
    case MGPU_B200_F32: return 4;
    case MGPU_B200_F16: case MGPU_B200_BF16: return 2;
  }
  return 0;
}
int token_size(int dtype) {
  return MGPU_B200_I32 == dtype ? 4 : MGPU_B200_I64 == dtype ? 8 : 0;
}

// A matrix argument: present where it has elements, aligned to them, rows at
// least `width` elements apart.
bool bad_matrix(const void* p, int64_t count, int64_t width, int64_t stride,
  int size) {
  return (count > 0 && width > 0 && !p) || (uintptr_t)p % (size_t)size ||
    (count > 1 && stride < width);
}

enum { max_merged = 0x7fffffff - 65536, max_width = 1 << 20 };

bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  return a_bytes > 0 && b_bytes > 0 && (uintptr_t)a < (uintptr_t)b + b_bytes &&
    (uintptr_t)b < (uintptr_t)a + a_bytes;
}

// Bytes from a matrix's first element to behind its last.
int64_t extent(int64_t count, int64_t width, int64_t stride, int size) {
  return count > 0 && width > 0 ? ((count - 1) * stride + width) * size : 0;
}

} // namespace
