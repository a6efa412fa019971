// C ABI of the embedding lookup and gradient. Declarations and contracts:
// include/moderngpu_b200.h.
#include "vocabulary.h"
#include <moderngpu/kernel_embedding.hxx>

namespace {

bool bad_embedding_sizes(int64_t count, int rows, int width) {
  return count < 0 || rows < 0 || width < 0 || width > max_width ||
    count + rows > max_merged;
}

} // namespace

extern "C" {

int mgpu_b200_embedding_lookup(int dtype, const void* table_device, int rows,
  int width, int64_t stride, int token_dtype, const void* tokens_device,
  int count, float scale, void* output_device, void* stream) {
  int size = real_size(dtype), token = token_size(token_dtype);
  if(!size || !token) return MGPU_B200_E_UNSUPPORTED;
  if(bad_embedding_sizes(count, rows, width) ||
    bad_matrix(table_device, rows, width, stride, size) ||
    bad_matrix(tokens_device, count, 1, 1, token) ||
    bad_matrix(output_device, count, width, width, size) ||
    overlap(table_device, extent(rows, width, stride, size), output_device,
      extent(count, width, width, size)))
    return MGPU_B200_E_INVALID;
  return with_real(dtype, [&](auto* r) {
    typedef typename std::remove_pointer<decltype(r)>::type real_t;
    return with_token(token_dtype, [&](auto* i) {
      typedef typename std::remove_pointer<decltype(i)>::type token_t;
      return guarded([&]() {
        detail::embedding_lookup_enqueue((const real_t*)table_device, rows,
          width, stride, (const token_t*)tokens_device, count, scale,
          (real_t*)output_device, (cudaStream_t)stream);
      });
    });
  });
}

size_t mgpu_b200_embedding_gradient_workspace_bytes(int count, int rows,
  int width, int accumulate) {
  if(bad_embedding_sizes(count, rows, width)) return 0;
  size_t bytes = detail::embedding_plan_t(count, rows, width).bytes;
  return bytes ? bytes : 128;
}

int mgpu_b200_embedding_gradient(int dtype, const void* grad_device,
  int64_t stride, int width, int token_dtype, const void* tokens_device,
  int count, int rows, float scale, int accumulate, int output_dtype,
  void* output_device, void* workspace_device, size_t workspace_bytes,
  void* stream) {
  int size = real_size(dtype), token = token_size(token_dtype),
    out_size = real_size(output_dtype);
  if(!size || !token || !out_size ||
    (output_dtype != dtype && MGPU_B200_F32 != output_dtype))
    return MGPU_B200_E_UNSUPPORTED;
  if(bad_embedding_sizes(count, rows, width) ||
    bad_matrix(grad_device, count, width, stride, size) ||
    bad_matrix(tokens_device, count, 1, 1, token) ||
    bad_matrix(output_device, rows, width, width, out_size) ||
    overlap(grad_device, extent(count, width, stride, size), output_device,
      extent(rows, width, width, out_size)) ||
    !workspace_device || (uintptr_t)workspace_device % 128)
    return MGPU_B200_E_INVALID;
  if(workspace_bytes < mgpu_b200_embedding_gradient_workspace_bytes(count, rows,
    width, accumulate)) return MGPU_B200_E_WORKSPACE;
  return with_real(dtype, [&](auto* r) {
    typedef typename std::remove_pointer<decltype(r)>::type real_t;
    return with_token(token_dtype, [&](auto* i) {
      typedef typename std::remove_pointer<decltype(i)>::type token_t;
      return guarded([&]() {
        if(output_dtype == dtype)
          detail::embedding_gradient_enqueue((const real_t*)grad_device, stride,
            width, (const token_t*)tokens_device, count, rows, scale,
            0 != accumulate, (real_t*)output_device, workspace_device,
            (cudaStream_t)stream);
        else
          detail::embedding_gradient_enqueue((const real_t*)grad_device, stride,
            width, (const token_t*)tokens_device, count, rows, scale,
            0 != accumulate, (float*)output_device, workspace_device,
            (cudaStream_t)stream);
      });
    });
  });
}

} // extern "C"
