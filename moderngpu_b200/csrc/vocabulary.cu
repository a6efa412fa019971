// C ABI of the vocabulary operators: embedding lookup and gradient,
// distillation from a teacher's top logits, token sampling. Declarations and
// contracts: include/moderngpu_b200.h.
#include <moderngpu_b200.h>
#include <moderngpu/kernel_embedding.hxx>
#include <moderngpu/kernel_distill.hxx>
#include <moderngpu/kernel_sample.hxx>

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

bool bad_embedding_sizes(int64_t count, int rows, int width) {
  return count < 0 || rows < 0 || width < 0 || width > max_width ||
    count + rows > max_merged;
}

bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  return a_bytes > 0 && b_bytes > 0 && (uintptr_t)a < (uintptr_t)b + b_bytes &&
    (uintptr_t)b < (uintptr_t)a + a_bytes;
}

// Bytes from a matrix's first element to behind its last.
int64_t extent(int64_t count, int64_t width, int64_t stride, int size) {
  return count > 0 && width > 0 ? ((count - 1) * stride + width) * size : 0;
}

int distill(bool want_grad, int dtype, const void* logits, int64_t stride,
  int count, int vocabulary, int token_dtype, const void* tokens,
  int teacher_dtype, const void* teacher, int entries, float temperature,
  const float* weights, float* losses, void* grad, int64_t grad_stride,
  void* stream) {
  int size = real_size(dtype), token = token_size(token_dtype),
    teacher_bytes = real_size(teacher_dtype);
  if(!size || !token || !teacher_bytes) return MGPU_B200_E_UNSUPPORTED;
  // The kernel computes with log2(e) / T in 32 bits.
  float c = 1.4426950408889634f / temperature;
  if(count < 0 || vocabulary < 0 || vocabulary > max_merged || entries < 0 ||
    entries > distill_max_entries || !(temperature > 0) || !(c > 0) ||
    !(c <= FLT_MAX) || !(temperature <= FLT_MAX) ||
    bad_matrix(logits, count, vocabulary, stride, size) ||
    bad_matrix(tokens, count, entries, entries, token) ||
    bad_matrix(teacher, count, entries, entries, teacher_bytes) ||
    bad_matrix(losses, count, 1, 1, 4) || (uintptr_t)weights % 4)
    return MGPU_B200_E_INVALID;
  if(want_grad) {
    if(bad_matrix(grad, count, vocabulary, grad_stride, size))
      return MGPU_B200_E_INVALID;
    bool same = grad == logits && (grad_stride == stride || count < 2);
    if(!same && overlap(logits, extent(count, vocabulary, stride, size), grad,
      extent(count, vocabulary, grad_stride, size)))
      return MGPU_B200_E_INVALID;
  }
  return with_real(dtype, [&](auto* r) {
    typedef typename std::remove_pointer<decltype(r)>::type real_t;
    return with_real(teacher_dtype, [&](auto* h) {
      typedef typename std::remove_pointer<decltype(h)>::type teacher_t;
      return with_token(token_dtype, [&](auto* i) {
        typedef typename std::remove_pointer<decltype(i)>::type token_t;
        return guarded([&]() {
          if(want_grad)
            detail::distill_enqueue<true>((const real_t*)logits, stride, count,
              vocabulary, (const token_t*)tokens, (const teacher_t*)teacher,
              entries, temperature, weights, losses, (real_t*)grad, grad_stride,
              (cudaStream_t)stream);
          else
            detail::distill_enqueue<false>((const real_t*)logits, stride, count,
              vocabulary, (const token_t*)tokens, (const teacher_t*)teacher,
              entries, temperature, (const float*)nullptr, losses,
              (real_t*)nullptr, (int64_t)0, (cudaStream_t)stream);
        });
      });
    });
  });
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

int mgpu_b200_distill_loss(int dtype, const void* logits_device, int64_t stride,
  int count, int vocabulary, int token_dtype, const void* tokens_device,
  int teacher_dtype, const void* teacher_device, int entries, float temperature,
  float* losses_device, void* stream) {
  return distill(false, dtype, logits_device, stride, count, vocabulary,
    token_dtype, tokens_device, teacher_dtype, teacher_device, entries,
    temperature, nullptr, losses_device, nullptr, 0, stream);
}

int mgpu_b200_distill_loss_gradient(int dtype, const void* logits_device,
  int64_t stride, int count, int vocabulary, int token_dtype,
  const void* tokens_device, int teacher_dtype, const void* teacher_device,
  int entries, float temperature, const float* weights_device,
  float* losses_device, void* grad_device, int64_t grad_stride, void* stream) {
  return distill(true, dtype, logits_device, stride, count, vocabulary,
    token_dtype, tokens_device, teacher_dtype, teacher_device, entries,
    temperature, weights_device, losses_device, grad_device, grad_stride,
    stream);
}

int mgpu_b200_sample_tokens(int dtype, const void* logits_device,
  int64_t stride, int count, int vocabulary, const float* uniforms_device,
  float temperature, const float* temperatures_device, int top_k,
  const int* top_ks_device, float top_p, const float* top_ps_device,
  float min_p, const float* min_ps_device, int* tokens_device, void* stream) {
  int size = real_size(dtype);
  if(!size) return MGPU_B200_E_UNSUPPORTED;
  if(count < 0 || vocabulary < 0 || vocabulary > max_merged ||
    bad_matrix(logits_device, count, vocabulary, stride, size) ||
    bad_matrix(uniforms_device, count, 1, 1, 4) ||
    bad_matrix(tokens_device, count, 1, 1, 4) ||
    (uintptr_t)temperatures_device % 4 || (uintptr_t)top_ks_device % 4 ||
    (uintptr_t)top_ps_device % 4 || (uintptr_t)min_ps_device % 4 ||
    (!temperatures_device && !(temperature >= 0 && temperature <= FLT_MAX)) ||
    (!top_ps_device && !(top_p >= 0)) || (!min_ps_device && !(min_p >= 0 &&
      min_p <= 1)))
    return MGPU_B200_E_INVALID;
  sampling_t settings;
  settings.temperature = temperature;
  settings.top_p = top_p;
  settings.min_p = min_p;
  settings.top_k = top_k;
  settings.temperatures = temperatures_device;
  settings.top_ps = top_ps_device;
  settings.min_ps = min_ps_device;
  settings.top_ks = top_ks_device;
  return with_real(dtype, [&](auto* r) {
    typedef typename std::remove_pointer<decltype(r)>::type real_t;
    return guarded([&]() {
      detail::sample_enqueue((const real_t*)logits_device, stride, count,
        vocabulary, uniforms_device, settings, tokens_device,
        (cudaStream_t)stream);
    });
  });
}

} // extern "C"
