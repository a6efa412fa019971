// C ABI of the distillation from a teacher's top logits. Declarations and
// contracts: include/moderngpu_b200.h.
#include "vocabulary.h"
#include <moderngpu/kernel_distill.hxx>

namespace {

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

} // extern "C"
