// C ABI of the token sampling. Declarations and contracts:
// include/moderngpu_b200.h.
#include "vocabulary.h"
#include <moderngpu/kernel_sample.hxx>

extern "C" {

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
