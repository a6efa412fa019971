// The number types of the vocabulary operators (embedding lookup and
// gradient, distillation, sampling): 32-bit floats and the two 16-bit formats,
// all computed with in 32 bits or more and rounded once when they are stored.
#pragma once
#include "runtime.hxx"
#include <atomic>

#ifdef __CUDACC__
#include <cuda_bf16.h>
#include <cuda_fp16.h>

BEGIN_MGPU_NAMESPACE
namespace detail {

template<typename real_t>
struct is_model_real : std::false_type { };
template<> struct is_model_real<float> : std::true_type { };
template<> struct is_model_real<__half> : std::true_type { };
template<> struct is_model_real<__nv_bfloat16> : std::true_type { };

MGPU_DEVICE __forceinline__ float to_f32(float x) { return x; }
MGPU_DEVICE __forceinline__ float to_f32(__half x) { return __half2float(x); }
MGPU_DEVICE __forceinline__ float to_f32(__nv_bfloat16 x) {
  return __bfloat162float(x);
}

// One rounding to nearest, ties to even.
template<typename real_t>
MGPU_DEVICE __forceinline__ real_t from_f32(float x);
template<>
MGPU_DEVICE __forceinline__ float from_f32<float>(float x) { return x; }
template<>
MGPU_DEVICE __forceinline__ __half from_f32<__half>(float x) {
  return __float2half_rn(x);
}
template<>
MGPU_DEVICE __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// `count` neighbouring values that are loaded and stored as one word of up to
// 16 bytes (two words for a pack of 32).
template<typename real_t, int count>
struct MGPU_ALIGN((sizeof(real_t) * count > 16 ? 16 : sizeof(real_t) * count))
pack_t {
  real_t v[count];
};

// A store of data that this kernel does not read again: first to leave the L2.
template<typename real_t, int count>
MGPU_DEVICE __forceinline__ void store_streaming(pack_t<real_t, count>* to,
  const pack_t<real_t, count>& word) {
  enum { size = sizeof(pack_t<real_t, count>) };
  static_assert(2 == size || 4 == size || 8 == size || 16 == size, "one word");
  if constexpr (16 == size) {
    uint4 bits;
    memcpy(&bits, &word, 16);
    __stcs((uint4*)to, bits);
  } else if constexpr (8 == size) {
    uint2 bits;
    memcpy(&bits, &word, 8);
    __stcs((uint2*)to, bits);
  } else if constexpr (4 == size) {
    uint32_t bits;
    memcpy(&bits, &word, 4);
    __stcs((uint32_t*)to, bits);
  } else {
    uint16_t bits;
    memcpy(&bits, &word, 2);
    __stcs((unsigned short*)to, bits);
  }
}

// The widest pack, in elements of `size` bytes, that divides `width` and that
// every row starts on a boundary of: rows `stride` elements apart from `base`.
inline int pack_limit(const void* base, int64_t stride, int64_t width,
  int size) {
  int pack = 16 / size;
  while(pack > 1 && ((uintptr_t)base % (size_t)(pack * size) ||
    stride % pack || width % pack)) pack /= 2;
  return pack;
}

// A pack of 1, 2, 4 or 8 elements as a constant for f.
template<typename func_t>
void with_pack(int pack, func_t f) {
  switch(pack) {
    case 8: f(std::integral_constant<int, 8>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    case 2: f(std::integral_constant<int, 2>()); break;
    default: f(std::integral_constant<int, 1>()); break;
  }
}

// Allows a kernel its dynamic shared memory, once per device. tag_t...: what
// tells its instantiations apart.
template<typename... tag_t, typename kernel_t>
void set_dynamic_smem(kernel_t kernel, int bytes) {
  static std::atomic<bool> done[64] = { };
  int device = 0;
  throw_on_error(cudaGetDevice(&device));
  if(device < 64 && done[device].load(std::memory_order_acquire)) return;
  throw_on_error(cudaFuncSetAttribute(kernel,
    cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if(device < 64) done[device].store(true, std::memory_order_release);
}

} // namespace detail
END_MGPU_NAMESPACE

#endif // __CUDACC__
