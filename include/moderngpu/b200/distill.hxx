// Distillation from a teacher's top logits.
//
// A row holds a student's logits s over the whole vocabulary, and the teacher's
// logits t_k of a few tokens j_k. With the temperature T,
//   p = softmax over the row's entries k of t_k / T,
//   q = softmax over the vocabulary of s_v / T,
//   loss = T^2 * sum_k p_k (log p_k - log q[j_k]),
//   d loss / d s_v = T * (q_v - sum of the p_k with j_k = v).
// The factor T^2 keeps the size of the gradient when T changes.
//
// An entry whose token lies outside of the vocabulary is unused. A row without
// a used entry (or with none above -infinity), a row whose logits are all
// -infinity, and a row of weight 0 have loss 0 and gradient 0; the logits of
// the first and the last are not read.
#pragma once
#include "runtime.hxx"
#include "real_types.hxx"

BEGIN_MGPU_NAMESPACE

enum { distill_max_entries = 1024 };

#ifdef __CUDACC__

namespace detail {

// 2^x to about 2 units in the last place; results below 2^-126 are 0, which
// adds less than 2^-100 to any sum that holds the row's maximum (2^0).
MGPU_DEVICE __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A running maximum with the sum of 2^((x - peak) * c) over the values seen.
struct peak_sum_t {
  float peak, sum;
};
// Both parts' sums relative to the greater peak. A part that has seen no value
// above -infinity has sum 0 or NaN, and its -infinity is no distance.
MGPU_DEVICE __forceinline__ peak_sum_t merge(peak_sum_t a, peak_sum_t b,
  float c) {
  float peak = fmaxf(a.peak, b.peak);
  float base = peak == -INFINITY ? 0.0f : peak;
  return peak_sum_t { peak, a.sum * exp2_fast((a.peak - base) * c) +
    b.sum * exp2_fast((b.peak - base) * c) };
}

template<int nt>
MGPU_DEVICE __forceinline__ peak_sum_t cta_merge(peak_sum_t x, float c,
  peak_sum_t* shared) {
  #pragma unroll
  for(int offset = 16; offset; offset /= 2) {
    peak_sum_t y { __shfl_xor_sync(0xffffffffu, x.peak, offset),
      __shfl_xor_sync(0xffffffffu, x.sum, offset) };
    x = merge(x, y, c);
  }
  if(0 == threadIdx.x % 32) shared[threadIdx.x / 32] = x;
  __syncthreads();
  x = shared[0];
  for(int w = 1; w < nt / 32; ++w) x = merge(x, shared[w], c);
  __syncthreads();
  return x;
}

template<int nt>
MGPU_DEVICE __forceinline__ float cta_sum(float x, float* shared) {
  #pragma unroll
  for(int offset = 16; offset; offset /= 2)
    x += __shfl_xor_sync(0xffffffffu, x, offset);
  if(0 == threadIdx.x % 32) shared[threadIdx.x / 32] = x;
  __syncthreads();
  x = shared[0];
  for(int w = 1; w < nt / 32; ++w) x += shared[w];
  __syncthreads();
  return x;
}

// One CTA per row: the teacher's entries, one pass over the logits for the
// maximum and the sum, the loss, and with want_grad a second pass for the
// gradient.
template<int nt, int pack, bool want_grad, typename real_t, typename teacher_t,
  typename token_t>
__global__ void __launch_bounds__(nt)
distill_k(const real_t* logits, int64_t stride, int vocabulary,
  const token_t* tokens, const teacher_t* teacher, int entries,
  float temperature, const float* weights, float* losses, real_t* grad,
  int64_t grad_stride) {
  typedef pack_t<real_t, pack> word_t;
  __shared__ float p[distill_max_entries];
  __shared__ float student[distill_max_entries];
  __shared__ int at[distill_max_entries];
  __shared__ peak_sum_t merged[nt / 32];
  __shared__ float summed[nt / 32];

  int64_t row = blockIdx.x;
  int tid = threadIdx.x;
  const real_t* x = logits + row * stride;
  const float c = 1.4426950408889634f / temperature;
  float weight = weights ? weights[row] : 1.0f;

  // The teacher's distribution. A NaN stays one.
  peak_sum_t t { -INFINITY, 0.0f };
  for(int k = tid; k < entries; k += nt) {
    int64_t j = (int64_t)tokens[row * entries + k];
    bool used = j >= 0 && j < vocabulary && weight != 0;
    at[k] = used ? (int)j : -1;
    p[k] = used ? to_f32(teacher[row * entries + k]) : -INFINITY;
    student[k] = used ? to_f32(x[j]) : 0.0f;
    t = merge(t, peak_sum_t { p[k], p[k] == -INFINITY ? 0.0f :
      (isnan(p[k]) ? p[k] : 1.0f) }, c);
  }
  t = cta_merge<nt>(t, c, merged);
  bool taught = t.peak > -INFINITY || isnan(t.sum);
  if(taught) {
    float log_sum = logf(t.sum);
    // One pass over the student's logits.
    peak_sum_t s { -INFINITY, 0.0f };
    for(int v = tid * pack; v < vocabulary; v += nt * pack) {
      word_t word = *(const word_t*)(x + v);
      float peak = s.peak;
      #pragma unroll
      for(int j = 0; j < pack; ++j) peak = fmaxf(peak, to_f32(word.v[j]));
      float base = peak == -INFINITY ? 0.0f : peak;
      float sum = s.sum * exp2_fast((s.peak - base) * c);
      #pragma unroll
      for(int j = 0; j < pack; ++j)
        sum += exp2_fast((to_f32(word.v[j]) - base) * c);
      s = peak_sum_t { peak, sum };
    }
    s = cta_merge<nt>(s, c, merged);
    bool empty = s.peak == -INFINITY && !isnan(s.sum);
    float loss = 0;
    float log_mass = logf(s.sum);
    for(int k = tid; k < entries; k += nt) {
      float log_p = (p[k] - t.peak) / temperature - log_sum;
      float prob = at[k] < 0 ? 0.0f : expf(log_p);
      float log_q = (student[k] - s.peak) / temperature - log_mass;
      if(prob != 0) loss += prob * (log_p - log_q);
      p[k] = prob;
    }
    loss = cta_sum<nt>(loss, summed);
    if(!tid) losses[row] = empty ? 0.0f : temperature * temperature * loss;
    if(want_grad) {
      real_t* g = grad + row * grad_stride;
      float factor = weight * temperature / s.sum;
      for(int v = tid * pack; v < vocabulary; v += nt * pack) {
        word_t word = *(const word_t*)(x + v);
        #pragma unroll
        for(int j = 0; j < pack; ++j)
          word.v[j] = from_f32<real_t>(empty ? 0.0f : factor *
            exp2_fast((to_f32(word.v[j]) - s.peak) * c));
        *(word_t*)(g + v) = word;
      }
      __syncthreads();
      // The teacher's tokens again, each with all of its entries.
      for(int k = tid; k < entries; k += nt) {
        if(at[k] < 0 || empty) continue;
        float sum = 0;
        for(int i = 0; i < entries; ++i)
          if(at[i] == at[k]) sum += p[i];
        g[at[k]] = from_f32<real_t>(factor *
          exp2_fast((student[k] - s.peak) * c) - weight * temperature * sum);
      }
    }
  } else {
    if(!tid) losses[row] = 0.0f;
    if(want_grad) {
      word_t word;
      #pragma unroll
      for(int j = 0; j < pack; ++j) word.v[j] = from_f32<real_t>(0.0f);
      for(int v = tid * pack; v < vocabulary; v += nt * pack)
        *(word_t*)(grad + row * grad_stride + v) = word;
    }
  }
}

template<bool want_grad, typename real_t, typename teacher_t, typename token_t>
void distill_enqueue(const real_t* logits, int64_t stride, int count,
  int vocabulary, const token_t* tokens, const teacher_t* teacher, int entries,
  float temperature, const float* weights, float* losses, real_t* grad,
  int64_t grad_stride, cudaStream_t stream) {
  if(!count) return;
  int pack = pack_limit(logits, stride, vocabulary, (int)sizeof(real_t));
  if(want_grad)
    pack = min(pack, pack_limit(grad, grad_stride, vocabulary,
      (int)sizeof(real_t)));
  auto launch = [&](auto tag) {
    enum { nt = 512 };
    distill_k<nt, decltype(tag)::value, want_grad, real_t, teacher_t, token_t>
      <<<(unsigned)count, nt, 0, stream>>>(logits, stride, vocabulary, tokens,
        teacher, entries, temperature, weights, losses, grad, grad_stride);
  };
  switch(pack) {
    case 8: launch(std::integral_constant<int,
      (sizeof(real_t) == 2 ? 8 : 4)>()); break;
    case 4: launch(std::integral_constant<int, 4>()); break;
    case 2: launch(std::integral_constant<int, 2>()); break;
    default: launch(std::integral_constant<int, 1>()); break;
  }
  throw_on_error(cudaGetLastError());
}

} // namespace detail

////////////////////////////////////////////////////////////////////////////////
// Public entry points. `tokens` and `teacher` are dense, `entries` to a row (at
// most distill_max_entries); rows of logits are `stride` elements apart.

template<typename real_t, typename teacher_t, typename token_t>
void distill_loss(const real_t* logits, int64_t stride, int count,
  int vocabulary, const token_t* tokens, const teacher_t* teacher, int entries,
  float temperature, float* losses, context_t& context) {
  detail::throw_on_device_status();
  detail::distill_enqueue<false>(logits, stride, count, vocabulary, tokens,
    teacher, entries, temperature, (const float*)nullptr, losses,
    (real_t*)nullptr, (int64_t)0, context.stream());
}

// Also grad = weight * d loss / d logits, row by row (weights may be null: 1).
// `grad` may be `logits` itself, with the same stride.
template<typename real_t, typename teacher_t, typename token_t>
void distill_loss_gradient(const real_t* logits, int64_t stride, int count,
  int vocabulary, const token_t* tokens, const teacher_t* teacher, int entries,
  float temperature, const float* weights, float* losses, real_t* grad,
  int64_t grad_stride, context_t& context) {
  detail::throw_on_device_status();
  detail::distill_enqueue<true>(logits, stride, count, vocabulary, tokens,
    teacher, entries, temperature, weights, losses, grad, grad_stride,
    context.stream());
}

#endif // __CUDACC__

END_MGPU_NAMESPACE
