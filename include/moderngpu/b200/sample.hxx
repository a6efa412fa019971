// One token per row of logits, drawn by given random numbers.
//
// A row has the logits x over the vocabulary, a number u in [0, 1) and the
// settings T (temperature), k (top-k), p (top-p) and m (min-p). With the
// weights w_v = exp((x_v - max x) / T):
//   1. the k tokens of the greatest logits are kept (k <= 0: all);
//   2. of these, in falling order, the shortest run whose weight is at least p
//      times the weight of them all (p >= 1: all; one token at least);
//   3. of these, those with w_v >= m;
//   4. of these, in the order of the vocabulary, the first token whose running
//      weight exceeds u times the weight of all that are left.
// Equal logits are ordered by their index. T = 0 takes the greatest logit. A
// row with a NaN, or without a logit above -infinity, gives -1.
//
// Weights and their sums are held in 64 bits: with a vocabulary of 2^17 tokens
// a sum in 32 bits would put the border between two tokens in the wrong place
// for about one row in a hundred.
#pragma once
#include "runtime.hxx"
#include "real_types.hxx"

BEGIN_MGPU_NAMESPACE

// One number for all rows, or one for each (device arrays; null: the number).
struct sampling_t {
  float temperature = 1.0f, top_p = 1.0f, min_p = 0.0f;
  int top_k = 0;
  const float* temperatures = nullptr;
  const float* top_ps = nullptr;
  const float* min_ps = nullptr;
  const int* top_ks = nullptr;
};

#ifdef __CUDACC__

namespace detail {

// Unsigned numbers in the order of the floats; -0 and +0 are the same one.
MGPU_DEVICE __forceinline__ uint32_t order_key(float x) {
  uint32_t bits = __float_as_uint(x + 0.0f);
  return bits ^ ((int32_t)bits < 0 ? 0xffffffffu : 0x80000000u);
}
MGPU_DEVICE __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float(key ^ ((int32_t)key < 0 ? 0x80000000u :
    0xffffffffu));
}

template<int nt, typename type_t, typename op_t>
MGPU_DEVICE __forceinline__ type_t cta_fold(type_t x, op_t op, void* shared) {
  type_t* parts = (type_t*)shared;
  #pragma unroll
  for(int offset = 16; offset; offset /= 2)
    x = op(x, __shfl_xor_sync(0xffffffffu, x, offset));
  if(0 == threadIdx.x % 32) parts[threadIdx.x / 32] = x;
  __syncthreads();
  x = parts[0];
  for(int w = 1; w < nt / 32; ++w) x = op(x, parts[w]);
  __syncthreads();
  return x;
}

template<int nt, typename real_t>
struct sample_row_t {
  const real_t* x;
  int vocabulary;
  float peak;
  double scale;
  void* shared;

  MGPU_DEVICE uint32_t key(int v) const { return order_key(to_f32(x[v])); }
  MGPU_DEVICE double weight(uint32_t key) const {
    float value = key_value(key);
    return value == peak ? 1.0 : exp(((double)value - (double)peak) * scale);
  }
  // The index of the nth (from 1) token with the given key.
  MGPU_DEVICE int nth_equal(uint32_t wanted, int nth) const {
    __shared__ int found;
    if(!threadIdx.x) found = vocabulary - 1;
    int seen = 0;
    for(int first = 0; first < vocabulary; first += nt) {
      int v = first + (int)threadIdx.x;
      int mine = v < vocabulary && key(v) == wanted;
      int here = __syncthreads_count(mine);
      if(seen + here >= nth) {
        // The tile that holds it: count in front of each thread.
        int* counts = (int*)shared;
        unsigned votes = __ballot_sync(0xffffffffu, mine);
        if(0 == threadIdx.x % 32) counts[threadIdx.x / 32] = __popc(votes);
        __syncthreads();
        int before = seen;
        for(int w = 0; w < (int)threadIdx.x / 32; ++w) before += counts[w];
        before += __popc(votes & ((1u << (threadIdx.x % 32)) - 1));
        if(mine && before + 1 == nth) found = v;
        break;
      }
      seen += here;
    }
    __syncthreads();
    int at = found;
    __syncthreads();
    return at;
  }
};

template<int nt, typename real_t>
__global__ void __launch_bounds__(nt)
sample_k(const real_t* logits, int64_t stride, int vocabulary,
  const float* uniforms, sampling_t settings, int* tokens) {
  __shared__ double shared[nt / 32];
  __shared__ int hist[256];
  __shared__ uint32_t chosen;
  __shared__ int chosen_left;

  int64_t at = blockIdx.x;
  int tid = threadIdx.x;
  sample_row_t<nt, real_t> row { logits + at * stride, vocabulary, 0, 0,
    shared };
  float temperature = settings.temperatures ? settings.temperatures[at] :
    settings.temperature;
  float top_p = settings.top_ps ? settings.top_ps[at] : settings.top_p;
  float min_p = settings.min_ps ? settings.min_ps[at] : settings.min_p;
  int top_k = settings.top_ks ? settings.top_ks[at] : settings.top_k;
  auto greater = [](uint32_t a, uint32_t b) { return a < b ? b : a; };
  auto lesser = [](int a, int b) { return a < b ? a : b; };
  auto add = [](double a, double b) { return a + b; };

  uint32_t peak_key = 0;
  bool nan = false;
  for(int v = tid; v < vocabulary; v += nt) {
    float x = to_f32(row.x[v]);
    nan = nan || isnan(x);
    peak_key = greater(peak_key, order_key(x));
  }
  nan = __syncthreads_or(nan);
  peak_key = cta_fold<nt>(peak_key, greater, shared);
  row.peak = key_value(peak_key);
  if(nan || !(row.peak > -INFINITY)) {
    if(!tid) tokens[at] = -1;
    return;
  }
  if(!(temperature > 0)) {
    int best = vocabulary;
    for(int v = tid; v < vocabulary; v += nt)
      if(row.key(v) == peak_key) { best = v; break; }
    best = cta_fold<nt>(best, lesser, shared);
    if(!tid) tokens[at] = best;
    return;
  }
  row.scale = 1.0 / (double)temperature;

  // What is kept: keys above `least`, and those equal to it up to index `last`.
  uint32_t least = 0;
  int last = vocabulary;
  auto kept = [&](uint32_t key, int v) {
    return key > least || (key == least && v <= last);
  };
  if(top_k > 0 && top_k < vocabulary) {
    uint32_t prefix = 0;
    int left = top_k;
    for(int shift = 24; shift >= 0; shift -= 8) {
      if(tid < 256) hist[tid] = 0;
      __syncthreads();
      for(int v = tid; v < vocabulary; v += nt) {
        uint32_t key = row.key(v);
        if(24 == shift || key >> (shift + 8) == prefix >> (shift + 8))
          atomicAdd(&hist[(key >> shift) & 255], 1);
      }
      __syncthreads();
      if(!tid) {
        int d = 255;
        while(d > 0 && hist[d] < left) left -= hist[d--];
        chosen = prefix | ((uint32_t)d << shift);
        chosen_left = left;
      }
      __syncthreads();
      prefix = chosen;
      left = chosen_left;
      __syncthreads();
    }
    least = prefix;
    last = row.nth_equal(least, left);
  }

  auto mass_from = [&](uint32_t from, bool above) {
    double sum = 0;
    for(int v = tid; v < vocabulary; v += nt) {
      uint32_t key = row.key(v);
      if(kept(key, v) && (above ? key > from : key >= from))
        sum += row.weight(key);
    }
    return cta_fold<nt>(sum, add, shared);
  };
  if(top_p < 1) {
    double target = (double)top_p * mass_from(0, false);
    uint32_t border = 0;
    for(int bit = 31; bit >= 0; --bit) {
      uint32_t from = border | (1u << bit);
      if(from <= peak_key && mass_from(from, false) >= target) border = from;
    }
    // How many of the tokens at the border.
    double above = mass_from(border, true);
    double one = row.weight(border);
    double need = ceil((target - above) / one);
    int nth = need > 1 ? (need < vocabulary ? (int)need : vocabulary) : 1;
    int limit = row.nth_equal(border, nth);
    if(border > least) {
      least = border;
      last = limit;
    } else
      last = lesser(last, limit);
  }

  auto left_weight = [&](int v) {
    if(v >= vocabulary) return 0.0;
    uint32_t key = row.key(v);
    if(!kept(key, v)) return 0.0;
    double w = row.weight(key);
    return w >= (double)min_p || key == peak_key ? w : 0.0;
  };
  double mass = 0;
  for(int first = 0; first < vocabulary; first += nt)
    mass += cta_fold<nt>(left_weight(first + tid), add, shared);
  double target = (double)uniforms[at] * mass;
  double before = 0;
  int fallback = 0;
  for(int first = 0; first < vocabulary; first += nt) {
    double w = left_weight(first + tid);
    double sum = w;
    #pragma unroll
    for(int offset = 1; offset < 32; offset *= 2) {
      double y = __shfl_up_sync(0xffffffffu, sum, offset);
      if(tid % 32 >= offset) sum += y;
    }
    if(31 == tid % 32) shared[tid / 32] = sum;
    __syncthreads();
    double ahead = before;
    for(int i = 0; i < tid / 32; ++i) ahead += shared[i];
    for(int i = 0; i < nt / 32; ++i) before += shared[i];
    __syncthreads();
    bool over = w > 0 && ahead + sum > target;
    int hit = cta_fold<nt>(over ? first + tid : vocabulary, lesser, shared);
    if(hit < vocabulary) {
      if(!tid) tokens[at] = hit;
      return;
    }
    // Where the last sum rounds to below the target, the last token left.
    fallback = cta_fold<nt>(w > 0 ? first + tid : fallback,
      [](int a, int b) { return a < b ? b : a; }, shared);
  }
  if(!tid) tokens[at] = fallback;
}

template<typename real_t>
void sample_enqueue(const real_t* logits, int64_t stride, int count,
  int vocabulary, const float* uniforms, const sampling_t& settings,
  int* tokens, cudaStream_t stream) {
  if(!count) return;
  enum { nt = 1024 };
  sample_k<nt><<<(unsigned)count, nt, 0, stream>>>(logits, stride, vocabulary,
    uniforms, settings, tokens);
  throw_on_error(cudaGetLastError());
}

} // namespace detail

////////////////////////////////////////////////////////////////////////////////
// Public entry point: rows of logits are `stride` elements apart.

template<typename real_t>
void sample_tokens(const real_t* logits, int64_t stride, int count,
  int vocabulary, const float* uniforms, const sampling_t& settings,
  int* tokens, context_t& context) {
  static_assert(detail::is_model_real<real_t>::value,
    "sample_tokens takes float, __half or __nv_bfloat16");
  detail::throw_on_device_status();
  detail::sample_enqueue(logits, stride, count, vocabulary, uniforms, settings,
    tokens, context.stream());
}

#endif // __CUDACC__

END_MGPU_NAMESPACE
