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
// -infinity, and a row of weight 0 have loss 0 and gradient 0, whatever else
// they hold.
#pragma once
#include "runtime.hxx"
#include "real_types.hxx"
#include "ptx.hxx"
#include "tile_state.hxx"
#ifdef __CUDACC__
#include <cooperative_groups.h>
#endif

BEGIN_MGPU_NAMESPACE

enum { distill_max_entries = 1024, distill_max_cluster = 8 };

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

MGPU_DEVICE __forceinline__ peak_sum_t warp_merge(peak_sum_t x, float c) {
  #pragma unroll
  for(int offset = 16; offset; offset /= 2) {
    peak_sum_t y { __shfl_xor_sync(0xffffffffu, x.peak, offset),
      __shfl_xor_sync(0xffffffffu, x.sum, offset) };
    x = merge(x, y, c);
  }
  return x;
}

// The teacher's arrays, of any type: read once per row, by few threads.
struct distill_teacher_t {
  const void* tokens;
  const void* logits;
  int wide, kind;                  // 64-bit tokens; 0 float, 1 half, 2 bfloat16
  int entries;
  MGPU_DEVICE int64_t token(int64_t i) const {
    return wide ? ((const int64_t*)tokens)[i] : ((const int*)tokens)[i];
  }
  MGPU_DEVICE float logit(int64_t i) const {
    switch(kind) {
      case 1: return to_f32(((const __half*)logits)[i]);
      case 2: return to_f32(((const __nv_bfloat16*)logits)[i]);
    }
    return ((const float*)logits)[i];
  }
};
inline int teacher_kind(const float*) { return 0; }
inline int teacher_kind(const __half*) { return 1; }
inline int teacher_kind(const __nv_bfloat16*) { return 2; }

// Rows of the logits and of the gradient that begin at different places of a
// 16-byte word: one CTA to a row, element by element, the second pass from the
// L2.
template<int nt, typename real_t>
__global__ void __launch_bounds__(nt)
distill_apart_k(const real_t* logits, int64_t stride, int vocabulary,
  distill_teacher_t teacher, float temperature, const float* weights,
  float* losses, real_t* grad, int64_t grad_stride) {
  enum { warps = nt / 32 };
  extern __shared__ int distill_memory[];
  __shared__ peak_sum_t part[warps], teacher_part[warps];
  __shared__ float loss_part[warps];
  int entries = teacher.entries;
  int* at = distill_memory;                  // -1: unused
  float* p = (float*)(distill_memory + entries);
  float* student = p + entries;
  int tid = (int)threadIdx.x, lane = tid % 32, warp = tid / 32;
  int64_t row = blockIdx.x;
  const real_t* x = logits + row * stride;
  real_t* g = grad + row * grad_stride;
  const float c = 1.4426950408889634f / temperature;
  auto weight_of = [](float value) {
    return value == -INFINITY ? 0.0f :
      isnan(value) || value == INFINITY ? NAN : 1.0f;
  };

  float weight = weights ? weights[row] : 1.0f;
  peak_sum_t t { -INFINITY, 0.0f };
  for(int k = tid; k < entries; k += nt) {
    int64_t j = teacher.token(row * entries + k);
    bool used = j >= 0 && j < vocabulary && weight != 0;
    at[k] = used ? (int)j : -1;
    p[k] = used ? teacher.logit(row * entries + k) : -INFINITY;
    student[k] = used ? to_f32(x[j]) : 0.0f;
    t = merge(t, peak_sum_t { p[k], weight_of(p[k]) }, c);
  }
  peak_sum_t s { -INFINITY, 0.0f };
  #pragma unroll 4
  for(int v = tid; v < vocabulary; v += nt) {
    float value = to_f32(x[v]);
    s = merge(s, peak_sum_t { value, weight_of(value) }, c);
  }
  t = warp_merge(t, c);
  s = warp_merge(s, c);
  if(!lane) {
    teacher_part[warp] = t;
    part[warp] = s;
  }
  __syncthreads();
  const peak_sum_t nothing { -INFINITY, 0.0f };
  t = warp_merge(lane < warps ? teacher_part[lane] : nothing, c);
  s = warp_merge(lane < warps ? part[lane] : nothing, c);
  bool taught = t.peak > -INFINITY || isnan(t.sum);
  bool none = !taught || (s.peak == -INFINITY && !isnan(s.sum));
  float log_sum = logf(t.sum), log_mass = logf(s.sum), loss = 0;
  for(int k = tid; k < entries; k += nt) {
    float log_p = (p[k] - t.peak) / temperature - log_sum;
    float prob = taught && p[k] != -INFINITY ? expf(log_p) : 0.0f;
    if(prob != 0)
      loss += prob * (log_p - ((student[k] - s.peak) / temperature - log_mass));
    else
      at[k] = -1;
    p[k] = prob;
  }
  #pragma unroll
  for(int offset = 16; offset; offset /= 2)
    loss += __shfl_xor_sync(0xffffffffu, loss, offset);
  if(!lane) loss_part[warp] = loss;

  float factor = none ? 0.0f : weight * temperature / s.sum;
  #pragma unroll 4
  for(int v = tid; v < vocabulary; v += nt)
    g[v] = from_f32<real_t>(none ? 0.0f :
      factor * exp2_fast((to_f32(x[v]) - s.peak) * c));
  __syncthreads();
  if(!tid) {
    loss = 0;
    for(int w = 0; w < warps; ++w) loss += loss_part[w];
    losses[row] = none ? 0.0f : temperature * temperature * loss;
  }
  // The teacher's tokens again, each with all of its entries.
  for(int k = tid; k < entries && !none; k += nt) {
    if(at[k] < 0) continue;
    float taken = 0;
    for(int i = 0; i < entries; ++i)
      if(at[i] == at[k]) taken += p[i];
    g[at[k]] = from_f32<real_t>(factor *
      exp2_fast((student[k] - s.peak) * c) - weight * temperature * taken);
  }
}

// The rows stream through a ring of landing buffers that one thread keeps filled
// by bulk copies, without a pause between rows: each row (or a CTA's part of it)
// passes once for its peak and mass and, with want_grad, at once again for the
// gradient, this time from the L2 (a row for each SM takes 40 MB of it at 2^17
// logits of 16 bits). HBM sees one read, and one write, of the logits, which
// bounds it: 4,096 x 131,072 bf16 with gradient 430 us, 5.0 TB/s; the loss alone
// 205 us, 5.2 TB/s. Without the exponentials the former takes 426 us, without the
// stores 382 us. Clusters that held a row in registers between the passes paid a
// barrier of eight CTAs for every 256 KB: 570 to 830 us. About 11 us of a call
// are the first rows' way in and the last ones' out.
//
// nt threads take the words; a warp of its own starts the copies, and another one
// is a row ahead with the teacher: it reduces the entries to what the CTA needs
// of them, the list of tokens in its part with their probabilities and the
// student's logits, and of p and p (s - the greatest of these logits) the sums,
// which is all that the loss needs: log q_j = (s_j - peak) / T - log mass.
// Long rows are worked on by two CTAs of 256 threads on each SM, shorter ones by
// four of 128: their barriers hide behind one another.
enum { distill_words = 4,          // a thread's words in a landing buffer
  distill_nt_large = 256, distill_large_per_sm = 2, distill_nt_small = 128,
  distill_small_per_sm = 4 };

struct distill_list_t {
  int listed, taught;
  float weight, entropy;           // entropy: sum of p log p over all entries
  float share, product, from;
};

template<int nt>
struct distill_shared_t {
  enum { warps = nt / 32, most_stages = 8 };
  uint64_t full[most_stages], empty[most_stages];
  uint64_t list_full[2], list_empty[2];
  uint64_t told[2];
  distill_list_t list[2];
  peak_sum_t part[2][warps];
  float4 news[2][distill_max_cluster];         // peak, sum, share, product
  float news_from[2][distill_max_cluster];
};
// Behind the landing buffers, for each entry: two lists of {token, p, p of all
// entries with the token, student's logit} and the teacher's own scratch.
enum { distill_entry_bytes = 2 * 16 + 8 };

// Two neighbouring values as a pair of floats, and back with one rounding.
MGPU_DEVICE __forceinline__ uint64_t two_values(const float* v) {
  return ptx::make_pair(v[0], v[1]);
}
MGPU_DEVICE __forceinline__ uint64_t two_values(const __nv_bfloat16* v) {
  uint32_t bits;
  memcpy(&bits, v, 4);
  return ptx::make_pair(__uint_as_float(bits << 16),
    __uint_as_float(bits & 0xffff0000u));
}
MGPU_DEVICE __forceinline__ uint64_t two_values(const __half* v) {
  __half2 two;
  memcpy(&two, v, 4);
  float2 f = __half22float2(two);
  return ptx::make_pair(f.x, f.y);
}
MGPU_DEVICE __forceinline__ void store_two(float* v, float2 f) {
  v[0] = f.x;
  v[1] = f.y;
}
MGPU_DEVICE __forceinline__ void store_two(__nv_bfloat16* v, float2 f) {
  __nv_bfloat162 two = __floats2bfloat162_rn(f.x, f.y);
  memcpy(v, &two, 4);
}
MGPU_DEVICE __forceinline__ void store_two(__half* v, float2 f) {
  __half2 two = __floats2half2_rn(f.x, f.y);
  memcpy(v, &two, 4);
}

// The greatest of a thread's words (a NaN only where there is nothing else).
template<int held, int pack>
MGPU_DEVICE __forceinline__ float words_peak(
  const pack_t<float, pack> (&word)[held]) {
  float peak = -INFINITY;
  #pragma unroll
  for(int i = 0; i < held; ++i)
    #pragma unroll
    for(int j = 0; j < pack; ++j) peak = fmaxf(peak, word[i].v[j]);
  return peak;
}
template<typename pair_t, typename real_t, int held, int pack>
MGPU_DEVICE __forceinline__ float pairs_peak(
  const pack_t<real_t, pack> (&word)[held]) {
  pair_t peak;
  memcpy(&peak, &word[0].v[0], 4);
  #pragma unroll
  for(int i = 0; i < held; ++i)
    #pragma unroll
    for(int j = 0; j < pack; j += 2) {
      pair_t two;
      memcpy(&two, &word[i].v[j], 4);
      peak = __hmax2(peak, two);
    }
  return fmaxf(to_f32(peak.x), to_f32(peak.y));
}
template<int held, int pack>
MGPU_DEVICE __forceinline__ float words_peak(
  const pack_t<__half, pack> (&word)[held]) {
  return pairs_peak<__half2>(word);
}
template<int held, int pack>
MGPU_DEVICE __forceinline__ float words_peak(
  const pack_t<__nv_bfloat16, pack> (&word)[held]) {
  return pairs_peak<__nv_bfloat162>(word);
}

template<int nt, int pack, bool want_grad, typename real_t>
__global__ void __launch_bounds__(nt + 64, nt == distill_nt_large ?
  distill_large_per_sm : distill_small_per_sm)
distill_stream_k(const real_t* logits, int64_t stride, int count,
  int vocabulary, int log_ctas, int stages, distill_teacher_t teacher,
  float temperature, const float* weights, float* losses, real_t* grad,
  int64_t grad_stride, uint64_t timeout_ns) {
  typedef pack_t<real_t, pack> word_t;
  typedef distill_shared_t<nt> shared_t;
  enum { warps = nt / 32, held = distill_words, chunk = nt * held };
  extern __shared__ __align__(128) char memory[];
  __shared__ shared_t shared;

  const int entries = teacher.entries, ctas = 1 << log_ctas;
  word_t* buffers = (word_t*)memory;
  float4* lists = (float4*)(memory + (size_t)stages * chunk * 16);
  int tid = (int)threadIdx.x, lane = tid % 32, warp = tid / 32;
  int rank = (int)blockIdx.x & (ctas - 1);
  int clusters = (int)gridDim.x >> log_ctas;
  const float c = 1.4426950408889634f / temperature;
  const float per_t = 1.0f / temperature;

  if(!tid) {
    for(int i = 0; i < stages; ++i) {
      ptx::mbar_init(&shared.full[i], 1);
      ptx::mbar_init(&shared.empty[i], warps);
    }
    for(int i = 0; i < 2; ++i) {
      ptx::mbar_init(&shared.list_full[i], 1);
      ptx::mbar_init(&shared.list_empty[i], warps);
      ptx::mbar_init(&shared.told[i], 1);
    }
    ptx::fence_mbar_init_cluster();
    ptx::fence_proxy_async();
  }
  if(ctas > 1) cooperative_groups::this_cluster().sync();
  else __syncthreads();

  // A row's whole words between its 16-byte borders, and this CTA's part: words
  // [begin, end). The elements outside are the first CTA's.
  int head, words, begin, end;
  auto cut = [&](const real_t* x) {
    head = min((int)((16 - (uintptr_t)x % 16) % 16 / sizeof(real_t)) % pack,
      vocabulary);
    words = (vocabulary - head) / pack;
    int per_cta = (words + ctas - 1) >> log_ctas;
    begin = min(rank * per_cta, words);
    end = min(begin + per_cta, words);
  };
  int64_t row = (int64_t)blockIdx.x >> log_ctas;
  int stage = 0;
  uint32_t parity = 0;
  auto next_stage = [&]() {
    if(++stage == stages) {
      stage = 0;
      parity ^= 1;
    }
  };

  if(warp == warps) {
    // The copies.
    if(lane) return;
    for(; row < count; row += clusters) {
      const real_t* x = logits + row * stride;
      cut(x);
      const word_t* from = (const word_t*)(x + head);
      #pragma unroll 1
      for(int pass = 0; pass < (want_grad ? 2 : 1); ++pass)
        for(int w = begin; w < end; w += chunk) {
          // The first round finds the buffers empty.
          if(!ptx::mbar_wait(&shared.empty[stage], parity ^ 1, timeout_ns))
            return;
          uint32_t bytes = (uint32_t)min((int)chunk, end - w) * 16;
          ptx::mbar_arrive_expect_tx(&shared.full[stage], bytes);
          ptx::bulk_load(buffers + stage * chunk, from + w, bytes,
            &shared.full[stage]);
          next_stage();
        }
    }
    return;
  }
  if(warp == warps + 1) {
    // The teacher.
    float* logit = (float*)(lists + 2 * entries);
    int* token = (int*)(logit + entries);
    // Entries on their way: the first ones of the next row already while this
    // one's are reduced.
    enum { batch = 4 };
    int64_t next_token[batch];
    float next_logit[batch], next_weight = 1.0f;
    auto request = [&](int64_t r, int first) {
      #pragma unroll
      for(int b = 0; b < batch; ++b) {
        int64_t k = first + b * 32 + lane;
        next_token[b] = k < entries ? teacher.token(r * entries + k) : -1;
        next_logit[b] = k < entries ? teacher.logit(r * entries + k) : 0.0f;
      }
      if(weights && !first) next_weight = weights[r];
    };
    if(row < count) request(row, 0);
    for(int turn = 0; row < count; ++turn, row += clusters) {
      int set = turn & 1;
      const real_t* x = logits + row * stride;
      cut(x);
      if(!ptx::mbar_wait(&shared.list_empty[set], (uint32_t)(turn >> 1 & 1) ^ 1,
        timeout_ns)) return;
      float weight = next_weight;
      float peak = -INFINITY, sum = 0;
      for(int first = 0; first < entries; first += batch * 32) {
        if(first) request(row, first);
        #pragma unroll
        for(int b = 0; b < batch; ++b) {
          int k = first + b * 32 + lane;
          bool used = next_token[b] >= 0 && next_token[b] < vocabulary &&
            weight != 0;
          if(k < entries) {
            token[k] = used ? (int)next_token[b] : -1;
            logit[k] = used ? next_logit[b] : -INFINITY;
          }
          if(used) peak = fmaxf(peak, next_logit[b]);
        }
      }
      if(row + clusters < count) request(row + clusters, 0);
      #pragma unroll
      for(int offset = 16; offset; offset /= 2)
        peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, offset));
      // A NaN stays one.
      for(int k = lane; k < entries; k += 32)
        if(logit[k] != -INFINITY) sum += expf((logit[k] - peak) * per_t);
      #pragma unroll
      for(int offset = 16; offset; offset /= 2)
        sum += __shfl_xor_sync(0xffffffffu, sum, offset);
      bool taught = peak > -INFINITY || isnan(sum);
      float log_sum = logf(sum), entropy = 0, from = -INFINITY;
      float4* list = lists + set * entries;
      int listed = 0;
      for(int first = 0; first < entries; first += 32) {
        int k = first + lane;
        float prob = 0;
        int j = -1;
        if(k < entries && taught && logit[k] != -INFINITY) {
          float log_p = (logit[k] - peak) * per_t - log_sum;
          prob = expf(log_p);
          if(prob != 0) {
            entropy += prob * log_p;
            j = token[k];
          }
        }
        int w = j < head ? -1 : (j - head) / pack;
        bool own = j >= 0 && (w < 0 || w >= words ? !rank :
          w >= begin && w < end);
        unsigned votes = __ballot_sync(0xffffffffu, own);
        if(own) list[listed + __popc(votes & ((1u << lane) - 1))] =
          make_float4(__int_as_float(j), prob, prob, 0.0f);
        listed += __popc(votes);
      }
      __syncwarp();
      // The student's logits: read before anybody waits for the list, which comes
      // before the gradient is written, perhaps in their place.
      #pragma unroll 4
      for(int i = lane; i < listed; i += 32) {
        float value = to_f32(x[__float_as_int(list[i].x)]);
        list[i].w = value;
        from = fmaxf(from, value);
      }
      #pragma unroll
      for(int offset = 16; offset; offset /= 2)
        from = fmaxf(from, __shfl_xor_sync(0xffffffffu, from, offset));
      if(from == -INFINITY) from = 0;
      float share = 0, product = 0;
      for(int i = lane; i < listed; i += 32) {
        float4 mine = list[i];
        share += mine.y;
        product += mine.y * (mine.w - from);
        if(want_grad) {
          // All of a token's entries together.
          float taken = 0;
          #pragma unroll 4
          for(int q = 0; q < listed; ++q) {
            float4 other = list[q];
            if(__float_as_int(other.x) == __float_as_int(mine.x))
              taken += other.y;
          }
          list[i].z = taken;
        }
      }
      #pragma unroll
      for(int offset = 16; offset; offset /= 2) {
        entropy += __shfl_xor_sync(0xffffffffu, entropy, offset);
        share += __shfl_xor_sync(0xffffffffu, share, offset);
        product += __shfl_xor_sync(0xffffffffu, product, offset);
      }
      if(!lane) shared.list[set] = distill_list_t { listed, (int)taught, weight,
        entropy, share, product, from };
      __syncwarp();
      if(!lane) ptx::mbar_arrive(&shared.list_full[set]);
    }
    return;
  }

  bool good = true;
  auto take = [&](word_t (&word)[held], int here) {
    good = good && ptx::mbar_wait(&shared.full[stage], parity, timeout_ns);
    const word_t* buffer = buffers + stage * chunk;
    #pragma unroll
    for(int i = 0; i < held; ++i) {
      int w = i * nt + tid;
      if(w < here) word[i] = buffer[w];
      else {
        #pragma unroll
        for(int j = 0; j < pack; ++j)
          word[i].v[j] = from_f32<real_t>(-INFINITY);
      }
    }
    // The next copy writes through another proxy than these loads read: without
    // the fence it overtakes some of them.
    ptx::fence_proxy_async();
    __syncwarp();
    if(!lane) ptx::mbar_arrive(&shared.empty[stage]);
    next_stage();
  };
  const uint64_t c_pair = ptx::make_pair(c, c);
  for(int turn = 0; row < count; ++turn, row += clusters) {
    int set = turn & 1;
    const real_t* x = logits + row * stride;
    cut(x);
    int tail = vocabulary - head - words * pack;
    int edge = rank ? -1 : tid < head ? tid :
      tid < head + tail ? vocabulary - tail + (tid - head) : -1;
    float edge_value = edge >= 0 ? to_f32(x[edge]) : -INFINITY;

    // The first pass: weights relative to the thread's peak so far.
    float peak = -INFINITY;
    uint64_t sums = 0;
    #pragma unroll 1
    for(int w = begin; w < end; w += chunk) {
      word_t word[held];
      take(word, end - w);
      float higher = fmaxf(peak, words_peak(word));
      float base = higher == -INFINITY ? 0.0f : higher;
      if(higher > peak) {
        float scale = exp2_fast((peak - base) * c);
        sums = ptx::mul_pair(sums, ptx::make_pair(scale, scale));
        peak = higher;
      }
      const uint64_t minus_base = ptx::make_pair(-base, -base);
      #pragma unroll
      for(int i = 0; i < held; ++i) {
        if(w + i * nt >= end) break;         // the same for the whole CTA
        #pragma unroll
        for(int j = 0; j < pack; j += 2) {
          float2 power = ptx::pair_values(ptx::mul_pair(ptx::add_pair(
            two_values(&word[i].v[j]), minus_base), c_pair));
          sums = ptx::add_pair(sums, ptx::make_pair(exp2_fast(power.x),
            exp2_fast(power.y)));
        }
      }
    }
    peak_sum_t s { peak, ptx::pair_values(sums).x + ptx::pair_values(sums).y };
    s = merge(s, peak_sum_t { edge_value, edge_value == -INFINITY ? 0.0f :
      isnan(edge_value) || edge_value == INFINITY ? NAN : 1.0f }, c);
    s = warp_merge(s, c);
    if(!lane) shared.part[set][warp] = s;
    ptx::named_sync<1, nt>();
    s = warp_merge(lane < warps ? shared.part[set][lane] :
      peak_sum_t { -INFINITY, 0.0f }, c);

    good = good && ptx::mbar_wait(&shared.list_full[set],
      (uint32_t)(turn >> 1 & 1), timeout_ns);
    distill_list_t list = shared.list[set];
    float share = list.share, distance = list.product;
    if(ctas > 1) {
      // Two sets of slots and barriers: a CTA sends the news of the turn after
      // the next only when it has this CTA's of the next, which are sent behind
      // the wait for those of this turn.
      if(!warp) {
        if(!lane) ptx::mbar_arrive_expect_tx(&shared.told[set],
          (uint32_t)ctas * 20);
        if(lane < ctas) {
          uint32_t bar = ptx::cluster_addr(&shared.told[set], lane);
          ptx::store_async(ptx::cluster_addr(&shared.news[set][rank], lane),
            s.peak, s.sum, list.share, list.product, bar);
          ptx::store_async(ptx::cluster_addr(&shared.news_from[set][rank], lane),
            list.from, bar);
        }
      }
      good = good && ptx::mbar_wait(&shared.told[set],
        (uint32_t)(turn >> 1 & 1), timeout_ns);
      float4 n = lane < ctas ? shared.news[set][lane] :
        make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
      s = warp_merge(peak_sum_t { n.x, n.y }, c);
    }
    float base = s.peak == -INFINITY ? 0.0f : s.peak, mass = s.sum;
    if(!good) {                              // a wait ran out: no result
      mass = NAN;
      list.taught = 1;
      list.listed = 0;
      if(!lane) raise_status(nullptr, (uint32_t)status_copy_timeout);
    }
    bool none = !list.taught || (s.peak == -INFINITY && !isnan(mass));
    if(!rank && !tid) {
      float to_peak = 0;
      if(1 == ctas) {
        if(share != 0) to_peak = distance + share * (list.from - base);
      } else {
        share = 0;
        for(int r = 0; r < ctas; ++r) {
          float4 n = shared.news[set][r];
          share += n.z;
          if(n.z != 0) to_peak += n.w + n.z * (shared.news_from[set][r] - base);
        }
      }
      float loss = list.entropy + share * logf(mass) - to_peak * per_t;
      losses[row] = none ? 0.0f : temperature * temperature * loss;
    }

    if(want_grad) {
      float factor = none ? 0.0f : list.weight * temperature / mass;
      real_t* g = grad + row * grad_stride;
      word_t* g_words = (word_t*)(g + head);
      const uint64_t minus_base = ptx::make_pair(-base, -base);
      const uint64_t factor_pair = ptx::make_pair(factor, factor);
      #pragma unroll 1
      for(int w = begin; w < end; w += chunk) {
        word_t word[held];
        take(word, end - w);
        #pragma unroll
        for(int i = 0; i < held; ++i) {
          if(w + i * nt >= end) break;
          #pragma unroll
          for(int j = 0; j < pack; j += 2) {
            float2 power = ptx::pair_values(ptx::mul_pair(ptx::add_pair(
              two_values(&word[i].v[j]), minus_base), c_pair));
            store_two(&word[i].v[j], ptx::pair_values(ptx::mul_pair(
              ptx::make_pair(exp2_fast(power.x), exp2_fast(power.y)),
              factor_pair)));
          }
          // A row without a gradient: 0, even where a logit is not a number.
          if(none) word[i] = word_t();
          int at = w + i * nt + tid;
          if(at < end) store_streaming(g_words + at, word[i]);
        }
      }
      if(edge >= 0) g[edge] = from_f32<real_t>(none ? 0.0f :
        factor * exp2_fast((edge_value - base) * c));
      // Then the teacher's tokens in this CTA's part again.
      ptx::named_sync<1, nt>();
      const float4* entry = lists + set * entries;
      for(int i = tid; i < list.listed && !none; i += nt)
        g[__float_as_int(entry[i].x)] = from_f32<real_t>(factor *
          exp2_fast((entry[i].w - base) * c) -
          list.weight * temperature * entry[i].z);
    }
    __syncwarp();
    if(!lane) ptx::mbar_arrive(&shared.list_empty[set]);
  }
}

// How many clusters of `ctas` CTAs the device holds at a time; asked once for
// each kernel, device, size of the cluster and number of stages.
template<typename... tag_t, typename kernel_t>
int resident_clusters(kernel_t kernel, cudaLaunchConfig_t config, int ctas,
  int stages) {
  static std::atomic<int> known[64][4][8];
  int device = 0;
  throw_on_error(cudaGetDevice(&device));
  int log = ctas < 2 ? 0 : ctas < 4 ? 1 : ctas < 8 ? 2 : 3;
  std::atomic<int>* at = device < 64 ? &known[device][log][stages & 7] : nullptr;
  int clusters = at ? at->load(std::memory_order_relaxed) : 0;
  if(!clusters) {
    config.gridDim = dim3((unsigned)ctas);
    throw_on_error(cudaOccupancyMaxActiveClusters(&clusters, kernel, &config));
    if(clusters < 1) clusters = 1;
    if(at) at->store(clusters, std::memory_order_relaxed);
  }
  return clusters;
}

template<bool want_grad, typename real_t, typename teacher_t, typename token_t>
void distill_enqueue(const real_t* logits, int64_t stride, int count,
  int vocabulary, const token_t* tokens, const teacher_t* teacher, int entries,
  float temperature, const float* weights, float* losses, real_t* grad,
  int64_t grad_stride, cudaStream_t stream,
  uint64_t timeout_ns = 2000000000ull) {
  if(!count) return;
  enum { size = sizeof(real_t) };
  // Words of 16 bytes where rows of the logits and of the gradient begin at the
  // same place of one.
  bool apart = want_grad && ((uintptr_t)logits % 16 != (uintptr_t)grad % 16 ||
    (count > 1 && (stride - grad_stride) * size % 16));
  int64_t row_bytes = (int64_t)vocabulary * size;
  distill_teacher_t source { tokens, teacher, sizeof(token_t) == 8,
    teacher_kind(teacher), entries };
  cudaLaunchConfig_t config = { };
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  if constexpr (want_grad) {
    if(apart) {
      enum { nt = 512 };
      distill_apart_k<nt><<<(unsigned)count, nt, 12 * (size_t)entries,
        stream>>>(logits, stride, vocabulary, source, temperature, weights,
          losses, grad, grad_stride);
      throw_on_error(cudaGetLastError());
      return;
    }
  }
  auto launch = [&](auto threads) {
    enum { nt = decltype(threads)::value,
      per_sm = nt == distill_nt_large ? distill_large_per_sm :
        distill_small_per_sm,
      stage_bytes = nt * distill_words * 16 };
    auto kernel = distill_stream_k<nt, 16 / (int)size, want_grad, real_t>;
    // What an SM has, less the shared variables of fixed size.
    const int room = (224 << 10) / per_sm - 2048;
    int lists = distill_entry_bytes * entries;
    int stages = (room - lists) / stage_bytes;
    stages = stages < 3 ? 3 : stages > 6 ? 6 : stages;
    set_dynamic_smem<decltype(threads), std::integral_constant<bool, want_grad>,
      real_t>(kernel, 224 << 10);
    config.blockDim = dim3(nt + 64);
    config.dynamicSmemBytes = (size_t)stages * stage_bytes + lists;
    // CTAs to a row: rounds of rows times what each takes, a round's barriers
    // being worth about 32 KB. The second pass finds the row in the L2 only
    // where the rows under way take no more than half of it.
    int ctas = 1, clusters = 1;
    int64_t least = 0;
    for(int n = 1; n <= distill_max_cluster; n *= 2) {
      if(n > 1 && row_bytes / n < stage_bytes) break;
      attribute.val.clusterDim.x = (unsigned)n;
      int most = resident_clusters<decltype(threads), std::integral_constant<
        bool, want_grad>, real_t>(kernel, config, n, stages);
      int64_t cost = div_up((int64_t)count, (int64_t)most) *
        (row_bytes / n + (32 << 10));
      bool crowded = want_grad && distill_max_cluster != n &&
        min(count, most) * row_bytes > (64 << 20);
      if(!crowded && (!least || cost < least)) {
        least = cost;
        ctas = n;
        clusters = most;
      }
    }
    int log_ctas = ctas < 2 ? 0 : ctas < 4 ? 1 : ctas < 8 ? 2 : 3;
    attribute.val.clusterDim.x = (unsigned)ctas;
    config.gridDim = dim3((unsigned)(min(count, clusters) * ctas));
    throw_on_error(cudaLaunchKernelEx(&config, kernel, logits, stride, count,
      vocabulary, log_ctas, stages, source, temperature, weights, losses, grad,
      grad_stride, timeout_ns));
  };
  // Measured with 2,048 rows of 64 KB (loss): 30.5 us in small CTAs, 36 us in
  // large ones; with gradient, 509 rows of 200 KB: 61 us small, 43 us large, and
  // 4,096 rows of 256 KB: 565 us small, 425 us large, 525 us with 75 MB of rows
  // under way. One CTA of 512 threads to an SM took 47 us and 432 us.
  if(row_bytes > (96 << 10))
    launch(std::integral_constant<int, distill_nt_large>());
  else
    launch(std::integral_constant<int, distill_nt_small>());
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
