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
#include "ptx.hxx"
#ifdef __CUDACC__
#include <cooperative_groups.h>
#endif

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

////////////////////////////////////////////////////////////////////////////////
// A cluster of CTAs works on one row. Each warp owns a run of neighbouring
// tokens, the same one in every pass, so that after the first pass the row comes
// from the L1 (or the L2, where it is too long for it).
//
//   pass 1  the greatest logit
//   pass 2  a histogram over the distance from it, in steps of T / 64: of counts
//           for top-k; of weights in fixed point, relative to the step's own
//           weight, for top-p. It says which steps may hold the border.
//   pass 3  the exact weight (64 bits) above these steps, and a list of their
//           tokens, which the first CTA sorts to find the border itself. With
//           few tokens above the border the list holds those too, and the first
//           CTA goes on alone, on the list.
//   pass 4  the weight that is left in each warp's run; the run that holds the
//           drawn number is searched by its warp.
// Where the steps hold more tokens than the list takes, their range of logits
// is halved with exact sums until it fits or is a single value, whose tokens
// are then taken by index.

enum { sample_bins = 2048, sample_steps = 64, sample_list = 1024,
  sample_max_cluster = 8 };

// What the CTAs of a cluster tell one another.
struct sample_news_t {
  double a, b, c;
  uint32_t p, q;
  int i, j;
};

template<int nt>
struct sample_shared_t {
  enum { warps = nt / 32 };
  uint32_t hist[sample_bins];
  unsigned long long list[sample_list];
  sample_news_t news[2][sample_max_cluster];
  double run_sums[sample_max_cluster * warps];
  double warp_sums[2][warps];
  double fold[warps];
  int list_count;
  int hit;
};

template<int nt, typename real_t>
struct sample_cta_t {
  enum { warps = nt / 32, pack = 16 / (int)sizeof(real_t),
    each_list = sample_list / nt };
  typedef pack_t<real_t, pack> word_t;
  typedef sample_shared_t<nt> shared_t;
  struct band_t { int lo, hi; double tokens, inside; };

  const real_t* x;
  int vocabulary;
  shared_t& shared;
  cooperative_groups::cluster_group cluster;
  int rank, ctas, tid, lane, warp, run;
  int64_t run_begin, run_end;     // in elements behind the row's 16-byte border
  int shift;                      // where on it the row begins
  int exchanges;

  float peak, inv_temperature;
  uint32_t peak_key;
  double scale;
  uint32_t least;      // what is kept: keys above this one,
  int last;            // and those equal to it up to this index

  MGPU_DEVICE sample_cta_t(const real_t* x_, int vocabulary_,
    shared_t& shared_) : x(x_), vocabulary(vocabulary_), shared(shared_),
    cluster(cooperative_groups::this_cluster()),
    rank((int)cluster.block_rank()), ctas((int)cluster.num_blocks()),
    tid((int)threadIdx.x), lane((int)threadIdx.x % 32),
    warp((int)threadIdx.x / 32), exchanges(0), least(0), last(vocabulary_) {
    run = rank * warps + warp;
    shift = (int)((uintptr_t)x % 16 / sizeof(real_t));
    int64_t end = (int64_t)vocabulary + shift, step = 32 * pack;
    int64_t length = div_up(div_up(end, (int64_t)ctas * warps), step) * step;
    run_begin = min(length * run, end);
    run_end = min(run_begin + length, end);
  }

  // f(logit, index) for the tokens of this warp's run.
  template<typename func_t>
  MGPU_DEVICE __forceinline__ void each(func_t f) const {
    enum { ahead = pack == 4 ? 4 : 2, step = 32 * pack };
    int64_t a = run_begin + lane * pack;
    // Whole words, some of them in flight at a time, then the ragged ends.
    if(a < shift) {
      some(a, f);
      a += step;
    }
    for(; a + ((ahead - 1) * step + pack) <= run_end; a += ahead * step) {
      const real_t* from = x + (a - shift);
      word_t words[ahead];
      #pragma unroll
      for(int i = 0; i < ahead; ++i)
        words[i] = *(const word_t*)(from + i * step);
      #pragma unroll
      for(int i = 0; i < ahead; ++i)
        #pragma unroll
        for(int j = 0; j < pack; ++j)
          f(to_f32(words[i].v[j]), (int)(a - shift) + i * step + j);
    }
    for(; a < run_end; a += step) {
      if(a + pack <= run_end) {
        word_t word = *(const word_t*)(x + (a - shift));
        #pragma unroll
        for(int j = 0; j < pack; ++j)
          f(to_f32(word.v[j]), (int)(a - shift) + j);
      } else
        some(a, f);
    }
  }
  template<typename func_t>
  MGPU_DEVICE __forceinline__ void some(int64_t a, func_t f) const {
    int64_t begin = max(a, (int64_t)shift), end = min(a + pack, run_end);
    for(int64_t i = begin; i < end; ++i)
      f(to_f32(x[i - shift]), (int)(i - shift));
  }

  template<typename type_t, typename op_t>
  MGPU_DEVICE type_t fold(type_t v, op_t op) {
    type_t* parts = (type_t*)shared.fold;
    #pragma unroll
    for(int offset = 16; offset; offset /= 2)
      v = op(v, __shfl_xor_sync(0xffffffffu, v, offset));
    if(!lane) parts[warp] = v;
    __syncthreads();
    v = parts[0];
    #pragma unroll
    for(int w = 1; w < warps; ++w) v = op(v, parts[w]);
    __syncthreads();
    return v;
  }
  MGPU_DEVICE double fold_sum(double v) {
    return fold(v, [](double a, double b) { return a + b; });
  }
  MGPU_DEVICE double fold_most(double v) {
    return fold(v, [](double a, double b) { return a < b ? b : a; });
  }
  MGPU_DEVICE int fold_min(int v) {
    return fold(v, [](int a, int b) { return a < b ? a : b; });
  }
  MGPU_DEVICE int fold_max(int v) {
    return fold(v, [](int a, int b) { return a < b ? b : a; });
  }
  MGPU_DEVICE uint32_t fold_max(uint32_t v) {
    return fold(v, [](uint32_t a, uint32_t b) { return a < b ? b : a; });
  }

  // Inclusive sums over the CTA's threads.
  MGPU_DEVICE double2 scan(double a, double b) {
    double2 sum = make_double2(a, b);
    #pragma unroll
    for(int offset = 1; offset < 32; offset *= 2) {
      double y = __shfl_up_sync(0xffffffffu, sum.x, offset);
      double z = __shfl_up_sync(0xffffffffu, sum.y, offset);
      if(lane >= offset) { sum.x += y; sum.y += z; }
    }
    if(31 == lane) {
      shared.warp_sums[0][warp] = sum.x;
      shared.warp_sums[1][warp] = sum.y;
    }
    __syncthreads();
    for(int w = 0; w < warp; ++w) {
      sum.x += shared.warp_sums[0][w];
      sum.y += shared.warp_sums[1][w];
    }
    __syncthreads();
    return sum;
  }

  // Every CTA's news (the same in all of its threads) to every CTA. Two sets
  // of slots: one is written again only behind a barrier that its readers have
  // passed.
  MGPU_DEVICE const sample_news_t* share(const sample_news_t& mine) {
    int set = exchanges++ & 1;
    if(tid < ctas)
      cluster.map_shared_rank(&shared, tid)->news[set][rank] = mine;
    cluster.sync();
    return shared.news[set];
  }

  MGPU_DEVICE bool kept(uint32_t key, int v) const {
    return key > least || (key == least && v <= last);
  }
  MGPU_DEVICE double weight(float value) const {
    return value == peak ? 1.0 : exp(((double)value - (double)peak) * scale);
  }
  template<bool by_count>
  MGPU_DEVICE double size(float value) const {
    return by_count ? 1.0 : weight(value);
  }
  // Neither rises where the logit does.
  MGPU_DEVICE float distance(float value) const {
    return value == peak ? 0.0f : (peak - value) * inv_temperature;
  }
  MGPU_DEVICE int bin(float distance) const {
    return (int)fminf(distance * (float)sample_steps, sample_bins - 1.0f);
  }

  MGPU_DEVICE uint32_t find_peak() {
    uint32_t key = 0;
    each([&](float value, int) {
      key = max(key, isnan(value) ? 0xffffffffu : order_key(value));
    });
    sample_news_t mine = { };
    mine.p = fold_max(key);
    ptx::cluster_wait();                     // every CTA has started
    const sample_news_t* news = share(mine);
    key = 0;
    for(int r = 0; r < ctas; ++r) key = max(key, news[r].p);
    return key;
  }

  MGPU_DEVICE int first_of(uint32_t wanted) {
    int at = vocabulary;
    each([&](float value, int v) {
      if(order_key(value) == wanted && v < at) at = v;
    });
    sample_news_t mine = { };
    mine.i = fold_min(at);
    const sample_news_t* news = share(mine);
    at = vocabulary;
    for(int r = 0; r < ctas; ++r) at = min(at, news[r].i);
    return at;
  }

  //////////////////////////////////////////////////////////////////////////////
  // Sums of the runs, in the order of the vocabulary.

  // Each warp's number (the same in its lanes) to every CTA.
  MGPU_DEVICE void share_run_sum(double mine) {
    if(lane < ctas)
      cluster.map_shared_rank(&shared, lane)->run_sums[run] = mine;
    cluster.sync();
  }
  // The first run with a sum for which test(sum up to its end), and the sum
  // before it; where there is none, the last run with a sum; -1 where all are
  // 0. The same in every thread of the cluster.
  template<typename test_t>
  MGPU_DEVICE int find_run(test_t test, double& before) {
    enum { each_lane = sample_max_cluster * warps / 32 };
    double own[each_lane], sum = 0;
    #pragma unroll
    for(int i = 0; i < each_lane; ++i) {
      int r = lane * each_lane + i;
      own[i] = r < ctas * warps ? shared.run_sums[r] : 0.0;
      sum += own[i];
    }
    double ahead = sum;
    #pragma unroll
    for(int offset = 1; offset < 32; offset *= 2) {
      double y = __shfl_up_sync(0xffffffffu, ahead, offset);
      if(lane >= offset) ahead += y;
    }
    ahead = __shfl_up_sync(0xffffffffu, ahead, 1);
    if(!lane) ahead = 0;
    int found = -1, any = -1;
    double found_before = 0, any_before = 0;
    #pragma unroll
    for(int i = 0; i < each_lane; ++i) {
      if(own[i] > 0) {
        any = lane * each_lane + i;
        any_before = ahead;
        if(found < 0 && test(ahead + own[i])) {
          found = any;
          found_before = ahead;
        }
      }
      ahead += own[i];
    }
    unsigned hits = __ballot_sync(0xffffffffu, found >= 0);
    unsigned some = __ballot_sync(0xffffffffu, any >= 0);
    if(hits) {
      int from = __ffs(hits) - 1;
      before = __shfl_sync(0xffffffffu, found_before, from);
      return __shfl_sync(0xffffffffu, found, from);
    }
    if(!some) return -1;
    int from = 31 - __clz(some);
    before = __shfl_sync(0xffffffffu, any_before, from);
    return __shfl_sync(0xffffffffu, any, from);
  }
  // All runs together, in every thread.
  MGPU_DEVICE double total_of_runs() const {
    enum { each_lane = sample_max_cluster * warps / 32 };
    double sum = 0;
    #pragma unroll
    for(int i = 0; i < each_lane; ++i) {
      int r = lane * each_lane + i;
      sum += r < ctas * warps ? shared.run_sums[r] : 0.0;
    }
    #pragma unroll
    for(int offset = 16; offset; offset /= 2)
      sum += __shfl_xor_sync(0xffffffffu, sum, offset);
    return sum;
  }
  // The CTA whose run `found` is searches it: size(value, index) of the tokens
  // is added up in order, from `before`, and the first token with a size whose
  // sum passes test is the result, else the last one with a size. Each warp adds
  // up a part of the run; the part with the token is gone through 32 by 32.
  template<typename size_t_, typename test_t>
  MGPU_DEVICE int search_run(int found, double before, size_t_ size,
    test_t test) {
    int64_t length = div_up(div_up((int64_t)vocabulary + shift,
      (int64_t)ctas * warps), (int64_t)(32 * pack)) * (32 * pack);
    int64_t begin = length * found;
    int64_t end = min(begin + length, (int64_t)vocabulary + shift);
    int64_t part = div_up(div_up(length, (int64_t)warps), (int64_t)32) * 32;
    int64_t part_begin = min(begin + part * warp, end);
    int64_t part_end = min(part_begin + part, end);
    double sum = 0;
    for(int64_t a = part_begin + lane; a < part_end; a += 32)
      if(a >= shift) sum += size(to_f32(x[a - shift]), (int)(a - shift));
    #pragma unroll
    for(int offset = 16; offset; offset /= 2)
      sum += __shfl_xor_sync(0xffffffffu, sum, offset);
    if(!lane) shared.warp_sums[0][warp] = sum;
    if(!tid) shared.hit = -1;
    __syncthreads();
    int chosen = -1;
    double chosen_before = 0;
    for(int w = 0; w < warps; ++w) {
      double own = shared.warp_sums[0][w];
      if(own > 0) {
        chosen = w;
        chosen_before = before;
        if(test(before + own)) break;
      }
      before += own;
    }
    if(chosen == warp) {
      before = chosen_before;
      int at = -1;
      bool done = false;
      for(int64_t first = part_begin; first < part_end && !done; first += 32) {
        int64_t a = first + lane;
        double own = a >= shift && a < part_end ?
          size(to_f32(x[a - shift]), (int)(a - shift)) : 0.0;
        double upto = own;
        #pragma unroll
        for(int offset = 1; offset < 32; offset *= 2) {
          double y = __shfl_up_sync(0xffffffffu, upto, offset);
          if(lane >= offset) upto += y;
        }
        unsigned some = __ballot_sync(0xffffffffu, own > 0);
        unsigned hits = __ballot_sync(0xffffffffu,
          own > 0 && test(before + upto));
        if(hits) {
          at = (int)(first - shift) + __ffs(hits) - 1;
          done = true;
        } else if(some)
          at = (int)(first - shift) + 31 - __clz(some);
        before += __shfl_sync(0xffffffffu, upto, 31);
      }
      if(!lane) shared.hit = at;
    }
    __syncthreads();
    return shared.hit;
  }

  // The index of the nth (from 1) kept token with this key.
  MGPU_DEVICE int nth_equal(uint32_t wanted, double nth) {
    auto one = [&](float value, int v) {
      return order_key(value) == wanted && kept(wanted, v) ? 1.0 : 0.0;
    };
    int mine = 0;
    each([&](float value, int v) { mine += one(value, v) > 0; });
    share_run_sum((double)__reduce_add_sync(0xffffffffu, mine));
    auto test = [&](double sum) { return sum >= nth; };
    double before = 0;
    int found = find_run(test, before);
    sample_news_t told = { };
    told.i = -1;
    if(found >= 0 && found / warps == rank)
      told.i = search_run(found, before, one, test);
    const sample_news_t* news = share(told);
    int at = -1;
    for(int r = 0; r < ctas; ++r) at = max(at, news[r].i);
    return at;
  }

  //////////////////////////////////////////////////////////////////////////////
  // Pass 2: the steps [lo, hi] that may hold the border, about how many tokens
  // are in them (`inside`), and the most that can be in [0, hi] (`tokens`).
  // The border is where the running count reaches `target`, or the running
  // weight `target` times the weight of all.

  template<bool by_count>
  MGPU_DEVICE band_t find_band(double target) {
    // Fixed-point weights: a step's sum stays below 2^32 whatever it holds.
    float unit = by_count ? 1.0f : fminf(4096.0f, 2147483648.0f / vocabulary);
    for(int b = tid; b < sample_bins; b += nt) shared.hist[b] = 0;
    __syncthreads();
    each([&](float value, int v) {
      if(!kept(order_key(value), v)) return;
      float d = distance(value);
      int b = bin(d);
      uint32_t add = 1;
      if(!by_count) {
        // exp(-f) for 0 <= f <= 1 / 64, to 1e-6.
        float f = fminf(fmaxf(d - b * (1.0f / sample_steps), 0.0f),
          1.0f / sample_steps);
        add = (uint32_t)__float2int_rn(unit * (1.0f - f + 0.5f * f * f));
      }
      atomicAdd(&shared.hist[b], add);
    });
    cluster.sync();

    // Each CTA adds up a slice of the steps, a few of them to a thread.
    enum { most = sample_bins / nt };
    int slice = sample_bins / ctas, each_thread = div_up(slice, (int)nt);
    int first = rank * slice + tid * each_thread;
    int mine_count = tid * each_thread < slice ? each_thread : 0;
    double weights[most], tokens[most], weight_sum = 0, token_sum = 0;
    // A token adds at least this much.
    double fewest = by_count ? 1.0 : (double)unit * 0.984 - 0.5;
    #pragma unroll
    for(int i = 0; i < most; ++i) {
      weights[i] = tokens[i] = 0;
      if(i < mine_count) {
        double sum = 0;
        for(int r = 0; r < ctas; ++r)
          sum += cluster.map_shared_rank(&shared, r)->hist[first + i];
        weights[i] = by_count ? sum :
          sum * exp(-(double)(first + i) / sample_steps);
        tokens[i] = fewest > 0 ? sum / fewest : sum * 1e30;
      }
      weight_sum += weights[i];
      token_sum += tokens[i];
    }
    double2 sums = scan(weight_sum, token_sum);
    sample_news_t mine = { };
    mine.a = fold_most(sums.x);
    mine.b = fold_most(sums.y);
    const sample_news_t* news = share(mine);
    double total = 0, all_tokens = 0, at = 0, at_tokens = 0;
    for(int r = 0; r < ctas; ++r) {
      if(r == rank) {
        at = total + sums.x - weight_sum;
        at_tokens = all_tokens + sums.y - token_sum;
      }
      total += news[r].a;
      all_tokens += news[r].b;
    }
    // Sum and total are each off by at most 0.51 / unit + 1e-5 of the total.
    double slack = by_count ? 0.0 : (2.0 / unit + 5e-5) * total;
    double goal = by_count ? target : target * total;
    int lo = sample_bins, hi = sample_bins;
    double lo_tokens = 0, hi_tokens = 0;
    #pragma unroll
    for(int i = 0; i < most; ++i) {
      if(i < mine_count) {
        at += weights[i];
        if(lo == sample_bins && at >= goal - slack) {
          lo = first + i;
          lo_tokens = at_tokens;
        }
        at_tokens += tokens[i];
        if(hi == sample_bins && at >= goal + slack) {
          hi = first + i;
          hi_tokens = at_tokens;
        }
      }
    }
    mine.i = fold_min(lo);
    mine.j = fold_min(hi);
    mine.a = fold_most(lo == mine.i ? lo_tokens : 0.0);
    mine.b = fold_most(hi == mine.j ? hi_tokens : 0.0);
    news = share(mine);
    band_t band { sample_bins, sample_bins, all_tokens, 0 };
    double before = 0;
    for(int r = ctas - 1; r >= 0; --r) {
      if(news[r].i < sample_bins) { band.lo = news[r].i; before = news[r].a; }
      if(news[r].j < sample_bins) {
        band.hi = news[r].j;
        band.tokens = news[r].b;
      }
    }
    band.hi = min(band.hi, sample_bins - 1);
    if(band.lo > band.hi) {
      band.lo = 0;
      before = 0;
    }
    band.inside = band.tokens - before;
    return band;
  }

  //////////////////////////////////////////////////////////////////////////////
  // The list, in the first CTA.

  MGPU_DEVICE void append(uint32_t key, int v) {
    shared_t* first = cluster.map_shared_rank(&shared, 0);
    int at = atomicAdd(&first->list_count, 1);
    if(at < sample_list)
      first->list[at] = (unsigned long long)key << 32 | (0xffffffffu - v);
  }
  MGPU_DEVICE uint32_t list_key(int i) const {
    return (uint32_t)(shared.list[i] >> 32);
  }
  MGPU_DEVICE int list_index(int i) const {
    return (int)(0xffffffffu - (uint32_t)shared.list[i]);
  }
  // The greatest first; equal keys by index.
  MGPU_DEVICE void sort_list(int count) {
    int n = 2;
    while(n < count) n *= 2;
    for(int i = count + tid; i < n; i += nt) shared.list[i] = 0;
    __syncthreads();
    for(int k = 2; k <= n; k *= 2)
      for(int j = k / 2; j; j /= 2) {
        for(int t = tid; t < n / 2; t += nt) {
          int i = (t & ~(j - 1)) * 2 + (t & (j - 1));
          unsigned long long a = shared.list[i], b = shared.list[i + j];
          if((a < b) == !(i & k)) {
            shared.list[i] = b;
            shared.list[i + j] = a;
          }
        }
        __syncthreads();
      }
  }
  // The first place, in the list's order, of an entry with a size for which
  // test(the sum up to it); else the last entry with a size. `sum`: of all.
  template<typename size_t_, typename test_t>
  MGPU_DEVICE int search_list(int count, size_t_ size, test_t test) {
    double own[each_list], sum = 0;
    #pragma unroll
    for(int i = 0; i < each_list; ++i) {
      int e = tid * each_list + i;
      own[i] = e < count ? size(e) : 0.0;
      sum += own[i];
    }
    double at = scan(sum, 0).x - sum;
    int found = sample_list, any = -1;
    #pragma unroll
    for(int i = 0; i < each_list; ++i) {
      at += own[i];
      if(own[i] > 0) {
        any = tid * each_list + i;
        if(found == sample_list && test(at)) found = any;
      }
    }
    found = fold_min(found);
    any = fold_max(any);
    return found < sample_list ? found : any;
  }
  template<typename size_t_>
  MGPU_DEVICE double sum_list(int count, size_t_ size) {
    double sum = 0;
    #pragma unroll
    for(int i = 0; i < each_list; ++i) {
      int e = tid * each_list + i;
      sum += e < count ? size(e) : 0.0;
    }
    return fold_sum(sum);
  }

  // The first CTA alone: the list holds every token that may be kept, `total`
  // is the weight that top-p refers to (below 0: the list's first `count`).
  MGPU_DEVICE int finish_list(int count, double total, float top_p, float min_p,
    double u) {
    auto by_place = [&](int e) { return weight(key_value(list_key(e))); };
    if(top_p < 1) {
      if(total < 0) total = sum_list(count, by_place);
      double target = (double)top_p * total;
      count = search_list(count, by_place,
        [&](double sum) { return sum >= target; }) + 1;
    }
    if(min_p > 0) {
      // Weights fall along the list.
      int fit = 0;
      for(int e = tid; e < count; e += nt)
        if(list_key(e) == peak_key || by_place(e) >= (double)min_p) fit = e + 1;
      count = fold_max(fit);
    }
    if(count < 2) return list_index(0);
    // By index, with the key in the low half.
    for(int e = tid; e < count; e += nt) {
      unsigned long long entry = shared.list[e];
      shared.list[e] = entry << 32 | entry >> 32;
    }
    sort_list(count);
    auto by_index = [&](int e) {
      return weight(key_value((uint32_t)shared.list[e]));
    };
    double target = u * sum_list(count, by_index);
    int e = search_list(count, by_index,
      [&](double sum) { return sum > target; });
    return (int)(0xffffffffu - (uint32_t)(shared.list[e] >> 32));
  }

  //////////////////////////////////////////////////////////////////////////////
  // Pass 3 and what follows from it: `least` and `last` for the tokens above
  // the border. True where the list holds all that is left; the weight of what
  // was kept before is in `total`, the list's length in `listed`.

  template<bool by_count>
  MGPU_DEVICE bool find_border(double target, double& total, int& listed) {
    band_t band = find_band<by_count>(target);
    bool whole = band.tokens <= sample_list;
    bool list = whole || band.inside <= 1.25 * sample_list;
    double above = 0, all = 0;
    uint32_t low = 0xffffffffu, high = 0;
    int inside = 0;
    each([&](float value, int v) {
      uint32_t key = order_key(value);
      if(!kept(key, v)) return;
      int b = bin(distance(value));
      if(by_count && b > band.hi) return;
      double w = size<by_count>(value);
      all += w;
      if(b > band.hi) return;
      if(b < band.lo) {
        above += w;
        if(whole) append(key, v);
      } else {
        ++inside;
        low = min(low, key);
        high = max(high, key);
        if(list) append(key, v);
      }
    });
    sample_news_t mine = { };
    mine.a = fold_sum(above);
    mine.b = fold_sum(all);
    mine.p = ~fold_max(~low);
    mine.q = fold_max(high);
    mine.i = (int)fold_sum((double)inside);
    const sample_news_t* news = share(mine);
    above = all = 0;
    low = 0xffffffffu;
    high = 0;
    inside = 0;
    for(int r = 0; r < ctas; ++r) {
      above += news[r].a;
      all += news[r].b;
      low = min(low, news[r].p);
      high = max(high, news[r].q);
      inside += news[r].i;
    }
    total = all;
    if(!by_count) target *= all;
    if(whole) {
      listed = min(shared.list_count, (int)sample_list);   // the first CTA's
      return true;
    }

    list = list && inside <= sample_list;
    while(inside > sample_list && low < high) {
      uint32_t middle = low + (high - low) / 2;
      double upper = 0;
      uint32_t upper_low = 0xffffffffu, lower_high = 0;
      int upper_count = 0;
      each([&](float value, int v) {
        uint32_t key = order_key(value);
        if(key < low || key > high || !kept(key, v)) return;
        if(key > middle) {
          upper += size<by_count>(value);
          ++upper_count;
          upper_low = min(upper_low, key);
        } else
          lower_high = max(lower_high, key);
      });
      mine = sample_news_t { };
      mine.a = fold_sum(upper);
      mine.p = ~fold_max(~upper_low);
      mine.q = fold_max(lower_high);
      mine.i = (int)fold_sum((double)upper_count);
      news = share(mine);
      upper = 0;
      upper_low = 0xffffffffu;
      lower_high = 0;
      upper_count = 0;
      for(int r = 0; r < ctas; ++r) {
        upper += news[r].a;
        upper_low = min(upper_low, news[r].p);
        lower_high = max(lower_high, news[r].q);
        upper_count += news[r].i;
      }
      if(above + upper >= target) {
        low = upper_low;
        inside = upper_count;
      } else {
        above += upper;
        high = lower_high;
        inside -= upper_count;
      }
    }
    if(inside > sample_list) {
      // One value: as many of its tokens as it takes.
      double need = ceil((target - above) / size<by_count>(key_value(low)));
      need = need > 1 ? (need < vocabulary ? need : vocabulary) : 1;
      if(!rank && !tid) shared.list_count = 0;   // behind the appends' barrier
      int at = nth_equal(low, need);
      least = low;
      last = at;
      return false;
    }
    if(!list) {
      if(!rank && !tid) shared.list_count = 0;
      cluster.sync();
      each([&](float value, int v) {
        uint32_t key = order_key(value);
        if(key >= low && key <= high && kept(key, v)) append(key, v);
      });
      cluster.sync();
    }
    mine = sample_news_t { };
    if(!rank) {
      sort_list(inside);
      int e = search_list(inside, [&](int e) {
          return size<by_count>(key_value(list_key(e)));
        }, [&](double sum) { return above + sum >= target; });
      e = max(e, 0);
      mine.p = list_key(e);
      mine.i = list_index(e);
      __syncthreads();
      if(!tid) shared.list_count = 0;
    }
    news = share(mine);
    least = news[0].p;
    last = news[0].i;
    return false;
  }

  // Pass 4.
  MGPU_DEVICE void draw(float min_p, double u, int* token) {
    auto left = [&](float value, int v) {
      uint32_t key = order_key(value);
      if(!kept(key, v)) return 0.0;
      double w = weight(value);
      return w >= (double)min_p || key == peak_key ? w : 0.0;
    };
    double sum = 0;
    each([&](float value, int v) { sum += left(value, v); });
    #pragma unroll
    for(int offset = 16; offset; offset /= 2)
      sum += __shfl_xor_sync(0xffffffffu, sum, offset);
    share_run_sum(sum);
    double target = u * total_of_runs(), before = 0;
    auto test = [&](double s) { return s > target; };
    int found = find_run(test, before);
    if(found >= 0 && found / warps == rank) {
      int at = search_run(found, before, left, test);
      if(!tid) *token = at;
    }
  }
};

template<int nt, typename real_t>
__global__ void __launch_bounds__(nt)
sample_k(const real_t* logits, int64_t stride, int vocabulary,
  const float* uniforms, sampling_t settings, int* tokens, int ctas) {
  __shared__ sample_shared_t<nt> shared;
  ptx::cluster_arrive_relaxed();
  int64_t at = (int64_t)blockIdx.x / ctas;
  float temperature = settings.temperatures ? settings.temperatures[at] :
    settings.temperature;
  if(temperature > FLT_MAX) temperature = FLT_MAX;
  float top_p = settings.top_ps ? settings.top_ps[at] : settings.top_p;
  float min_p = settings.min_ps ? settings.min_ps[at] : settings.min_p;
  int top_k = settings.top_ks ? settings.top_ks[at] : settings.top_k;
  double u = (double)uniforms[at];

  sample_cta_t<nt, real_t> cta(logits + at * stride, vocabulary, shared);
  bool leader = !cta.rank && !cta.tid;
  if(!cta.tid) shared.list_count = 0;
  cta.peak_key = cta.find_peak();
  cta.peak = key_value(cta.peak_key);
  // A NaN has the greatest key of all.
  if(0xffffffffu == cta.peak_key || !(cta.peak > -INFINITY)) {
    if(leader) tokens[at] = -1;
  } else if(!(temperature > 0)) {
    int first = cta.first_of(cta.peak_key);
    if(leader) tokens[at] = first;
  } else {
    cta.scale = 1.0 / (double)temperature;
    cta.inv_temperature = 1.0f / temperature;
    bool listed = false;
    double total = -1;
    int count = 0;
    if(top_k > 0 && top_k < vocabulary) {
      listed = cta.template find_border<true>((double)top_k, total, count);
      // The weight that top-p refers to is that of the first top_k.
      total = -1;
    }
    bool by_k = listed;
    if(!listed && top_p < 1)
      listed = cta.template find_border<false>((double)top_p, total, count);
    if(!listed)
      cta.draw(min_p, u, tokens + at);
    else if(!cta.rank) {
      cta.sort_list(count);
      int token = cta.finish_list(by_k ? min(count, top_k) : count, total,
        top_p, min_p, u);
      if(!cta.tid) tokens[at] = token;
    }
  }
  // No CTA leaves while another may still write to it: the last exchange of
  // every path above ends with a barrier behind the writes.
}

template<typename real_t>
void sample_enqueue(const real_t* logits, int64_t stride, int count,
  int vocabulary, const float* uniforms, const sampling_t& settings,
  int* tokens, cudaStream_t stream) {
  if(!count) return;
  enum { nt = 512 };
  int ctas = 1;
  while(ctas < sample_max_cluster && (int64_t)count * ctas < 296 &&
    vocabulary / ctas > 2 * nt) ctas *= 2;
  cudaLaunchConfig_t config = { };
  config.gridDim = dim3((unsigned)((int64_t)count * ctas));
  config.blockDim = dim3(nt);
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = (unsigned)ctas;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  throw_on_error(cudaLaunchKernelEx(&config, sample_k<nt, real_t>, logits,
    stride, vocabulary, uniforms, settings, tokens, ctas));
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
