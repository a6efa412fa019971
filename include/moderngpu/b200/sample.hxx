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
// Few tokens kept by top-k: every CTA finds the step of a histogram of its own
// part that holds its own top_k-th token and lists the tokens down to this step,
// which hold the row's greatest top_k. The first CTA sorts the lists of all and
// goes on alone.
//
// Otherwise:
//   pass 1  the greatest logit
//   pass 2  a histogram over the distance from it, in steps of T / 64: of counts
//           for top-k; of weights in fixed point, relative to the step's own
//           weight, for top-p. It says which steps may hold the border.
//   pass 3  the exact weight (64 bits) above these steps, and a list of their
//           tokens, which the first CTA sorts to find the border itself. With
//           few tokens above the border the list holds those too, and the first
//           CTA goes on alone, on the list.
//   pass 4  the weight that is left in each warp's run; the run that holds the
//           drawn number is searched by its CTA.
// Where the steps hold more tokens than the list takes, their range of logits
// is halved with exact sums until it fits or is a single value, whose tokens
// are then taken by index.
//
// What a warp finds it tells all CTAs at once, and every warp adds up what all
// warps told: one barrier of the cluster (1,300 cycles) to an exchange, and none
// of the CTA.
//
// Not bound by bytes: one row of 131,072 takes 16 us by the latency of some eight
// exchanges and of the list; 64 rows of them under top-p alone 80 us by the
// instructions of passes 2 and 3, of which a fourth are operations of 64 bits.

enum { sample_bins = 2048, sample_steps = 64, sample_list = 1024,
  sample_max_cluster = 8, sample_powers = 64, sample_groups = 64 };

// What a warp tells all CTAs of its cluster.
struct sample_news_t {
  double a, b;
  uint32_t p, q;
  int i, j;
};

template<int nt>
struct sample_shared_t {
  enum { warps = nt / 32, runs = sample_max_cluster * warps };
  uint32_t hist[sample_bins];
  unsigned long long list[sample_list];
  double list_weights[sample_list];
  sample_news_t news[2][runs];
  double powers[sample_powers];              // 2^(i / 64)
  // Of 32 threads' steps each: weight and tokens.
  double group_weights[sample_groups], group_tokens[sample_groups];
  double band_before, band_tokens;
  int band_lo, band_hi;
  double fold[2][warps];
  int list_count, hit;
};

template<int nt, bool staged, typename real_t>
struct sample_cta_t {
  enum { warps = nt / 32, pack = 16 / (int)sizeof(real_t), batch = 4,
    each_list = sample_list / nt, runs = sample_max_cluster * warps,
    each_lane = runs / 32 };
  typedef pack_t<real_t, pack> word_t;
  typedef sample_shared_t<nt> shared_t;
  struct band_t { int lo, hi; double tokens, inside; };

  const real_t* x;
  word_t* stage;       // the CTA's part, where it fits into shared memory
  int vocabulary;
  shared_t& shared;
  cooperative_groups::cluster_group cluster;
  int rank, ctas, tid, lane, warp, run;
  // In elements behind the row's 16-byte border.
  int64_t part_begin, run_begin, run_end;
  int shift;                      // where on it the row begins
  int exchanges;

  float peak, steps_per_logit;
  uint32_t peak_key;
  double log2_scale;   // log2(e) / T
  float weightless;    // logits below have no weight
  double run_left;     // see find_border
  uint32_t least;      // what is kept: keys above this one,
  int last;            // and those equal to it up to this index

  MGPU_DEVICE sample_cta_t(const real_t* x_, word_t* stage_, int vocabulary_,
    shared_t& shared_) : x(x_), stage(stage_), vocabulary(vocabulary_),
    shared(shared_),
    cluster(cooperative_groups::this_cluster()),
    rank((int)cluster.block_rank()), ctas((int)cluster.num_blocks()),
    tid((int)threadIdx.x), lane((int)threadIdx.x % 32),
    warp((int)threadIdx.x / 32), exchanges(0), least(0), last(vocabulary_) {
    run = rank * warps + warp;
    shift = (int)((uintptr_t)x % 16 / sizeof(real_t));
    int64_t end = (int64_t)vocabulary + shift, length = run_length();
    part_begin = length * rank * warps;
    run_begin = min(length * run, end);
    run_end = min(run_begin + length, end);
  }
  MGPU_DEVICE int64_t run_length() const {
    int64_t step = 32 * pack;
    return div_up(div_up((int64_t)vocabulary + shift, (int64_t)ctas * warps),
      step) * step;
  }

  // The word at element a of the row itself; -infinity outside of it, which has
  // no weight and is never drawn.
  MGPU_DEVICE __forceinline__ word_t load(int64_t a) const {
    word_t word;
    if(a >= shift && a + pack <= run_end)
      word = *(const word_t*)(x + (a - shift));
    else {
      #pragma unroll
      for(int j = 0; j < pack; ++j)
        word.v[j] = a + j >= shift && a + j < run_end ? x[a + j - shift] :
          from_f32<real_t>(-INFINITY);
    }
    return word;
  }
  MGPU_DEVICE __forceinline__ float logit_at(int64_t a) const {
    return to_f32(staged ? ((const real_t*)stage)[a - part_begin] :
      x[a - shift]);
  }

  // The first pass: the run's greatest logit as a key, a NaN's the greatest of
  // all; where there is room the run moves into shared memory, because a barrier
  // of the cluster empties the L1. Several words are in flight.
  MGPU_DEVICE uint32_t part_peak() const {
    enum { ahead = 4, step = 32 * pack };
    float peak = -INFINITY;
    for(int64_t a = run_begin + lane * pack; a < run_end; a += ahead * step) {
      word_t words[ahead];
      #pragma unroll
      for(int i = 0; i < ahead; ++i)
        if(a + i * step < run_end) words[i] = load(a + i * step);
      #pragma unroll
      for(int i = 0; i < ahead; ++i)
        if(a + i * step < run_end) {
          if(staged) stage[(a - part_begin) / pack + i * 32] = words[i];
          #pragma unroll
          for(int j = 0; j < pack; ++j)
            peak = max_or_nan(peak, to_f32(words[i].v[j]));
        }
    }
    uint32_t key = isnan(peak) ? 0xffffffffu : order_key(peak);
    __syncwarp();
    return __reduce_max_sync(0xffffffffu, run_begin < run_end ? key : 0u);
  }
  MGPU_DEVICE static float max_or_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
  }

  // f(logits, index of the first) for four neighbouring tokens of this warp's
  // run at a time. One copy of f's code for every part of a word: these passes
  // run once, and wait for instructions where they are long.
  template<typename func_t>
  MGPU_DEVICE __forceinline__ void each_four(func_t f) const {
    enum { step = 32 * pack };
    int64_t a = run_begin + lane * pack;
    if(a >= run_end) return;
    word_t next = staged ? stage[(a - part_begin) / pack] : load(a);
    #pragma unroll 1
    for(; a < run_end; a += step) {
      word_t word = next;
      if(a + step < run_end)
        next = staged ? stage[(a + step - part_begin) / pack] : load(a + step);
      #pragma unroll
      for(int h = 0; h < pack; h += batch) {
        float logits[batch];
        #pragma unroll
        for(int j = 0; j < batch; ++j) logits[j] = to_f32(word.v[h + j]);
        f(logits, (int)(a - shift) + h);
      }
    }
  }
  // f(logit, index) for the tokens of this warp's run.
  template<typename func_t>
  MGPU_DEVICE __forceinline__ void each(func_t f) const {
    each_four([&](const float (&logits)[batch], int v) {
      #pragma unroll
      for(int j = 0; j < batch; ++j) f(logits[j], v + j);
    });
  }
  // Whether no token has been dropped so far.
  MGPU_DEVICE bool all_kept() const { return 0 == least; }

  //////////////////////////////////////////////////////////////////////////////
  // Sums.

  MGPU_DEVICE static double warp_sum(double v) {
    #pragma unroll
    for(int offset = 16; offset; offset /= 2)
      v += __shfl_xor_sync(0xffffffffu, v, offset);
    return v;
  }
  MGPU_DEVICE double upto(double v) const {
    #pragma unroll
    for(int offset = 1; offset < 32; offset *= 2) {
      double y = __shfl_up_sync(0xffffffffu, v, offset);
      if(lane >= offset) v += y;
    }
    return v;
  }
  // Over the CTA's threads, in the order of the warps.
  MGPU_DEVICE double cta_upto(double v) {
    v = upto(v);
    if(31 == lane) shared.fold[0][warp] = v;
    __syncthreads();
    double others = upto(lane < warps ? shared.fold[0][lane] : 0.0);
    others = __shfl_sync(0xffffffffu, others, (warp + 31) % 32);
    __syncthreads();
    return warp ? v + others : v;
  }
  MGPU_DEVICE double cta_sum(double v) {
    v = warp_sum(v);
    if(!lane) shared.fold[0][warp] = v;
    __syncthreads();
    v = warp_sum(lane < warps ? shared.fold[0][lane] : 0.0);
    __syncthreads();
    return v;
  }
  MGPU_DEVICE uint32_t cta_max(uint32_t v) {
    uint32_t* parts = (uint32_t*)shared.fold[0];
    v = __reduce_max_sync(0xffffffffu, v);
    if(!lane) parts[warp] = v;
    __syncthreads();
    v = __reduce_max_sync(0xffffffffu, lane < warps ? parts[lane] : 0u);
    __syncthreads();
    return v;
  }
  MGPU_DEVICE uint32_t cta_min(uint32_t v) { return ~cta_max(~v); }

  // Every warp's news (the same in its lanes) to every CTA. Two sets of slots:
  // one is written again only behind a barrier that its readers have passed.
  MGPU_DEVICE const sample_news_t* share(const sample_news_t& mine) {
    if(!exchanges) ptx::cluster_wait();      // every CTA has started
    int set = exchanges++ & 1;
    if(lane < ctas)
      cluster.map_shared_rank(&shared, lane)->news[set][run] = mine;
    cluster.sync();
    return shared.news[set];
  }
  // f(news) for a part of all warps' news in each lane.
  template<typename func_t>
  MGPU_DEVICE __forceinline__ void all_news(const sample_news_t* news,
    func_t f) const {
    #pragma unroll
    for(int i = 0; i < each_lane; ++i) {
      int r = i * 32 + lane;
      if(r < ctas * warps) f(news[r]);
    }
  }

  //////////////////////////////////////////////////////////////////////////////
  // Weights.

  MGPU_DEVICE bool kept(uint32_t key, int v) const {
    return key > least || (key == least && v <= last);
  }
  // 2^(i / 64), i < 64, in shared memory.
  MGPU_DEVICE void make_powers() {
    if(tid < sample_powers)
      shared.powers[tid] = exp2((double)tid / sample_powers);
  }
  // exp((value - peak) / T) to about 1e-14 (the rounding of log2(e) / T times a
  // distance of up to 60). With y = (value - peak) log2(e) / T = i / 64 + r, r
  // at most 1/128 in size, it is 2^(i / 64) 2^r: a power from the table and the
  // Taylor series of exp(r ln 2), whose sixth-degree term is below 4e-17. Eleven
  // operations of 64 bits; the library's exp takes several times as many, and
  // these passes are bound by instructions. Below about 2^-1000 it is 0.
  MGPU_DEVICE double weight(float value) const {
    if(peak == INFINITY) return value == peak ? 1.0 : 0.0;
    const double magic = 1.5 * 70368744177664.0;       // 1.5 * 2^46: ulp 2^-6
    double d = (double)value - (double)peak;
    double z = fma(d, log2_scale, magic);
    double r = fma(d, log2_scale, -(z - magic));
    int i = __double2loint(z);
    // ln2^n / n!
    double p = 1.3333558146428443e-3;
    p = fma(p, r, 9.618129107628477e-3);
    p = fma(p, r, 5.550410866482158e-2);
    p = fma(p, r, 2.402265069591007e-1);
    p = fma(p, r, 6.931471805599453e-1);
    double t = shared.powers[i & (sample_powers - 1)];
    t = fma(t, p * r, t);
    double w = __hiloint2double(__double2hiint(t) +
      (i & ~(sample_powers - 1)) * (1 << 14), __double2loint(t));
    return value < weightless ? 0.0 : w;
  }
  template<bool by_count>
  MGPU_DEVICE double size(float value) const {
    return by_count ? 1.0 : weight(value);
  }
  // The distance from the peak in steps, at most the last one; it does not rise
  // where the logit does. The step is the nearest whole number.
  MGPU_DEVICE float steps_below(float from, float value) const {
    if(from == INFINITY) return value == from ? 0.0f : sample_bins - 1.0f;
    return fminf((from - value) * steps_per_logit, sample_bins - 1.0f);
  }
  MGPU_DEVICE static float rounder() { return 12582912.0f; }   // 1.5 * 2^23
  MGPU_DEVICE static int nearest(float rounded) {
    return __float_as_int(rounded) - 0x4b400000;
  }
  MGPU_DEVICE int bin(float value) const {
    return nearest(steps_below(peak, value) + rounder());
  }

  MGPU_DEVICE void find_peak() {
    sample_news_t mine = { };
    mine.p = part_peak();
    const sample_news_t* news = share(mine);
    uint32_t key = 0;
    all_news(news, [&](const sample_news_t& n) { key = max(key, n.p); });
    peak_key = __reduce_max_sync(0xffffffffu, key);
  }
  MGPU_DEVICE int first_of(uint32_t wanted) {
    uint32_t at = 0xffffffffu;
    each([&](float value, int v) {
      if(order_key(value) == wanted) at = min(at, (uint32_t)v);
    });
    sample_news_t mine = { };
    mine.p = __reduce_min_sync(0xffffffffu, at);
    const sample_news_t* news = share(mine);
    at = 0xffffffffu;
    all_news(news, [&](const sample_news_t& n) { at = min(at, n.p); });
    return (int)__reduce_min_sync(0xffffffffu, at);
  }

  //////////////////////////////////////////////////////////////////////////////
  // Sums of the runs, in the order of the vocabulary: the `a` of the news.

  // All runs together, in every lane.
  MGPU_DEVICE double total_of_runs(const sample_news_t* news) const {
    double sum = 0;
    all_news(news, [&](const sample_news_t& n) { sum += n.a; });
    return warp_sum(sum);
  }
  // The first run with a sum for which test(sum up to its end), and the sum
  // before it; where there is none, the last run with a sum; -1 where all are
  // 0. The same in every thread of the cluster.
  template<typename test_t>
  MGPU_DEVICE int find_run(const sample_news_t* news, test_t test,
    double& before) const {
    double own[each_lane], sum = 0;
    #pragma unroll
    for(int i = 0; i < each_lane; ++i) {
      int r = lane * each_lane + i;
      own[i] = r < ctas * warps ? news[r].a : 0.0;
      sum += own[i];
    }
    double ahead = __shfl_up_sync(0xffffffffu, upto(sum), 1);
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
  // The CTA whose run `found` is searches it: size(value, index) of the tokens
  // is added up in order, from `before`, and the first token with a size whose
  // sum passes test is the result, else the last one with a size. Each warp adds
  // up a part of the run; the part with the token is gone through 32 by 32.
  template<typename size_t_, typename test_t>
  MGPU_DEVICE int search_run(int found, double before, size_t_ size,
    test_t test) {
    int64_t length = run_length(), begin = length * found;
    int64_t end = min(begin + length, (int64_t)vocabulary + shift);
    int64_t part = div_up(div_up(length, (int64_t)warps), (int64_t)32) * 32;
    int64_t part_begin = min(begin + part * warp, end);
    int64_t part_end = min(part_begin + part, end);
    double sum = 0;
    for(int64_t a = part_begin + lane; a < part_end; a += 32)
      if(a >= shift) sum += size(logit_at(a), (int)(a - shift));
    sum = warp_sum(sum);
    if(!lane) shared.fold[0][warp] = sum;
    if(!tid) shared.hit = -1;
    __syncthreads();
    int chosen = -1;
    double chosen_before = 0;
    for(int w = 0; w < warps; ++w) {
      double own = shared.fold[0][w];
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
          size(logit_at(a), (int)(a - shift)) : 0.0;
        double sum = upto(own);
        unsigned some = __ballot_sync(0xffffffffu, own > 0);
        unsigned hits = __ballot_sync(0xffffffffu, own > 0 && test(before + sum));
        if(hits) {
          at = (int)(first - shift) + __ffs(hits) - 1;
          done = true;
        } else if(some)
          at = (int)(first - shift) + 31 - __clz(some);
        before += __shfl_sync(0xffffffffu, sum, 31);
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
    int count = 0;
    each([&](float value, int v) { count += one(value, v) > 0; });
    sample_news_t mine = { };
    mine.a = (double)__reduce_add_sync(0xffffffffu, count);
    const sample_news_t* news = share(mine);
    auto test = [&](double sum) { return sum >= nth; };
    double before = 0;
    int found = find_run(news, test, before);
    sample_news_t told = { };
    told.i = -1;
    if(found >= 0 && found / warps == rank)
      told.i = search_run(found, before, one, test);
    news = share(told);
    int at = -1;
    all_news(news, [&](const sample_news_t& n) { at = max(at, n.i); });
    return __reduce_max_sync(0xffffffffu, at);
  }

  //////////////////////////////////////////////////////////////////////////////
  // Pass 2: the steps [lo, hi] that may hold the border, about how many tokens
  // are in them (`inside`), and the most that can be in [0, hi] (`tokens`).
  // The border is where the running count reaches `target`, or the running
  // weight `target` times the weight of all.

  MGPU_DEVICE void clear_hist() {
    for(int b = tid; b < sample_bins; b += nt) shared.hist[b] = 0;
    if(!tid) shared.list_count = 0;
    __syncthreads();
  }

  template<bool by_count>
  MGPU_DEVICE band_t find_band(double target) {
    // Fixed-point weights: a step's sum stays below 2^32 whatever it holds.
    float unit = by_count ? 1.0f : fminf(4096.0f, 2147483648.0f / vocabulary);
    clear_hist();
    bool every = all_kept();
    each([&](float value, int v) {
      float s = steps_below(peak, value), rounded = s + rounder();
      uint32_t add = 1;
      if(!by_count) {
        // exp(-r / 64) for |r| <= 1/2, to 1e-7.
        float r = s - (rounded - rounder());
        add = __float_as_uint(fmaf(r, fmaf(r, unit / 8192, -unit / 64), unit) +
          8388608.0f) & 0x7fffff;
      }
      if(every || kept(order_key(value), v))
        atomicAdd(&shared.hist[nearest(rounded)], add);
    });
    if(!tid) {
      shared.band_lo = shared.band_hi = sample_bins;
      shared.band_before = shared.band_tokens = 0;
    }
    cluster.sync();

    // Each CTA adds up a slice of the steps, a few neighbouring ones to a
    // thread; a warp's are a group.
    enum { most = sample_bins / nt };
    int slice = sample_bins / ctas, each_thread = div_up(slice, (int)nt);
    int active = slice / (32 * each_thread);   // warps with steps
    int first = rank * slice + tid * each_thread;
    double weights[most], tokens[most], weight_sum = 0, token_sum = 0;
    // A token adds at least this much.
    double fewest = by_count ? 1.0 : (double)unit * 0.992 - 0.5;
    #pragma unroll
    for(int i = 0; i < most; ++i) {
      weights[i] = tokens[i] = 0;
      if(warp < active && i < each_thread) {
        uint32_t parts[sample_max_cluster];
        #pragma unroll
        for(int r = 0; r < sample_max_cluster; ++r)
          parts[r] = r < ctas ?
            cluster.map_shared_rank(&shared, r)->hist[first + i] : 0;
        double sum = 0;
        #pragma unroll
        for(int r = 0; r < sample_max_cluster; ++r) sum += parts[r];
        weights[i] = by_count ? sum :
          sum * exp(-(double)(first + i) / sample_steps);
        tokens[i] = fewest > 0 ? sum / fewest : sum * 1e30;
      }
      weight_sum += weights[i];
      token_sum += tokens[i];
    }
    double at = upto(weight_sum), at_tokens = upto(token_sum);
    int group = rank * active + warp;
    if(warp < active) {
      double w = __shfl_sync(0xffffffffu, at, 31);
      double t = __shfl_sync(0xffffffffu, at_tokens, 31);
      if(lane < ctas) {
        shared_t* there = cluster.map_shared_rank(&shared, lane);
        there->group_weights[group] = w;
        there->group_tokens[group] = t;
      }
    }
    cluster.sync();
    // Two groups to a lane: what is in front of this warp's, and of all.
    int groups = ctas * active;
    double w0 = 2 * lane < groups ? shared.group_weights[2 * lane] : 0.0;
    double w1 = 2 * lane + 1 < groups ? shared.group_weights[2 * lane + 1] : 0.0;
    double t0 = 2 * lane < groups ? shared.group_tokens[2 * lane] : 0.0;
    double t1 = 2 * lane + 1 < groups ? shared.group_tokens[2 * lane + 1] : 0.0;
    double w_upto = upto(w0 + w1), t_upto = upto(t0 + t1);
    double total = __shfl_sync(0xffffffffu, w_upto, 31);
    double all_tokens = __shfl_sync(0xffffffffu, t_upto, 31);
    double w_front = w_upto - (group & 1 ? w1 : w0 + w1);
    double t_front = t_upto - (group & 1 ? t1 : t0 + t1);
    at += __shfl_sync(0xffffffffu, w_front, group / 2 % 32) - weight_sum;
    at_tokens += __shfl_sync(0xffffffffu, t_front, group / 2 % 32) - token_sum;
    // Sum and total are each off by at most 0.51 / unit + 1e-5 of the total.
    double slack = by_count ? 0.0 : (2.0 / unit + 5e-5) * total;
    double goal = by_count ? target : target * total;
    // The thread whose steps pass a border tells all CTAs, unless the sum was
    // past it before.
    #pragma unroll
    for(int i = 0; i < most; ++i) {
      if(warp < active && i < each_thread) {
        double to = at + weights[i];
        bool is_lo = to >= goal - slack && (at < goal - slack ||
          0 == first + i);
        bool is_hi = to >= goal + slack && (at < goal + slack ||
          0 == first + i);
        if(is_lo || is_hi)
          for(int r = 0; r < ctas; ++r) {
            shared_t* there = cluster.map_shared_rank(&shared, r);
            if(is_lo) {
              there->band_lo = first + i;
              there->band_before = at_tokens;
            }
            if(is_hi) {
              there->band_hi = first + i;
              there->band_tokens = at_tokens + tokens[i];
            }
          }
        at = to;
        at_tokens += tokens[i];
      }
    }
    cluster.sync();
    band_t band { shared.band_lo, shared.band_hi, shared.band_tokens, 0 };
    double before = shared.band_before;
    if(band.hi == sample_bins) {
      band.hi = sample_bins - 1;
      band.tokens = all_tokens;
    }
    if(band.lo > band.hi) {
      band.lo = 0;
      before = 0;
    }
    band.inside = band.tokens - before;
    return band;
  }

  //////////////////////////////////////////////////////////////////////////////
  // The list, in the first CTA.

  MGPU_DEVICE static unsigned long long entry(uint32_t key, int v) {
    return (unsigned long long)key << 32 | (0xffffffffu - v);
  }
  // Each CTA appends to a list of its own; the first one fetches them.
  MGPU_DEVICE void append(uint32_t key, int v) {
    int at = atomicAdd(&shared.list_count, 1);
    if(at < sample_list) shared.list[at] = entry(key, v);
  }
  // For at most sample_list entries in all, behind a barrier of the cluster. The
  // others keep their lists until they have passed another one. The histogram's
  // memory is free by now.
  MGPU_DEVICE void fetch_lists() {
    unsigned long long* all = (unsigned long long*)shared.hist;
    int counts[sample_max_cluster], count = 0;
    #pragma unroll
    for(int r = 0; r < sample_max_cluster; ++r)
      counts[r] = r < ctas ?
        min(cluster.map_shared_rank(&shared, r)->list_count, (int)sample_list) :
        0;
    #pragma unroll
    for(int r = 0; r < sample_max_cluster; ++r) {
      for(int i = tid; i < counts[r]; i += nt)
        if(count + i < sample_list)
          all[count + i] = cluster.map_shared_rank(&shared, r)->list[i];
      count += counts[r];
    }
    // The first CTA's own entries stay in front, in its weights' memory.
    unsigned long long* own = (unsigned long long*)shared.list_weights;
    for(int i = tid; i < counts[0]; i += nt) own[i] = shared.list[i];
    __syncthreads();
    for(int i = tid; i < count && i < sample_list; i += nt)
      shared.list[i] = all[i];
    __syncthreads();
  }
  // The CTA's own list behind fetch_lists.
  MGPU_DEVICE const unsigned long long* own_list() const {
    return rank ? shared.list : (unsigned long long*)shared.list_weights;
  }
  MGPU_DEVICE uint32_t list_key(int i) const {
    return (uint32_t)(shared.list[i] >> 32);
  }
  MGPU_DEVICE int list_index(int i) const {
    return (int)(0xffffffffu - (uint32_t)shared.list[i]);
  }
  // The greatest first; equal keys by index. A bitonic network: what stays
  // within 64 entries is a warp's own.
  MGPU_DEVICE void sort_list(int count) {
    int n = 64;
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
        if(j > 32 || (1 == j && k >= 64)) __syncthreads();
        else __syncwarp();
      }
    __syncthreads();
  }
  // The first place, in the list's order, of an entry with a size for which
  // test(the sum up to it); else the last entry with a size.
  template<typename size_t_, typename test_t>
  MGPU_DEVICE int search_list(int count, size_t_ size, test_t test) {
    double own[each_list], sum = 0;
    #pragma unroll
    for(int i = 0; i < each_list; ++i) {
      int e = tid * each_list + i;
      own[i] = e < count ? size(e) : 0.0;
      sum += own[i];
    }
    double at = cta_upto(sum) - sum;
    uint32_t found = 0xffffffffu, any = 0;
    #pragma unroll
    for(int i = 0; i < each_list; ++i) {
      at += own[i];
      if(own[i] > 0) {
        any = tid * each_list + i + 1;
        if(0xffffffffu == found && test(at)) found = any - 1;
      }
    }
    found = cta_min(found);
    any = cta_max(any);
    return 0xffffffffu != found ? (int)found : (int)any - 1;
  }

  // The first CTA alone: the sorted list's first `count` entries are all tokens
  // that may be kept, `total` is the weight that top-p refers to (below 0: that
  // of these entries).
  MGPU_DEVICE int finish_list(int count, double total, float top_p, float min_p,
    double u) {
    for(int e = tid; e < count; e += nt)
      shared.list_weights[e] = weight(key_value(list_key(e)));
    __syncthreads();
    if(count <= 128) {
      if(!warp) {
        int token = finish_short(count, total, top_p, min_p, u);
        if(!lane) shared.hit = token;
      }
      __syncthreads();
      return shared.hit;
    }
    auto by_place = [&](int e) { return shared.list_weights[e]; };
    if(top_p < 1) {
      if(total < 0) {
        double sum = 0;
        for(int e = tid; e < count; e += nt) sum += by_place(e);
        total = cta_sum(sum);
      }
      double target = (double)top_p * total;
      count = search_list(count, by_place,
        [&](double sum) { return sum >= target; }) + 1;
    }
    if(min_p > 0) {
      // Weights fall along the list.
      uint32_t fit = 0;
      for(int e = tid; e < count; e += nt)
        if(list_key(e) == peak_key || by_place(e) >= (double)min_p) fit = e + 1;
      count = (int)cta_max(fit);
    }
    // By index, with the key in the low half.
    for(int e = tid; e < count; e += nt) {
      unsigned long long old = shared.list[e];
      shared.list[e] = old << 32 | old >> 32;
    }
    sort_list(count);
    double sum = 0;
    for(int e = tid; e < count; e += nt) {
      shared.list_weights[e] = weight(key_value((uint32_t)shared.list[e]));
      sum += shared.list_weights[e];
    }
    double target = u * cta_sum(sum);
    int e = search_list(count, by_place,
      [&](double sum) { return sum > target; });
    return (int)(0xffffffffu - (uint32_t)(shared.list[e] >> 32));
  }
  // The same for at most 128 entries, by one warp with four to a lane. The draw
  // adds up, for each entry, those of no higher index.
  MGPU_DEVICE int finish_short(int count, double total, float top_p,
    float min_p, double u) {
    double own[4], sum = 0;
    #pragma unroll
    for(int i = 0; i < 4; ++i) {
      int e = lane * 4 + i;
      own[i] = e < count ? shared.list_weights[e] : 0.0;
      sum += own[i];
    }
    if(top_p < 1) {
      double at = upto(sum);
      if(total < 0) total = __shfl_sync(0xffffffffu, at, 31);
      double target = (double)top_p * total;
      at -= sum;
      uint32_t found = 0xffffffffu, any = 0;
      #pragma unroll
      for(int i = 0; i < 4; ++i) {
        at += own[i];
        if(own[i] > 0) {
          any = lane * 4 + i + 1;
          if(0xffffffffu == found && at >= target) found = any;
        }
      }
      found = __reduce_min_sync(0xffffffffu, found);
      any = __reduce_max_sync(0xffffffffu, any);
      count = (int)(0xffffffffu != found ? found : any);
    }
    if(min_p > 0) {
      uint32_t fit = 0;
      #pragma unroll
      for(int i = 0; i < 4; ++i) {
        int e = lane * 4 + i;
        if(e < count && (list_key(e) == peak_key || own[i] >= (double)min_p))
          fit = e + 1;
      }
      count = (int)__reduce_max_sync(0xffffffffu, fit);
    }
    double upto_mine[4] = { 0, 0, 0, 0 };
    int index[4];
    #pragma unroll
    for(int i = 0; i < 4; ++i)
      index[i] = lane * 4 + i < count ? list_index(lane * 4 + i) : -1;
    sum = 0;
    #pragma unroll 4
    for(int q = 0; q < count; ++q) {
      double w = shared.list_weights[q];
      int at = list_index(q);
      sum += w;
      #pragma unroll
      for(int i = 0; i < 4; ++i)
        upto_mine[i] += at <= index[i] ? w : 0.0;
    }
    double target = u * sum;
    uint32_t hit = 0xffffffffu, any = 0;
    #pragma unroll
    for(int i = 0; i < 4; ++i) {
      int e = lane * 4 + i;
      if(e < count && own[i] > 0) {
        uint32_t at = (uint32_t)index[i];
        any = max(any, at);
        if(upto_mine[i] > target) hit = min(hit, at);
      }
    }
    hit = __reduce_min_sync(0xffffffffu, hit);
    any = __reduce_max_sync(0xffffffffu, any);
    return (int)(0xffffffffu != hit ? hit : any);
  }

  //////////////////////////////////////////////////////////////////////////////
  // Top-k of few tokens. Instead of a common histogram every CTA takes one of
  // its own part, from its own peak down, and lists what may be among the row's
  // greatest. The row's peak key is known behind it. True where the first CTA's
  // list, `listed` long, holds the greatest top_k; false where a part has too
  // many equal tokens for its share of the list.
  MGPU_DEVICE bool list_greatest(int top_k, int& listed) {
    uint32_t part_key = cta_max(part_peak());
    float from = key_value(part_key);
    bool some = part_key != 0xffffffffu && from > -INFINITY;
    clear_hist();
    auto step = [&](float value) {
      return nearest(steps_below(from, value) + rounder());
    };
    if(some)
      each([&](float value, int) { atomicAdd(&shared.hist[step(value)], 1u); });
    __syncthreads();
    // The step in which the count reaches top_k.
    enum { most = sample_bins / nt };
    int counts[most], sum = 0;
    #pragma unroll
    for(int i = 0; i < most; ++i) {
      counts[i] = (int)shared.hist[tid * most + i];
      sum += counts[i];
    }
    int at = (int)cta_upto((double)sum) - sum;
    uint32_t border = sample_bins - 1, taken = 0;
    #pragma unroll
    for(int i = 0; i < most; ++i) {
      at += counts[i];
      if(at >= top_k && border == sample_bins - 1) {
        border = tid * most + i;
        taken = at;
      }
    }
    border = cta_min(border);
    // What is in the steps up to it: the count of the thread that has it, or
    // all.
    bool has = (int)border / most == tid && taken;
    uint32_t in_list = cta_max(has ? taken : 0);
    uint32_t all = cta_max(tid == nt - 1 ? (uint32_t)at : 0);
    if(border == sample_bins - 1) in_list = all;
    sample_news_t mine = { };
    mine.p = part_key;
    mine.i = (int)in_list;
    const sample_news_t* news = share(mine);
    uint32_t key = 0;
    int before = 0, total = 0;
    bool fits = true;
    for(int r = 0; r < ctas; ++r) {
      key = max(key, news[r * warps].p);
      if(r == rank) before = total;
      total += news[r * warps].i;
    }
    fits = total <= sample_list;
    peak_key = key;
    listed = total;
    if(!fits || 0xffffffffu == key) return fits;
    if(!tid) shared.list_count = before;
    __syncthreads();
    if(some) {
      shared_t* first = cluster.map_shared_rank(&shared, 0);
      each([&](float value, int v) {
        if(step(value) <= (int)border) {
          int to = atomicAdd(&shared.list_count, 1);
          if(to < sample_list) first->list[to] = entry(order_key(value), v);
        }
      });
    }
    cluster.sync();
    return true;
  }

  //////////////////////////////////////////////////////////////////////////////
  // Pass 3 and what follows from it: `least` and `last` for the tokens above
  // the border. True where the list holds all that is left; the weight of what
  // was kept before is in `total`, the list's length in `listed`. Where it is known
  // at the end what is left in each run, it is in run_left, and `drawable` is set.

  template<bool by_count>
  MGPU_DEVICE bool find_border(double target, float min_p, double& total,
    int& listed, bool& drawable) {
    band_t band = find_band<by_count>(target);
    bool whole = band.tokens <= sample_list;
    bool list = whole || band.inside <= 1.25 * sample_list;
    double above = 0, all = 0, left = 0;
    uint32_t low = 0xffffffffu, high = 0;
    int inside = 0, appended = 0;
    bool every = all_kept();
    each_four([&](const float (&logits)[batch], int v) {
      // Without branches between the four, so that their chains of dependent
      // 64-bit operations overlap.
      bool live[batch], some = false;
      int bins[batch];
      #pragma unroll
      for(int j = 0; j < batch; ++j) {
        bins[j] = bin(logits[j]);
        live[j] = every || kept(order_key(logits[j]), v + j);
        if(by_count) live[j] = live[j] && bins[j] <= band.hi;
        some = some || live[j];
      }
      if(!some) return;
      double weights[batch];
      #pragma unroll
      for(int j = 0; j < batch; ++j) weights[j] = size<by_count>(logits[j]);
      bool listed = false;
      #pragma unroll
      for(int j = 0; j < batch; ++j) {
        double w = live[j] ? weights[j] : 0.0;
        live[j] = live[j] && bins[j] <= band.hi;
        bool in = live[j] && bins[j] >= band.lo;
        all += w;
        w = bins[j] < band.lo ? w : 0.0;
        above += w;
        if(!by_count && min_p > 0)
          left += w >= (double)min_p || logits[j] == peak ? w : 0.0;
        inside += in;
        live[j] = whole ? live[j] : in;
        listed = listed || live[j];
      }
      if(listed) {
        #pragma unroll
        for(int j = 0; j < batch; ++j)
          if(live[j]) {
            uint32_t key = order_key(logits[j]);
            low = min(low, key);
            high = max(high, key);
            if(list) {
              append(key, v + j);
              ++appended;
            }
          }
      }
    });
    sample_news_t mine = { };
    mine.a = warp_sum(above);
    mine.b = warp_sum(all);
    run_left = !by_count && min_p > 0 ? warp_sum(left) : mine.a;
    mine.p = __reduce_min_sync(0xffffffffu, low);
    mine.q = __reduce_max_sync(0xffffffffu, high);
    mine.i = __reduce_add_sync(0xffffffffu, inside);
    mine.j = __reduce_add_sync(0xffffffffu, appended);
    const sample_news_t* news = share(mine);
    above = all = 0;
    low = 0xffffffffu;
    high = 0;
    inside = appended = 0;
    all_news(news, [&](const sample_news_t& n) {
      above += n.a;
      all += n.b;
      low = min(low, n.p);
      high = max(high, n.q);
      inside += n.i;
      appended += n.j;
    });
    above = warp_sum(above);
    all = warp_sum(all);
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    inside = __reduce_add_sync(0xffffffffu, inside);
    appended = __reduce_add_sync(0xffffffffu, appended);
    total = all;
    listed = appended;
    if(!by_count) target *= all;
    // Holds by the bound on the steps' tokens; else the border is looked for.
    if(whole && appended <= sample_list) {
      if(!rank) fetch_lists();
      cluster.sync();
      return true;
    }
    list = list && !whole && appended <= sample_list;

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
      mine.a = warp_sum(upper);
      mine.p = __reduce_min_sync(0xffffffffu, upper_low);
      mine.q = __reduce_max_sync(0xffffffffu, lower_high);
      mine.i = __reduce_add_sync(0xffffffffu, upper_count);
      news = share(mine);
      upper = 0;
      upper_low = 0xffffffffu;
      lower_high = 0;
      upper_count = 0;
      all_news(news, [&](const sample_news_t& n) {
        upper += n.a;
        upper_low = min(upper_low, n.p);
        lower_high = max(lower_high, n.q);
        upper_count += n.i;
      });
      upper = warp_sum(upper);
      upper_low = __reduce_min_sync(0xffffffffu, upper_low);
      lower_high = __reduce_max_sync(0xffffffffu, lower_high);
      upper_count = __reduce_add_sync(0xffffffffu, upper_count);
      if(above + upper >= target) {
        low = upper_low;
        inside = upper_count;
      } else {
        above += upper;
        high = lower_high;
        inside -= upper_count;
      }
    }
    if(inside > sample_list || low == high) {
      // One value: as many of its tokens as it takes.
      double need = ceil((target - above) / size<by_count>(key_value(low)));
      need = need > 1 ? (need < vocabulary ? need : vocabulary) : 1;
      int at = nth_equal(low, need);
      least = low;
      last = at;
      return false;
    }
    if(!list) {
      if(!tid) shared.list_count = 0;
      __syncthreads();
      each([&](float value, int v) {
        uint32_t key = order_key(value);
        if(key >= low && key <= high && kept(key, v)) append(key, v);
      });
      cluster.sync();
    }
    mine = sample_news_t { };
    int own_listed = shared.list_count;
    if(!rank) {
      fetch_lists();
      sort_list(inside);
      int e = search_list(inside, [&](int e) {
          return size<by_count>(key_value(list_key(e)));
        }, [&](double sum) { return above + sum >= target; });
      e = max(e, 0);
      mine.p = list_key(e);
      mine.i = list_index(e);
    }
    news = share(mine);
    least = news[0].p;
    last = news[0].i;
    if(list && !by_count) {
      // Of the steps at the border only the listed tokens matter.
      int64_t length = run_length();
      double sum = 0;
      for(int i = lane; i < own_listed; i += 32) {
        unsigned long long e = own_list()[i];
        uint32_t key = (uint32_t)(e >> 32);
        int v = (int)(0xffffffffu - (uint32_t)e);
        double w = weight(key_value(key));
        if((v + (int64_t)shift) / length == run && kept(key, v) &&
          (w >= (double)min_p || key == peak_key)) sum += w;
      }
      run_left += warp_sum(sum);
      drawable = true;
    }
    return false;
  }

  // Pass 4.
  MGPU_DEVICE void draw(float min_p, double u, bool drawable, int* token) {
    auto left = [&](float value, int v) {
      uint32_t key = order_key(value);
      if(!kept(key, v)) return 0.0;
      double w = weight(value);
      return w >= (double)min_p || key == peak_key ? w : 0.0;
    };
    double sum = 0;
    bool every = all_kept();
    if(!drawable) each_four([&](const float (&logits)[batch], int v) {
      bool live[batch], some = false;
      #pragma unroll
      for(int j = 0; j < batch; ++j) {
        live[j] = every || kept(order_key(logits[j]), v + j);
        some = some || live[j];
      }
      if(!some) return;
      double weights[batch];
      #pragma unroll
      for(int j = 0; j < batch; ++j) weights[j] = weight(logits[j]);
      #pragma unroll
      for(int j = 0; j < batch; ++j) {
        live[j] = live[j] &&
          (weights[j] >= (double)min_p || logits[j] == peak);
        sum += live[j] ? weights[j] : 0.0;
      }
    });
    sample_news_t mine = { };
    mine.a = drawable ? run_left : warp_sum(sum);
    const sample_news_t* news = share(mine);
    double target = u * total_of_runs(news), before = 0;
    auto test = [&](double s) { return s > target; };
    int found = find_run(news, test, before);
    if(found >= 0 && found / warps == rank) {
      int at = search_run(found, before, left, test);
      if(!tid) *token = at;
    }
  }
};

template<int nt, bool staged, typename real_t>
__global__ void __launch_bounds__(nt, 1024 / nt)
sample_k(const real_t* logits, int64_t stride, int vocabulary,
  const float* uniforms, sampling_t settings, int* tokens, int ctas) {
  extern __shared__ __align__(16) char sample_memory[];
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

  typedef sample_cta_t<nt, staged, real_t> cta_t;
  cta_t cta(logits + at * stride, (typename cta_t::word_t*)sample_memory,
    vocabulary, shared);
  bool leader = !cta.rank && !cta.tid;
  if(!cta.tid) shared.list_count = 0;
  cta.make_powers();
  cta.log2_scale = 1.4426950408889634 / (double)temperature;
  cta.steps_per_logit = (float)sample_steps / temperature;
  // A part's list holds its greatest top_k and its border's equals.
  bool by_k = temperature > 0 && top_k > 0 && top_k < vocabulary;
  bool listed = false, peaked = false, drawable = false;
  double total = -1;
  int count = 0;
  if(by_k && top_k <= sample_list / 2 / ctas) {
    listed = cta.list_greatest(top_k, count);
    peaked = true;
  }
  if(!peaked) cta.find_peak();
  cta.peak = key_value(cta.peak_key);
  // (-infinity has none, whatever the temperature.)
  cta.weightless = fmaxf(cta.peak - 690.0f * temperature, -FLT_MAX);
  if(0xffffffffu == cta.peak_key || !(cta.peak > -INFINITY)) {
    if(leader) tokens[at] = -1;
  } else if(!(temperature > 0)) {
    int first = cta.first_of(cta.peak_key);
    if(leader) tokens[at] = first;
  } else {
    if(by_k && !listed) {
      listed = cta.template find_border<true>((double)top_k, min_p, total,
        count, drawable);
      // The weight that top-p refers to is that of the first top_k.
      total = -1;
    }
    bool first_k = listed;
    if(!listed && top_p < 1)
      listed = cta.template find_border<false>((double)top_p, min_p, total,
        count, drawable);
    if(!listed)
      cta.draw(min_p, u, drawable, tokens + at);
    else if(!cta.rank) {
      cta.sort_list(count);
      int token = cta.finish_list(first_k ? min(count, top_k) : count, total,
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
  // CTAs to a row: at most 65,536 tokens to a CTA, so that no row takes much
  // longer than the others (256 mixed rows of 100,003: 224 us with one CTA to a
  // row, 142 us with two, 151 us with four), and a CTA for each SM where there
  // are few rows (64 rows of 131,072: 80 us with four, 102 us with eight, whose
  // clusters need two rounds). Parts up to 72 KB stay in shared memory, which
  // leaves room for two CTAs on an SM.
  enum { nt = 512, most_stage = 72 << 10, sms = 148 };
  auto stage_bytes = [&](int n) {
    int64_t step = 32 * (16 / (int)sizeof(real_t));
    return div_up(div_up((int64_t)vocabulary + 8, (int64_t)n * (nt / 32)), step) *
      step * (nt / 32) * (int64_t)sizeof(real_t);
  };
  int ctas = 1;
  while(ctas < sample_max_cluster && vocabulary / ctas > 2 * nt &&
    ((int64_t)count * ctas < sms || vocabulary / ctas > (1 << 16))) ctas *= 2;
  bool staged = stage_bytes(ctas) <= most_stage;
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
  auto launch = [&](auto kernel) {
    throw_on_error(cudaLaunchKernelEx(&config, kernel, logits, stride,
      vocabulary, uniforms, settings, tokens, ctas));
  };
  if(staged) {
    auto kernel = sample_k<nt, true, real_t>;
    set_dynamic_smem<real_t>(kernel, most_stage);
    config.dynamicSmemBytes = (size_t)stage_bytes(ctas);
    launch(kernel);
  } else
    launch(sample_k<nt, false, real_t>);
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
