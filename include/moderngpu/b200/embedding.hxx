// Embedding rows by token, and the gradient of the table they come from.
//
//   lookup:    output[i] = scale * table[tokens[i]]
//   gradient:  output[r] = scale * sum of grad[i] over the i with tokens[i] = r
//
// The lookup is interval_gather with whole rows for elements. The gradient is
// a segmented reduction with whole rows for items: the positions are sorted by
// token (stable, so that equal tokens keep the order of their positions), and
// the sorted positions are cut into tiles of equal length, whatever the lengths
// of the runs of equal tokens. A run that crosses tiles leaves a partial sum in
// each; the CTA that comes last adds them up, in order. Rows that no token
// names are segments without items: a kernel of their own zeroes them while the
// sort, which needs few SMs, is running.
//
// A token outside of [0, rows) stands for no row (padding): the lookup gives
// zeros for it, the gradient leaves its position out.
//
// Sums are held in 32 bits in the order of the positions; the same call gives
// the same bits every time.
#pragma once
#include "runtime.hxx"
#include "real_types.hxx"
#include "scan.hxx"
#ifdef __CUDACC__
#include <cooperative_groups.h>
#endif

BEGIN_MGPU_NAMESPACE

#ifdef __CUDACC__

namespace detail {

////////////////////////////////////////////////////////////////////////////////
// Lookup.

// Rows of a table are read once each and written once: the kernel is bound by
// HBM bytes. `lanes` threads (a power of two) share a row, so that a narrow row
// does not idle most of a CTA; each thread has packs of up to 16 bytes of `batch`
// rows in flight.
template<int nt, int pack, int batch, typename real_t, typename token_t>
__global__ void __launch_bounds__(nt)
embedding_lookup_k(const real_t* table, int64_t rows, int width,
  int64_t stride, const token_t* tokens, int64_t count, float scale,
  real_t* output, int lanes, int streaming) {
  typedef pack_t<real_t, pack> word_t;
  int lane = (int)threadIdx.x & (lanes - 1), groups = nt / lanes;
  int64_t first = (int64_t)blockIdx.x * (groups * batch) +
    (int)threadIdx.x / lanes;
  int64_t from[batch];
  #pragma unroll
  for(int b = 0; b < batch; ++b) {
    int64_t i = first + b * groups;
    int64_t row = i < count ? (int64_t)tokens[i] : -1;
    from[b] = row >= 0 && row < rows ? row * stride : -1;
  }
  for(int c = lane * pack; c < width; c += lanes * pack) {
    word_t words[batch];
    #pragma unroll
    for(int b = 0; b < batch; ++b)
      if(from[b] >= 0) words[b] = *(const word_t*)(table + from[b] + c);
    #pragma unroll
    for(int b = 0; b < batch; ++b) {
      int64_t i = first + b * groups;
      #pragma unroll
      for(int j = 0; j < pack; ++j)
        words[b].v[j] = from_f32<real_t>(from[b] >= 0 ?
          to_f32(words[b].v[j]) * scale : 0.0f);
      word_t* to = (word_t*)(output + i * width + c);
      if(i < count) {
        if(streaming) store_streaming(to, words[b]);
        else *to = words[b];
      }
    }
  }
}

template<typename real_t, typename token_t>
void embedding_lookup_enqueue(const real_t* table, int64_t rows, int width,
  int64_t stride, const token_t* tokens, int64_t count, float scale,
  real_t* output, cudaStream_t stream) {
  if(!count || !width) return;
  int pack = min(pack_limit(table, stride, width, (int)sizeof(real_t)),
    pack_limit(output, width, width, (int)sizeof(real_t)));
  // Rows that stay in the L2 for whoever reads them next are stored plainly; an
  // output beyond half of the L2 leaves it at once, and the rows of frequent
  // tokens stay instead (16,384 rows of 8 KB: 37.2 us, 40.7 us without).
  int streaming = (size_t)count * width * sizeof(real_t) > (64u << 20);
  auto launch = [&](auto pack_tag, auto nt_tag, auto batch_tag) {
    enum { nt = decltype(nt_tag)::value, batch = decltype(batch_tag)::value };
    int lanes = 1;
    while(lanes < nt && lanes * pack < width) lanes *= 2;
    unsigned grid = (unsigned)div_up(count, (int64_t)(nt / lanes) * batch);
    embedding_lookup_k<nt, decltype(pack_tag)::value, batch, real_t, token_t>
      <<<grid, nt, 0, stream>>>(table, rows, width, stride, tokens, count,
        scale, output, lanes, streaming);
  };
  // With a word for each of the GPU's threads a call is bound by latency: one
  // row for each thread in the largest CTAs (16 rows of 8 KB: 2.1 us, four rows
  // a thread 3.5 us); above, by the loads in flight: four rows (16,384 rows:
  // 42.2 us and 37.2 us; 5,003 rows of 1,021 floats: 9.3 us and 7.5 us).
  bool small = count * (int64_t)div_up(width, pack) <= 148 * 2048;
  with_pack(pack, [&](auto tag) {
    typedef std::integral_constant<int, (sizeof(real_t) == 2 ||
      (int)decltype(tag)::value < 8 ? (int)decltype(tag)::value : 4)> pack_tag;
    if(small) launch(pack_tag(), std::integral_constant<int, 256>(),
      std::integral_constant<int, 1>());
    else launch(pack_tag(), std::integral_constant<int, 128>(),
      std::integral_constant<int, 4>());
  });
  throw_on_error(cudaGetLastError());
}

////////////////////////////////////////////////////////////////////////////////
// Positions sorted by token: a stable radix sort, least significant digit
// first, of the pairs (row, position). Tokens that name no row become the key
// `rows` and end up behind all others. Two forms: one cluster of CTAs that keeps
// the pairs in shared memory (up to 131,072 positions, one launch), and three
// launches a digit for any number.

enum { token_sort_nt = 256, token_sort_vt = 16,
  token_sort_nv = token_sort_nt * token_sort_vt, token_digit_bits = 9,
  token_digits = 1 << token_digit_bits };

inline int token_bits(int rows) {
  int bits = 1;
  while(bits < 32 && ((uint64_t)rows >> bits)) ++bits;   // keys 0 .. rows
  return bits;
}

// The keys of the first pass come from the caller's tokens.
template<typename token_t>
struct token_keys_t {
  const token_t* tokens;
  int rows;
  MGPU_DEVICE uint32_t key(int i) const {
    int64_t t = (int64_t)tokens[i];
    return t >= 0 && t < rows ? (uint32_t)t : (uint32_t)rows;
  }
  MGPU_DEVICE int position(int i) const { return i; }
};
struct sorted_keys_t {
  const uint32_t* keys;
  const int* positions;
  MGPU_DEVICE uint32_t key(int i) const { return keys[i]; }
  MGPU_DEVICE int position(int i) const { return positions[i]; }
};

// The live lanes of a warp with the same digit: a vote for each bit, all in
// flight at once; one match instruction takes longer.
MGPU_DEVICE __forceinline__ unsigned warp_peers(uint32_t digit, int bits,
  bool live) {
  unsigned peers = __ballot_sync(0xffffffffu, live);
  #pragma unroll
  for(int b = 0; b < token_digit_bits; ++b)
    if(b < bits) {
      bool one = digit >> b & 1;
      unsigned votes = __ballot_sync(0xffffffffu, one);
      peers &= one ? votes : ~votes;
    }
  return peers;
}

// counts[digit * tiles + tile]: how often the digit occurs in the tile.
template<typename source_t>
__global__ void __launch_bounds__(token_sort_nt)
token_count_k(source_t source, int count, int shift, int tiles, int* counts) {
  __shared__ int hist[token_digits];
  for(int d = threadIdx.x; d < token_digits; d += token_sort_nt) hist[d] = 0;
  __syncthreads();
  int first = (int)blockIdx.x * token_sort_nv;
  for(int j = 0; j < token_sort_vt; ++j) {
    int64_t i = (int64_t)first + j * token_sort_nt + threadIdx.x;
    if(i < count)
      atomicAdd(&hist[(source.key((int)i) >> shift) & (token_digits - 1)], 1);
  }
  __syncthreads();
  for(int d = threadIdx.x; d < token_digits; d += token_sort_nt)
    counts[(size_t)d * tiles + blockIdx.x] = hist[d];
}

// Each warp owns a run of 32 * vt neighbouring elements and takes them 32 at a
// time in order; lanes with equal digits find one another by votes, so
// an element's place among its equals follows its index.
template<typename source_t>
__global__ void __launch_bounds__(token_sort_nt)
token_scatter_k(source_t source, int count, int shift, int tiles,
  const int* starts, uint32_t* keys_out, int* positions_out) {
  enum { warps = token_sort_nt / 32 };
  __shared__ int seen[warps][token_digits];
  int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for(int d = threadIdx.x; d < warps * token_digits; d += token_sort_nt)
    (&seen[0][0])[d] = 0;
  __syncthreads();
  int64_t first = (int64_t)blockIdx.x * token_sort_nv +
    warp * (32 * token_sort_vt);
  uint32_t keys[token_sort_vt];
  int places[token_sort_vt];
  #pragma unroll
  for(int j = 0; j < token_sort_vt; ++j) {
    int64_t i = first + j * 32 + lane;
    keys[j] = i < count ? source.key((int)i) : 0xffffffffu;
  }
  #pragma unroll
  for(int j = 0; j < token_sort_vt; ++j) {
    bool live = first + j * 32 + lane < count;
    uint32_t digit = (keys[j] >> shift) & (token_digits - 1);
    unsigned peers = warp_peers(digit, token_digit_bits, live);
    int ahead = __popc(peers & ((1u << lane) - 1));
    int before = seen[warp][digit];
    __syncwarp();
    if(live && !ahead) seen[warp][digit] = before + __popc(peers);
    __syncwarp();
    places[j] = before + ahead;
  }
  __syncthreads();
  for(int d = threadIdx.x; d < token_digits; d += token_sort_nt) {
    int sum = starts[(size_t)d * tiles + blockIdx.x];
    for(int w = 0; w < warps; ++w) {
      int c = seen[w][d];
      seen[w][d] = sum;
      sum += c;
    }
  }
  __syncthreads();
  #pragma unroll
  for(int j = 0; j < token_sort_vt; ++j) {
    int64_t i = first + j * 32 + lane;
    if(i < count) {
      int to = seen[warp][(keys[j] >> shift) & (token_digits - 1)] + places[j];
      // Within the array also where the scan has given up.
      if((unsigned)to < (unsigned)count) {
        keys_out[to] = keys[j];
        positions_out[to] = source.position((int)i);
      }
    }
  }
}

// Each warp owns a run of neighbouring pairs, 32 at a time in order, and has
// them in registers between the passes. Lanes with equal digits find one another
// by votes; a pair's place is the number of pairs with a smaller digit, of the
// CTAs and warps before it with the same digit, and of its equals before it in
// its own warp. Bound by the latency of its barriers and votes: 2,048 positions
// 8 us, 16,384 14 us, two passes each. A
// local order in front of the writes to other CTAs gained nothing, one match
// instruction instead of the votes cost 0.2 us, 2,048 pairs to a CTA instead of
// 512 cost 2 us.
enum { token_cluster_nt = 512, token_cluster_most = 8 };

template<int vt>
struct token_cluster_shared_t {
  enum { warps = token_cluster_nt / 32, nv = token_cluster_nt * vt };
  unsigned long long pairs[nv];          // key, and the position above it
  MGPU_ALIGN(16) uint16_t seen[warps][token_digits];
  int2 totals[token_cluster_most][token_digits / 2];
  int starts[token_digits];
  int warp_sums[warps];
};

template<int vt, typename token_t>
__global__ void __launch_bounds__(token_cluster_nt)
token_cluster_sort_k(token_keys_t<token_t> source, int count, int bits,
  int passes, int ctas, uint32_t* keys_out, int* positions_out, int* counters,
  int64_t num_counters) {
  enum { nt = token_cluster_nt, warps = nt / 32 };
  static_assert((int)nt * 2 >= (int)token_digits && (int)nt * vt < 65536,
    "two digits to a thread, places in 16 bits");
  extern __shared__ __align__(16) char token_cluster_memory[];
  typedef token_cluster_shared_t<vt> shared_t;
  shared_t& shared = *(shared_t*)token_cluster_memory;
  auto cluster = cooperative_groups::this_cluster();
  ptx::cluster_arrive_relaxed();
  // The kernel that follows zeroes the rows without a token meanwhile.
  ptx::grid_launch_dependents();

  int rank = (int)cluster.block_rank(), tid = (int)threadIdx.x;
  int warp = tid / 32, lane = tid % 32;
  int rounds = div_up(div_up(count, ctas * warps), 32);
  int per_warp = rounds * 32, per_cta = per_warp * warps;
  int first = rank * per_cta + warp * per_warp;

  uint32_t keys[vt];
  int positions[vt];
  #pragma unroll
  for(int j = 0; j < vt; ++j) {
    int i = first + j * 32 + lane;
    if(j < rounds) keys[j] = i < count ? source.key(i) : 0;
    positions[j] = i;
  }
  for(int64_t i = rank * nt + tid; i < num_counters; i += ctas * nt)
    counters[i] = 0;
  int digit_bits = div_up(bits, passes), digits = 1 << digit_bits;
  for(int pass = 0; pass < passes; ++pass) {
    int shift = pass * digit_bits;
    for(int d = tid * 8; d < warps * token_digits; d += nt * 8)
      if(d % token_digits < digits)
        *(uint4*)(&shared.seen[0][0] + d) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    uint32_t places[vt];
    #pragma unroll
    for(int j = 0; j < vt; ++j) {
      if(j < rounds) {
        bool live = first + j * 32 + lane < count;
        uint32_t digit = keys[j] >> shift & (digits - 1);
        unsigned peers = warp_peers(digit, digit_bits, live);
        int ahead = __popc(peers & ((1u << lane) - 1));
        int before = shared.seen[warp][digit];
        __syncwarp();
        if(live && !ahead)
          shared.seen[warp][digit] = (uint16_t)(before + __popc(peers));
        __syncwarp();
        places[j] = before + ahead;
      }
    }
    __syncthreads();
    if(!pass) ptx::cluster_wait();           // every CTA has started
    // Two digits to a thread, in the halves of a word: the warps' counts become
    // places in the CTA, and every CTA is told the CTA's totals.
    if(tid * 2 < digits) {
      uint32_t sum = 0, counts[warps];
      #pragma unroll
      for(int w = 0; w < warps; ++w)
        counts[w] = ((uint32_t*)shared.seen[w])[tid];
      #pragma unroll
      for(int w = 0; w < warps; ++w) {
        ((uint32_t*)shared.seen[w])[tid] = sum;
        sum += counts[w];
      }
      for(int r = 0; r < ctas; ++r)
        cluster.map_shared_rank(&shared, r)->totals[rank][tid] =
          make_int2(sum & 0xffff, sum >> 16);
    }
    // Also: every CTA has its pairs in registers.
    cluster.sync();
    int2 before = make_int2(0, 0), all = before;
    int upto = 0;
    if(tid * 2 < digits) {
      #pragma unroll
      for(int r = 0; r < token_cluster_most; ++r) {
        if(r < ctas) {
          int2 c = shared.totals[r][tid];
          if(r < rank) { before.x += c.x; before.y += c.y; }
          all.x += c.x;
          all.y += c.y;
        }
      }
      upto = all.x + all.y;
    }
    #pragma unroll
    for(int offset = 1; offset < 32; offset *= 2) {
      int y = __shfl_up_sync(0xffffffffu, upto, offset);
      if(lane >= offset) upto += y;
    }
    if(31 == lane) shared.warp_sums[warp] = upto;
    __syncthreads();
    if(tid * 2 < digits) {
      for(int w = 0; w < warp; ++w) upto += shared.warp_sums[w];
      shared.starts[2 * tid] = upto - all.x - all.y + before.x;
      shared.starts[2 * tid + 1] = upto - all.y + before.y;
    }
    __syncthreads();
    bool done = pass + 1 == passes;
    #pragma unroll
    for(int j = 0; j < vt; ++j) {
      if(j < rounds && first + j * 32 + lane < count) {
        uint32_t digit = keys[j] >> shift & (digits - 1);
        int to = shared.starts[digit] + shared.seen[warp][digit] + places[j];
        if(done) {
          keys_out[to] = keys[j];
          positions_out[to] = positions[j];
        } else {
          int r = to / per_cta;
          cluster.map_shared_rank(&shared, r)->pairs[to - r * per_cta] =
            (unsigned long long)(uint32_t)positions[j] << 32 | keys[j];
        }
      }
    }
    if(done) break;      // nothing is written to other CTAs any more
    cluster.sync();
    #pragma unroll
    for(int j = 0; j < vt; ++j) {
      int i = warp * per_warp + j * 32 + lane;
      if(j < rounds && rank * per_cta + i < count) {
        unsigned long long pair = shared.pairs[i];
        keys[j] = (uint32_t)pair;
        positions[j] = (int)(pair >> 32);
      }
    }
  }
}

template<int nt>
__global__ void __launch_bounds__(nt) embedding_clear_k(int* counters,
  int64_t n) {
  for(int64_t i = (int64_t)blockIdx.x * nt + threadIdx.x; i < n;
    i += (int64_t)gridDim.x * nt) counters[i] = 0;
}

////////////////////////////////////////////////////////////////////////////////
// Sums.

enum { embedding_most_tile = 256, embedding_nt = 128, embedding_depth = 8,
  embedding_fan = 16, embedding_zero_ctas = 444,
  embedding_zero_rows = 8192, embedding_zero_bytes = 4096 };

// Tokens of either width, for a kernel that reads them in one place only.
struct any_tokens_t {
  const void* tokens;
  int wide, rows;
};

// Rows without a token. CTA b of `ctas` owns the rows b, b + ctas, ... (tokens
// crowd at low numbers), marks those among them that the tokens name in a
// bitmap, and zeroes the others, where rows are whole 16-byte words by the copy
// engine from a block of zeros.
template<int pack, typename out_t, typename token_t>
MGPU_DEVICE void embedding_zero(token_keys_t<token_t> source, int count,
  int width, uint32_t cta, uint32_t ctas, out_t* output, bool bulk,
  uint32_t* named, uint4* zeros) {
  typedef pack_t<out_t, pack> word_t;
  enum { ahead = 8 };
  const int nt = (int)blockDim.x;
  int64_t row_bytes = (int64_t)width * sizeof(out_t);
  int owned = (int)(((uint32_t)source.rows + ctas - 1 - cta) / ctas);
  for(int i = threadIdx.x; i < embedding_zero_bytes / 16; i += nt)
    zeros[i] = make_uint4(0, 0, 0, 0);
  ptx::fence_proxy_async();
  for(int base = 0; base < owned; base += embedding_zero_rows) {
    int here = min(owned - base, (int)embedding_zero_rows);
    for(int i = threadIdx.x; i < div_up(here, 32); i += nt) named[i] = 0;
    __syncthreads();
    for(int64_t first = threadIdx.x; first < count; first += ahead * nt) {
      uint32_t rows[ahead];
      #pragma unroll
      for(int i = 0; i < ahead; ++i)
        rows[i] = first + i * nt < count ? source.key((int)(first + i * nt)) :
          (uint32_t)source.rows;
      #pragma unroll
      for(int i = 0; i < ahead; ++i) {
        uint32_t place = rows[i] / ctas;
        int at = (int)place - base;
        if(rows[i] - place * ctas == cta && rows[i] < (uint32_t)source.rows &&
          at >= 0 && at < here) atomicOr(&named[at / 32], 1u << (at % 32));
      }
    }
    __syncthreads();
    if(bulk) {
      for(int i = threadIdx.x; i < here; i += nt) {
        if(named[i / 32] >> (i % 32) & 1) continue;
        char* to = (char*)(output + ((size_t)(base + i) * ctas + cta) * width);
        for(int64_t at = 0; at < row_bytes; at += embedding_zero_bytes)
          ptx::bulk_store(to + at, zeros,
            (uint32_t)min(row_bytes - at, (int64_t)embedding_zero_bytes));
      }
      ptx::bulk_commit();
    } else {
      word_t zero;
      #pragma unroll
      for(int j = 0; j < pack; ++j) zero.v[j] = from_f32<out_t>(0.0f);
      for(int i = (int)threadIdx.x / 32; i < here; i += nt / 32) {
        if(named[i / 32] >> (i % 32) & 1) continue;
        out_t* to = output + ((size_t)(base + i) * ctas + cta) * width;
        for(int c = (int)threadIdx.x % 32 * pack; c < width; c += 32 * pack)
          *(word_t*)(to + c) = zero;
      }
    }
    __syncthreads();
  }
  ptx::bulk_wait<0>();
}

// `pack` values of a row as words of up to 16 bytes.
template<typename out_t, int pack>
struct row_part_t {
  enum { piece = (int)sizeof(out_t) * pack > 16 ? 16 / (int)sizeof(out_t) :
    pack };
  pack_t<out_t, piece> words[pack / piece];
  MGPU_DEVICE out_t get(int j) const { return words[j / piece].v[j % piece]; }
  MGPU_DEVICE void set(int j, out_t x) { words[j / piece].v[j % piece] = x; }
};

// `old` is what the sums are added to.
template<bool accumulate, typename out_t, int pack>
MGPU_DEVICE __forceinline__ void store_row_part(out_t* to,
  const float (&sum)[pack], float scale, const row_part_t<out_t, pack>& old) {
  row_part_t<out_t, pack> part;
  #pragma unroll
  for(int j = 0; j < pack; ++j) {
    float v = sum[j] * scale;
    part.set(j, from_f32<out_t>(accumulate ? to_f32(old.get(j)) + v : v));
  }
  *(row_part_t<out_t, pack>*)to = part;
}

// One CTA per tile and slab of columns; every thread walks the tile's entries for
// its own columns with the running sum in registers. Bound by HBM: each row of
// grad is read once, and what is written most are the rows without a token (of
// 131,072 x 2,048 bf16 with 16,384 tokens 490 MB of 600). That call takes 116 us,
// 5.2 TB/s; pure stores reach about 5.5 TB/s on this GPU. Rows through registers
// instead of copies kept the SMs waiting (36 us instead of 24 us for the sums);
// 296 CTAs for the zeros instead of 444 cost 2 us, 148 cost 20 us; tiles of twice
// the length 10 us where tokens are few.
//
// parts holds two sums for each tile: of the run that was begun in an earlier
// tile (2 t), and of one that begins here and goes on (2 t + 1); behind them two
// for each 16 tiles, and so on, so that a token that fills the batch is added
// up in a few steps. counters, one for each sum and slab, start at 0.
//
// The first `zero_ctas` CTAs of a slab zero the rows without a token instead.
// They need nothing of the sort and run beside it; the others wait for it.
template<int pack, bool accumulate, typename real_t, typename out_t>
__global__ void __launch_bounds__(embedding_nt)
embedding_sum_k(const real_t* grad, int64_t stride, int width, int slab,
  any_tokens_t source, const uint32_t* keys, const int* positions, int count,
  int tile_size, float scale, out_t* output, float* parts, int* counters,
  int zero_ctas, int zero_bulk) {
  typedef pack_t<real_t, pack> word_t;
  typedef row_part_t<out_t, pack> out_part_t;
  typedef row_part_t<float, pack> part_t;
  // Rows on their way: each thread copies its own columns, `group` rows at a
  // time, and reads back only what it copied itself; with accumulate also the
  // row of the output, for the first entry of a run. Words of 2 bytes, which
  // cannot be copied so, go through registers.
  enum { group = 4, depth = embedding_depth, staged = sizeof(word_t) >= 4,
    staged_out = accumulate && staged && sizeof(out_part_t) >= 4 };
  extern __shared__ __align__(128) char memory[];
  const int nt = (int)blockDim.x, tid = (int)threadIdx.x;
  word_t* ring = (word_t*)memory + tid;
  out_part_t* out_ring = (out_part_t*)(memory + depth * nt * sizeof(word_t)) +
    tid;
  __shared__ uint32_t tile_keys[embedding_most_tile];
  __shared__ int tile_positions[embedding_most_tile];
  __shared__ int told, told_from, told_to;
  if((int)blockIdx.x < zero_ctas) {
    enum { words = pack * sizeof(out_t) > 16 ? 4 : pack };
    uint32_t* named = (uint32_t*)(memory + embedding_zero_bytes);
    if(!blockIdx.y) {
      if(source.wide)
        embedding_zero<words>(token_keys_t<int64_t> {
          (const int64_t*)source.tokens, source.rows }, count, width,
          blockIdx.x, (uint32_t)zero_ctas, output, 0 != zero_bulk, named,
          (uint4*)memory);
      else
        embedding_zero<words>(token_keys_t<int> { (const int*)source.tokens,
          source.rows }, count, width, blockIdx.x, (uint32_t)zero_ctas, output,
          0 != zero_bulk, named, (uint4*)memory);
    }
    return;
  }
  ptx::grid_dependency_wait();
  const int rows = source.rows;
  int tile = (int)blockIdx.x - zero_ctas;
  int begin = tile * tile_size, end = min(begin + tile_size, count);
  int entries = end - begin;
  for(int e = tid; e < entries; e += nt) {
    tile_keys[e] = keys[begin + e];
    // In range also where a scan of the sort has given up (status word).
    tile_positions[e] = (int)min((uint32_t)positions[begin + e],
      (uint32_t)count - 1);
  }
  uint32_t row = keys[begin];
  if(row >= (uint32_t)rows) return;
  bool carried = begin > 0 && keys[begin - 1] == row;
  uint32_t next = end < count ? keys[end] : (uint32_t)rows;
  __syncthreads();
  // Entries that name no row are the last ones of all.
  while(tile_keys[entries - 1] >= (uint32_t)rows) --entries;
  bool goes_on = tile_keys[entries - 1] == next;

  int column = ((int)blockIdx.y * slab + tid) * pack;
  bool live = tid < slab && column < width;
  float sum[pack];
  #pragma unroll
  for(int j = 0; j < pack; ++j) sum[j] = 0;
  auto keep_part = [&](int64_t slot) {
    if(!live) return;
    part_t part;
    #pragma unroll
    for(int j = 0; j < pack; ++j) part.set(j, sum[j]);
    *(part_t*)(parts + slot * width + column) = part;
  };
  // The first tile of the run begun earlier and the last one of the run that
  // goes on: each thread looks at the border of one tile in either direction,
  // while the rows are on their way.
  if(!tid) {
    told_from = -1;
    told_to = 0x7fffffff;
  }
  bool head = carried;
  auto from_row = [&](int e) {
    return (const word_t*)(grad + (int64_t)tile_positions[e] * stride + column);
  };
  auto out_row = [&](uint32_t r) {
    return (out_part_t*)(output + (size_t)r * width + column);
  };
  // Whether an entry begins a run of the tile that began in no earlier one.
  auto begins = [&](int e) {
    return e ? tile_keys[e] != tile_keys[e - 1] : !carried;
  };
  auto request = [&](int e) {
    if constexpr (staged) {
      #pragma unroll
      for(int i = 0; i < group; ++i)
        if(e + i < entries && live) {
          int place = (e + i) % depth * nt;
          ptx::cp_async<(int)sizeof(word_t)>(ring + place, from_row(e + i));
          if constexpr (staged_out)
            if(begins(e + i) && tile_keys[e + i] < (uint32_t)rows) {
              const out_part_t* from = out_row(tile_keys[e + i]);
              enum { size = sizeof(from->words[0]) };
              #pragma unroll
              for(int w = 0; w < (int)sizeof(out_part_t) / (int)size; ++w)
                ptx::cp_async<size>(&out_ring[place].words[w],
                  &from->words[w]);
            }
        }
      ptx::cp_async_commit();
    }
  };
  #pragma unroll
  for(int e = 0; e < depth; e += group) request(e);
  __syncthreads();
  // Is border b (the first entry of tile b) outside of the run?
  auto before_run = [&](int b, uint32_t key) {
    return b <= 0 || keys[(size_t)b * tile_size - 1] != key;
  };
  auto behind_run = [&](int64_t b, uint32_t key) {
    return b * tile_size >= count || keys[b * tile_size] != key;
  };
  if(carried && before_run(tile - tid, tile_keys[0]))
    atomicMax(&told_from, max(tile - tid, 0));
  if(goes_on && behind_run((int64_t)tile + 1 + tid, next))
    atomicMin(&told_to, tile + tid);
  out_part_t old;
  auto store = [&](uint32_t r) {
    if(r >= (uint32_t)rows) return;
    if constexpr (accumulate && !staged_out) old = *out_row(r);
    store_row_part<accumulate>((out_t*)out_row(r), sum, scale, old);
  };
  for(int e = 0; e < entries; e += group) {
    word_t words[group];
    if constexpr (staged) ptx::cp_async_wait<depth / group - 1>();
    #pragma unroll
    for(int i = 0; i < group; ++i)
      if(e + i < entries && live)
        words[i] = staged ? ring[(e + i) % depth * nt] : *from_row(e + i);
    #pragma unroll
    for(int i = 0; i < group; ++i) {
      if(e + i < entries) {
        uint32_t key = tile_keys[e + i];
        if(key != row) {
          if(head) keep_part(2 * (int64_t)tile);
          else if(live) store(row);
          head = false;
          row = key;
          #pragma unroll
          for(int j = 0; j < pack; ++j) sum[j] = 0;
        }
        if constexpr (staged_out)
          if(live && begins(e + i)) old = out_ring[(e + i) % depth * nt];
        #pragma unroll
        for(int j = 0; j < pack; ++j) sum[j] += to_f32(words[i].v[j]);
      }
    }
    request(e + depth);
  }
  if(head || goes_on) keep_part(2 * (int64_t)tile + (head ? 0 : 1));
  else if(live) store(row);

  // The runs that cross tiles: the one begun earlier, and the one that goes on
  // (they are the same one where it fills the tile: `head` is still set).
  if(!carried && !goes_on) return;
  __syncthreads();
  for(int which = 0; which < 2; ++which) {
    if(which ? !(goes_on && !head) : !carried) continue;
    uint32_t key = which ? row : tile_keys[0];
    int from = which ? tile : told_from;
    int to = which || head ? (goes_on ? told_to : tile) : tile;
    // Runs longer than the threads could see.
    for(int b = tile - nt; from < 0; b -= nt) {
      if(before_run(b - tid, key)) atomicMax(&told_from, max(b - tid, 0));
      __syncthreads();
      from = told_from;
      __syncthreads();
    }
    for(int64_t b = (int64_t)tile + 1 + nt; to == 0x7fffffff; b += nt) {
      if(behind_run(b + tid, key)) atomicMin(&told_to, (int)(b + tid) - 1);
      __syncthreads();
      to = told_to;
      __syncthreads();
    }
    // This CTA's sum is stored. Of each 16 neighbouring tiles the last one of
    // the run to say so adds up theirs, of 16 such sums the last one again.
    enum { fan = embedding_fan };
    int node = tile, nodes = (int)gridDim.x - zero_ctas;
    int64_t base = 0;
    while(true) {
      int low = max(from, node & ~(fan - 1)), high = min(to, node | (fan - 1));
      int64_t slot = base + 2 * (int64_t)low + (low == from);
      if(low < high) {
        __syncthreads();
        if(!tid) {
          __threadfence();
          told = atomicAdd(counters + slot * gridDim.y + blockIdx.y, 1);
          __threadfence();
        }
        __syncthreads();
        bool last = told == high - low;
        __syncthreads();
        if(!last) break;
      }
      float total[pack];
      #pragma unroll
      for(int j = 0; j < pack; ++j) total[j] = 0;
      if(live)
        for(int t = low; t <= high; t += group) {
          part_t some[group];
          #pragma unroll
          for(int i = 0; i < group; ++i)
            if(t + i <= high)
              some[i] = *(const part_t*)(parts + (base +
                2 * (int64_t)(t + i) + (t + i == from)) * width + column);
          #pragma unroll
          for(int i = 0; i < group; ++i)
            if(t + i <= high) {
              #pragma unroll
              for(int j = 0; j < pack; ++j) total[j] += some[i].get(j);
            }
        }
      if(low == from && high == to) {
        if(live) {
          if(accumulate) old = *out_row(key);
          store_row_part<accumulate>((out_t*)out_row(key), total, scale, old);
        }
        break;
      }
      base += 2 * (int64_t)nodes;
      nodes = div_up(nodes, (int)fan);
      node /= fan;
      from /= fan;
      to /= fan;
      #pragma unroll
      for(int j = 0; j < pack; ++j) sum[j] = total[j];
      keep_part(base + 2 * (int64_t)node + (node == from));
    }
  }
}

// Sizes and scratch of a call: a header with the status word that every
// workspace has (the scan's, where one runs; else 0), the counters behind it,
// the sorted pairs (two sets and the digit counts where one cluster does not take
// them) and the partial sums.
enum { embedding_header = 32 };              // words
struct embedding_plan_t {
  int tile_size, tiles, vt, ctas, sort_tiles;
  int64_t sums;
  size_t keys[2], positions[2], counts, scan, parts, counters, bytes;

  embedding_plan_t(int count, int rows, int width) {
    // About eight tiles for each SM; fewer entries than 8 in a tile would make
    // partial sums a third of the traffic.
    tile_size = 8;
    while(tile_size < embedding_most_tile &&
      (int64_t)tile_size * 1184 < (int64_t)count * div_up(width, 1024))
      tile_size *= 2;
    tiles = div_up(count, tile_size);
    sums = 0;
    for(int nodes = tiles; nodes;
      nodes = nodes > 1 ? div_up(nodes, (int)embedding_fan) : 0)
      sums += 2 * nodes;
    vt = count <= 8 * token_cluster_nt * token_cluster_most ? 8 : 32;
    ctas = 0;
    if(count <= vt * token_cluster_nt * token_cluster_most) {
      ctas = 1;
      while(ctas < token_cluster_most && ctas * 512 < count) ctas *= 2;
    }
    sort_tiles = ctas ? 0 : div_up(count, (int)token_sort_nv);
    size_t at = 0;
    auto take = [&](size_t n) {
      size_t here = at;
      at += (n + 127) / 128 * 128;
      return here;
    };
    int cells = sort_tiles * token_digits;
    scan = take(ctas ? 4 * embedding_header : scan_workspace_bytes<
      typename scan_default_tuning<int>::type, int>(cells));
    // A slab has about embedding_nt columns at least.
    counters = take(4 * (size_t)sums * div_up(width, (int)embedding_nt));
    for(int i = 0; i < (ctas ? 1 : 2); ++i) {
      keys[i] = take(4 * (size_t)count);
      positions[i] = take(4 * (size_t)count);
    }
    if(ctas) {
      keys[1] = keys[0];
      positions[1] = positions[0];
    }
    counts = take(4 * (size_t)cells);
    parts = take(4 * (size_t)sums * width);
    bytes = at;
  }
};

// A launch that may begin while its predecessor in the stream still runs.
template<typename... params_t, typename... args_t>
void launch_beside(void (*kernel)(params_t...), dim3 grid, int nt, size_t smem,
  cudaStream_t stream, bool beside, args_t... args) {
  cudaLaunchConfig_t config = { };
  config.gridDim = grid;
  config.blockDim = dim3((unsigned)nt);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = beside ? 1 : 0;
  throw_on_error(cudaLaunchKernelEx(&config, kernel, params_t(args)...));
}

template<int vt, typename token_t>
void token_cluster_sort(const embedding_plan_t& plan,
  token_keys_t<token_t> source, int count, uint32_t* keys, int* positions,
  int* counters, int64_t num_counters, cudaStream_t stream) {
  auto kernel = token_cluster_sort_k<vt, token_t>;
  const int smem = (int)sizeof(token_cluster_shared_t<vt>);
  set_dynamic_smem<token_cluster_shared_t<vt>, token_t>(kernel, smem);
  cudaLaunchConfig_t config = { };
  config.gridDim = dim3((unsigned)plan.ctas);
  config.blockDim = dim3(token_cluster_nt);
  config.dynamicSmemBytes = (size_t)smem;
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = (unsigned)plan.ctas;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  int bits = token_bits(source.rows);
  throw_on_error(cudaLaunchKernelEx(&config, kernel, source, count, bits,
    div_up(bits, (int)token_digit_bits), plan.ctas, keys, positions, counters,
    num_counters));
}

template<typename real_t, typename out_t, typename token_t>
void embedding_gradient_enqueue(const real_t* grad, int64_t stride, int width,
  const token_t* tokens, int count, int rows, float scale, bool accumulate,
  out_t* output, void* workspace, cudaStream_t stream) {
  if(!rows || !width || (accumulate && !count)) return;
  embedding_plan_t plan(count, rows, width);
  char* base = (char*)workspace;
  uint32_t* keys[2] = { (uint32_t*)(base + plan.keys[0]),
    (uint32_t*)(base + plan.keys[1]) };
  int* positions[2] = { (int*)(base + plan.positions[0]),
    (int*)(base + plan.positions[1]) };
  float* parts = (float*)(base + plan.parts);
  int* counters = (int*)(base + plan.counters);
  int out_pack = pack_limit(output, width, width, (int)sizeof(out_t));
  bool bulk = 16 / (int)sizeof(out_t) == out_pack;
  // A pack of 8 columns is stored as two words where the sums are 32 bits wide.
  if(bulk) out_pack = 8;
  int pack = min(pack_limit(grad, stride, width, (int)sizeof(real_t)), out_pack);
  // Slabs of equal width, in packs, and the warps they take.
  int packs = div_up(width, pack);
  int slabs = div_up(packs, (int)embedding_nt), slab = div_up(packs, slabs);
  int nt = div_up(slab, 32) * 32;
  int64_t num_counters = plan.sums * slabs;
  token_keys_t<token_t> source { tokens, rows };

  int into = 0;
  if(!count)
    embedding_clear_k<256><<<1, 256, 0, stream>>>((int*)base, embedding_header);
  if(count && plan.ctas) {
    if(8 == plan.vt)
      token_cluster_sort<8>(plan, source, count, keys[0], positions[0],
        (int*)base, embedding_header + num_counters, stream);
    else
      token_cluster_sort<32>(plan, source, count, keys[0], positions[0],
        (int*)base, embedding_header + num_counters, stream);
  } else if(count) {
    typedef scan_route_t<empty_t, int, int*, int*> route_t;
    int* counts = (int*)(base + plan.counts);
    auto pass = [&](auto from, int shift, int to) {
      token_count_k<<<plan.sort_tiles, token_sort_nt, 0, stream>>>(from,
        count, shift, plan.sort_tiles, counts);
      scan_dispatch<route_t, scan_type_exc, int>(counts,
        plan.sort_tiles * token_digits, counts, plus_t<int>(),
        discard_iterator_t<int>(), base + plan.scan, stream);
      token_scatter_k<<<plan.sort_tiles, token_sort_nt, 0, stream>>>(from,
        count, shift, plan.sort_tiles, counts, keys[to], positions[to]);
    };
    embedding_clear_k<256><<<148, 256, 0, stream>>>(counters, num_counters);
    int passes = div_up(token_bits(rows), (int)token_digit_bits);
    pass(source, 0, 0);
    for(int p = 1; p < passes; ++p, into ^= 1)
      pass(sorted_keys_t { keys[into], positions[into] },
        p * token_digit_bits, into ^ 1);
    throw_on_error(cudaGetLastError());
  }
  int zero_ctas = accumulate ? 0 : min(rows, (int)embedding_zero_ctas);
  if(zero_ctas) nt = max(nt, 128);         // they work with whole CTAs
  any_tokens_t any { tokens, sizeof(token_t) == 8, rows };
  with_pack(pack, [&](auto tag) {
    enum { vt = sizeof(real_t) == 2 || (int)decltype(tag)::value < 8 ?
      (int)decltype(tag)::value : 4 };
    auto launch = [&](auto kernel, auto adds, size_t smem) {
      // Beyond 48 KB with the shared variables of fixed size.
      if(smem > (40u << 10))
        set_dynamic_smem<decltype(tag), decltype(adds), real_t, out_t>(kernel,
          embedding_depth * embedding_nt * 48);
      dim3 grid((unsigned)(plan.tiles + zero_ctas), (unsigned)slabs);
      // Beside the sort, which was launched behind everything before it; without
      // one this kernel may begin no earlier than any other.
      launch_beside(kernel, grid, nt, smem, stream, 0 != count, grad, stride,
        width, slab, any, keys[into], positions[into], count, plan.tile_size,
        scale, output, parts, counters, zero_ctas, (int)bulk);
    };
    size_t smem = (size_t)embedding_depth * nt * vt * sizeof(real_t);
    if(accumulate)
      launch(embedding_sum_k<vt, true, real_t, out_t>, std::true_type(), smem +
        (size_t)embedding_depth * nt * vt * sizeof(out_t));
    else
      launch(embedding_sum_k<vt, false, real_t, out_t>, std::false_type(), max(smem,
        (size_t)embedding_zero_rows / 8 + embedding_zero_bytes));
  });
  throw_on_error(cudaGetLastError());
}

} // namespace detail

////////////////////////////////////////////////////////////////////////////////
// Public entry points. real_t and out_t are float, __half or __nv_bfloat16,
// token_t is int or int64_t. Rows of table and grad are `stride` elements
// apart, those of the outputs are dense.

template<typename real_t, typename token_t>
void embedding_lookup(const real_t* table, int rows, int width, int64_t stride,
  const token_t* tokens, int count, float scale, real_t* output,
  context_t& context) {
  static_assert(detail::is_model_real<real_t>::value,
    "embedding_lookup takes float, __half or __nv_bfloat16");
  detail::throw_on_device_status();
  detail::embedding_lookup_enqueue(table, rows, width, stride, tokens, count,
    scale, output, context.stream());
}

// With `accumulate` the sums are added to the output, and rows that no token
// names are neither read nor written; without it such rows become zero.
template<typename real_t, typename token_t, typename out_t>
void embedding_gradient(const real_t* grad, int64_t stride, int width,
  const token_t* tokens, int count, int rows, float scale, bool accumulate,
  out_t* output, context_t& context) {
  static_assert(detail::is_model_real<real_t>::value &&
    detail::is_model_real<out_t>::value,
    "embedding_gradient takes float, __half or __nv_bfloat16");
  detail::throw_on_device_status();
  mem_t<char> workspace(detail::embedding_plan_t(count, rows, width).bytes,
    context);
  detail::embedding_gradient_enqueue(grad, stride, width, tokens, count, rows,
    scale, accumulate, output, workspace.data(), context.stream());
}

#endif // __CUDACC__

END_MGPU_NAMESPACE
