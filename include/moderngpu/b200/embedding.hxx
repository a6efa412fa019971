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
// does not idle most of a CTA; each moves packs of up to 16 bytes.
template<int nt, int pack, typename real_t, typename token_t>
__global__ void __launch_bounds__(nt)
embedding_lookup_k(const real_t* table, int64_t rows, int width,
  int64_t stride, const token_t* tokens, int64_t count, float scale,
  real_t* output, int lanes) {
  typedef pack_t<real_t, pack> word_t;
  int lane = (int)threadIdx.x & (lanes - 1);
  int per_cta = nt / lanes;
  int64_t i = (int64_t)blockIdx.x * per_cta + (int)threadIdx.x / lanes;
  if(i >= count) return;
  int64_t row = (int64_t)tokens[i];
  bool found = row >= 0 && row < rows;
  const real_t* from = table + (found ? row : 0) * stride;
  real_t* to = output + i * width;
  for(int c = lane * pack; c < width; c += lanes * pack) {
    word_t word;
    if(found) word = *(const word_t*)(from + c);
    #pragma unroll
    for(int j = 0; j < pack; ++j)
      word.v[j] = found ? from_f32<real_t>(to_f32(word.v[j]) * scale) :
        from_f32<real_t>(0.0f);
    *(word_t*)(to + c) = word;
  }
}

template<typename real_t, typename token_t>
void embedding_lookup_enqueue(const real_t* table, int64_t rows, int width,
  int64_t stride, const token_t* tokens, int64_t count, float scale,
  real_t* output, cudaStream_t stream) {
  if(!count || !width) return;
  enum { nt = 256 };
  int pack = min(pack_limit(table, stride, width, (int)sizeof(real_t)),
    pack_limit(output, width, width, (int)sizeof(real_t)));
  int lanes = 1;
  while(lanes < nt && lanes * pack < width) lanes *= 2;
  unsigned grid = (unsigned)div_up(count, (int64_t)(nt / lanes));
  auto launch = [&](auto tag) {
    embedding_lookup_k<nt, decltype(tag)::value, real_t, token_t>
      <<<grid, nt, 0, stream>>>(table, rows, width, stride, tokens, count,
        scale, output, lanes);
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
// time in order; lanes with equal digits find one another by a match vote, so
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
    int digit = live ? (int)((keys[j] >> shift) & (token_digits - 1)) :
      (int)token_digits;
    unsigned peers = __match_any_sync(0xffffffffu, digit);
    int ahead = __popc(peers & ((1u << lane) - 1));
    int before = live ? seen[warp][digit] : 0;
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
      keys_out[to] = keys[j];
      positions_out[to] = source.position((int)i);
    }
  }
}

// Each warp owns a run of neighbouring pairs, 32 at a time in order, and has
// them in registers between the passes. Lanes with equal digits find one another
// by a match vote; a pair's place is the number of pairs with a smaller digit,
// of the CTAs and warps before it with the same digit, and of its equals before
// it in its own warp.
enum { token_cluster_nt = 1024, token_cluster_most = 8 };

template<int vt>
struct token_cluster_shared_t {
  enum { warps = token_cluster_nt / 32, nv = token_cluster_nt * vt };
  uint32_t keys[nv];
  int positions[nv];
  uint16_t seen[warps][token_digits];
  int totals[token_digits];
  int starts[token_digits];
  int warp_sums[token_digits / 32];
};

template<int vt, typename token_t>
__global__ void __launch_bounds__(token_cluster_nt)
token_cluster_sort_k(token_keys_t<token_t> source, int count, int bits,
  int passes, int ctas, uint32_t* keys_out, int* positions_out, int* counters,
  int64_t num_counters) {
  enum { nt = token_cluster_nt, warps = nt / 32 };
  extern __shared__ __align__(16) char token_cluster_memory[];
  typedef token_cluster_shared_t<vt> shared_t;
  shared_t& shared = *(shared_t*)token_cluster_memory;
  auto cluster = cooperative_groups::this_cluster();
  // The kernel that follows zeroes the rows without a token meanwhile.
  ptx::grid_launch_dependents();

  int rank = (int)cluster.block_rank(), tid = (int)threadIdx.x;
  int warp = tid / 32, lane = tid % 32;
  int rounds = div_up(div_up(count, ctas * warps), 32);
  int per_warp = rounds * 32, per_cta = per_warp * warps;
  int first = rank * per_cta + warp * per_warp;
  for(int64_t i = rank * nt + tid; i < num_counters; i += ctas * nt)
    counters[i] = 0;

  uint32_t keys[vt];
  int positions[vt];
  #pragma unroll
  for(int j = 0; j < vt; ++j) {
    int i = first + j * 32 + lane;
    bool live = j < rounds && i < count;
    keys[j] = live ? source.key(i) : 0;
    positions[j] = i;
  }
  int digit_bits = div_up(bits, passes), digits = 1 << digit_bits;
  for(int pass = 0; pass < passes; ++pass) {
    int shift = pass * digit_bits;
    for(int d = tid; d < warps * token_digits / 2; d += nt)
      ((uint32_t*)shared.seen)[d] = 0;
    __syncthreads();
    int places[vt];
    #pragma unroll
    for(int j = 0; j < vt; ++j) {
      if(j < rounds) {
        bool live = first + j * 32 + lane < count;
        int digit = live ? (int)((keys[j] >> shift) & (digits - 1)) : digits;
        unsigned peers = __match_any_sync(0xffffffffu, digit);
        int ahead = __popc(peers & ((1u << lane) - 1));
        int before = live ? shared.seen[warp][digit] : 0;
        __syncwarp();
        if(live && !ahead)
          shared.seen[warp][digit] = (uint16_t)(before + __popc(peers));
        __syncwarp();
        places[j] = before + ahead;
      }
    }
    __syncthreads();
    // A thread for each digit: the warps' counts become places in the CTA.
    if(tid < digits) {
      int sum = 0;
      #pragma unroll 8
      for(int w = 0; w < warps; ++w) {
        int c = shared.seen[w][tid];
        shared.seen[w][tid] = (uint16_t)sum;
        sum += c;
      }
      shared.totals[tid] = sum;
    }
    cluster.sync();
    int before = 0, all = 0, upto = 0;
    if(tid < token_digits) {
      if(tid < digits)
        for(int r = 0; r < ctas; ++r) {
          int c = cluster.map_shared_rank(&shared, r)->totals[tid];
          if(r < rank) before += c;
          all += c;
        }
      upto = all;
      #pragma unroll
      for(int offset = 1; offset < 32; offset *= 2) {
        int y = __shfl_up_sync(0xffffffffu, upto, offset);
        if(lane >= offset) upto += y;
      }
      if(31 == lane) shared.warp_sums[warp] = upto;
    }
    __syncthreads();
    if(tid < digits) {
      for(int w = 0; w < warp; ++w) upto += shared.warp_sums[w];
      shared.starts[tid] = upto - all + before;
    }
    __syncthreads();
    bool done = pass + 1 == passes;
    #pragma unroll
    for(int j = 0; j < vt; ++j) {
      if(j < rounds && first + j * 32 + lane < count) {
        int digit = (int)((keys[j] >> shift) & (digits - 1));
        int to = shared.starts[digit] + shared.seen[warp][digit] + places[j];
        if(done) {
          keys_out[to] = keys[j];
          positions_out[to] = positions[j];
        } else {
          int r = to / per_cta;
          shared_t* there = cluster.map_shared_rank(&shared, r);
          there->keys[to - r * per_cta] = keys[j];
          there->positions[to - r * per_cta] = positions[j];
        }
      }
    }
    // Also: no CTA leaves, or counts again, while another reads its totals.
    cluster.sync();
    if(!done) {
      #pragma unroll
      for(int j = 0; j < vt; ++j) {
        int i = warp * per_warp + j * 32 + lane;
        if(j < rounds && rank * per_cta + i < count) {
          keys[j] = shared.keys[i];
          positions[j] = shared.positions[i];
        }
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
// Rows without a token. CTA b owns the rows b, b + gridDim.x, ... (tokens crowd
// at low numbers), marks those among them that the tokens name in a bitmap, and
// zeroes the others.

enum { embedding_zero_nt = 512, embedding_zero_rows = 32768 };

template<int pack, typename out_t, typename token_t>
__global__ void __launch_bounds__(embedding_zero_nt)
embedding_zero_k(token_keys_t<token_t> source, int count, int width, int lanes,
  out_t* output) {
  enum { nt = embedding_zero_nt };
  typedef pack_t<out_t, pack> word_t;
  __shared__ uint32_t named[embedding_zero_rows / 32];
  word_t zero;
  #pragma unroll
  for(int j = 0; j < pack; ++j) zero.v[j] = from_f32<out_t>(0.0f);
  uint32_t ctas = gridDim.x, cta = blockIdx.x;
  int owned = (int)(((uint32_t)source.rows + ctas - 1 - cta) / ctas);
  int lane = (int)threadIdx.x & (lanes - 1), group = (int)threadIdx.x / lanes;
  for(int base = 0; base < owned; base += embedding_zero_rows) {
    int here = min(owned - base, (int)embedding_zero_rows);
    for(int i = threadIdx.x; i < div_up(here, 32); i += nt) named[i] = 0;
    __syncthreads();
    #pragma unroll 4
    for(int64_t i = threadIdx.x; i < count; i += nt) {
      uint32_t row = source.key((int)i);
      uint32_t place = row / ctas;
      if(row - place * ctas == cta && row < (uint32_t)source.rows) {
        int at = (int)place - base;
        if(at >= 0 && at < here) atomicOr(&named[at / 32], 1u << (at % 32));
      }
    }
    __syncthreads();
    for(int i = group; i < here; i += nt / lanes) {
      if(named[i / 32] >> (i % 32) & 1) continue;
      out_t* to = output + ((size_t)(base + i) * ctas + cta) * width;
      for(int c = lane * pack; c < width; c += lanes * pack)
        *(word_t*)(to + c) = zero;
    }
    __syncthreads();
  }
  // Where this kernel runs beside the sort: the sums that follow need both.
  ptx::grid_dependency_wait();
}

////////////////////////////////////////////////////////////////////////////////
// Sums.

enum { embedding_most_tile = 256 };

template<typename out_t, int pack>
MGPU_DEVICE __forceinline__ void store_row_part(out_t* to,
  const float (&sum)[pack], float scale, bool accumulate) {
  enum { size = (int)sizeof(out_t) * pack,
    piece = size > 16 ? 16 / (int)sizeof(out_t) : pack };
  typedef pack_t<out_t, piece> word_t;
  #pragma unroll
  for(int p = 0; p < pack; p += piece) {
    word_t word;
    if(accumulate) word = *(const word_t*)(to + p);
    #pragma unroll
    for(int j = 0; j < piece; ++j) {
      float v = sum[p + j] * scale;
      word.v[j] = from_f32<out_t>(accumulate ? to_f32(word.v[j]) + v : v);
    }
    *(word_t*)(to + p) = word;
  }
}

// A partial sum, as words of up to 16 bytes.
template<int pack>
struct part_t {
  enum { piece = pack > 4 ? 4 : pack };
  pack_t<float, piece> words[pack / piece];
};

// One CTA per tile and slab of nt * pack columns; every thread walks the tile's
// entries for its own columns, `batch` rows in flight, with the running sum in
// registers. Bound by HBM: each row of grad is read once.
//
// parts holds two sums for each tile: of the run that was begun in an earlier
// tile (2 t), and of one that begins here and goes on (2 t + 1). counters, one
// for each tile and slab, start at 0 and count the sums of the run that begins
// in the tile.
template<int nt, int pack, typename real_t, typename out_t>
__global__ void __launch_bounds__(nt)
embedding_sum_k(const real_t* grad, int64_t stride, int width,
  const uint32_t* keys, const int* positions, int count, int rows, int tile_size,
  float scale, int accumulate, out_t* output, float* parts, int* counters) {
  typedef pack_t<real_t, pack> word_t;
  enum { batch = 8 };
  __shared__ uint32_t tile_keys[embedding_most_tile];
  __shared__ int tile_positions[embedding_most_tile];
  __shared__ int told;
  ptx::grid_dependency_wait();
  int tile = (int)blockIdx.x, tid = (int)threadIdx.x;
  int begin = tile * tile_size, end = min(begin + tile_size, count);
  int entries = end - begin;
  for(int e = tid; e < entries; e += nt) {
    tile_keys[e] = keys[begin + e];
    tile_positions[e] = positions[begin + e];
  }
  uint32_t row = keys[begin];
  if(row >= (uint32_t)rows) return;
  bool carried = begin > 0 && keys[begin - 1] == row;
  uint32_t next = end < count ? keys[end] : (uint32_t)rows;
  __syncthreads();
  // Entries that name no row are the last ones of all.
  while(tile_keys[entries - 1] >= (uint32_t)rows) --entries;
  bool goes_on = tile_keys[entries - 1] == next;

  int column = (int)(blockIdx.y * nt + tid) * pack;
  bool live = column < width;
  float sum[pack];
  #pragma unroll
  for(int j = 0; j < pack; ++j) sum[j] = 0;
  auto keep_part = [&](int slot) {
    if(!live) return;
    part_t<pack> part;
    #pragma unroll
    for(int j = 0; j < pack; ++j)
      part.words[j / part_t<pack>::piece].v[j % part_t<pack>::piece] = sum[j];
    *(part_t<pack>*)(parts + (size_t)slot * width + column) = part;
  };
  bool head = carried;
  for(int e = 0; e < entries; e += batch) {
    word_t words[batch];
    #pragma unroll
    for(int i = 0; i < batch; ++i)
      if(e + i < entries && live)
        words[i] = *(const word_t*)(grad +
          (int64_t)tile_positions[e + i] * stride + column);
    #pragma unroll
    for(int i = 0; i < batch; ++i) {
      if(e + i < entries) {
        uint32_t key = tile_keys[e + i];
        if(key != row) {
          if(head)
            keep_part(2 * tile);
          else if(live)
            store_row_part<out_t, pack>(output + (size_t)row * width + column,
              sum, scale, 0 != accumulate);
          head = false;
          row = key;
          #pragma unroll
          for(int j = 0; j < pack; ++j) sum[j] = 0;
        }
        #pragma unroll
        for(int j = 0; j < pack; ++j) sum[j] += to_f32(words[i].v[j]);
      }
    }
  }
  if(head || goes_on)
    keep_part(2 * tile + (head ? 0 : 1));
  else if(live)
    store_row_part<out_t, pack>(output + (size_t)row * width + column, sum,
      scale, 0 != accumulate);

  // The runs that cross tiles: the one begun earlier, and the one that goes on
  // (they are the same one where it fills the tile: `head` is still set).
  for(int which = 0; which < 2; ++which) {
    if(which ? !(goes_on && !head) : !carried) continue;
    uint32_t key = which ? row : tile_keys[0];
    // Its first and last tile: threads look at the tiles' borders.
    int from = tile, to = tile;
    if(!which) {
      bool found = false;
      for(int b = tile; !found; b -= nt) {
        int border = b - tid;
        bool out = border <= 0 || keys[(size_t)border * tile_size - 1] != key;
        if(!tid) told = -1;
        __syncthreads();
        if(out) atomicMax(&told, max(border, 0));
        __syncthreads();
        found = told >= 0;
        from = told;
        __syncthreads();
      }
    }
    if(which || head) {
      if(goes_on) {
        bool found = false;
        for(int b = tile + 1; !found; b += nt) {
          int64_t border = (int64_t)b + tid;
          bool out = border * tile_size >= count ||
            keys[border * tile_size] != key;
          if(!tid) told = 0x7fffffff;
          __syncthreads();
          if(out) atomicMin(&told, (int)border - 1);
          __syncthreads();
          found = told != 0x7fffffff;
          to = told;
          __syncthreads();
        }
      }
    }
    // This CTA's sum is stored; the last to say so adds up.
    __syncthreads();
    if(!tid) {
      __threadfence();
      told = atomicAdd(counters + (size_t)from * gridDim.y + blockIdx.y, 1);
      __threadfence();
    }
    __syncthreads();
    bool last = told == to - from;
    __syncthreads();
    if(!last || !live) continue;
    float total[pack];
    #pragma unroll
    for(int j = 0; j < pack; ++j) total[j] = 0;
    for(int t = from; t <= to; t += batch) {
      part_t<pack> some[batch];
      #pragma unroll
      for(int i = 0; i < batch; ++i)
        if(t + i <= to) {
          const part_t<pack>* at = (const part_t<pack>*)(parts +
            (size_t)(2 * (t + i) + (t + i == from)) * width + column);
          some[i] = *at;
        }
      #pragma unroll
      for(int i = 0; i < batch; ++i)
        if(t + i <= to) {
          #pragma unroll
          for(int j = 0; j < pack; ++j)
            total[j] += some[i].words[j / part_t<pack>::piece].v[
              j % part_t<pack>::piece];
        }
    }
    store_row_part<out_t, pack>(output + (size_t)key * width + column, total,
      scale, 0 != accumulate);
  }
}

// Sizes and scratch of a call: the sorted pairs (two sets and the digit counts
// with their scan where one cluster does not take them), the partial sums and
// their counters.
struct embedding_plan_t {
  int tile_size, tiles, slab_limit, vt, ctas, sort_tiles;
  size_t keys[2], positions[2], counts, scan, parts, counters, bytes;

  embedding_plan_t(int count, int rows, int width) {
    // About eight tiles for each SM; fewer entries than 8 in a tile would make
    // partial sums a third of the traffic.
    tile_size = 8;
    while(tile_size < embedding_most_tile &&
      (int64_t)tile_size * 1184 < count) tile_size *= 2;
    tiles = div_up(count, tile_size);
    slab_limit = div_up(width, 32);        // a slab has 32 columns at least
    vt = count <= 4 * token_cluster_nt * token_cluster_most ? 4 : 16;
    ctas = 0;
    if(count <= vt * token_cluster_nt * token_cluster_most) {
      ctas = 1;
      while(ctas < token_cluster_most && ctas * 2048 < count) ctas *= 2;
    }
    sort_tiles = ctas ? 0 : div_up(count, (int)token_sort_nv);
    size_t at = 0;
    auto take = [&](size_t n) {
      size_t here = at;
      at += (n + 127) / 128 * 128;
      return here;
    };
    for(int i = 0; i < (ctas ? 1 : 2); ++i) {
      keys[i] = take(4 * (size_t)count);
      positions[i] = take(4 * (size_t)count);
    }
    if(ctas) {
      keys[1] = keys[0];
      positions[1] = positions[0];
    }
    int cells = sort_tiles * token_digits;
    counts = take(4 * (size_t)cells);
    scan = take(ctas ? 0 : scan_workspace_bytes<
      typename scan_default_tuning<int>::type, int>(cells));
    parts = take(8 * (size_t)tiles * width);
    counters = take(4 * (size_t)tiles * slab_limit);
    bytes = at;
  }
};

// Launch that may begin while its predecessor in the stream still runs.
template<typename... params_t, typename... args_t>
void launch_beside(void (*kernel)(params_t...), dim3 grid, int nt,
  cudaStream_t stream, args_t... args) {
  cudaLaunchConfig_t config = { };
  config.gridDim = grid;
  config.blockDim = dim3((unsigned)nt);
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
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

// The widest pack for `width` columns on both sides, as a constant for f.
template<typename func_t>
void with_pack(int pack, func_t f) {
  switch(pack) {
    case 8: f(std::integral_constant<int, 8>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    case 2: f(std::integral_constant<int, 2>()); break;
    default: f(std::integral_constant<int, 1>()); break;
  }
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
  int64_t num_counters = (int64_t)plan.tiles * plan.slab_limit;
  token_keys_t<token_t> source { tokens, rows };

  int into = 0;
  if(count && plan.ctas) {
    if(4 == plan.vt)
      token_cluster_sort<4>(plan, source, count, keys[0], positions[0],
        counters, num_counters, stream);
    else
      token_cluster_sort<16>(plan, source, count, keys[0], positions[0],
        counters, num_counters, stream);
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
  int out_pack = pack_limit(output, width, width, (int)sizeof(out_t));
  if(!accumulate)
    with_pack(out_pack, [&](auto tag) {
      enum { vt = sizeof(out_t) == 2 || (int)decltype(tag)::value < 8 ?
        (int)decltype(tag)::value : 4 };
      int lanes = 1;
      while(lanes < embedding_zero_nt && lanes * vt < width) lanes *= 2;
      // Beside the sort, which was launched behind everything before it; without
      // one this kernel may begin no earlier than any other.
      dim3 grid((unsigned)min(rows, 296));
      if(count)
        launch_beside(embedding_zero_k<vt, out_t, token_t>, grid,
          embedding_zero_nt, stream, source, count, width, lanes, output);
      else
        embedding_zero_k<vt, out_t, token_t><<<grid, embedding_zero_nt, 0,
          stream>>>(source, count, width, lanes, output);
    });
  if(!count) return;
  // A pack of 8 columns is stored as two words where the sums are 32 bits wide.
  if(16 / (int)sizeof(out_t) == out_pack) out_pack = 8;
  with_pack(min(pack_limit(grad, stride, width, (int)sizeof(real_t)), out_pack),
    [&](auto tag) {
      enum { vt = sizeof(real_t) == 2 || (int)decltype(tag)::value < 8 ?
        (int)decltype(tag)::value : 4 };
      auto launch = [&](auto threads) {
        enum { nt = decltype(threads)::value };
        launch_beside(embedding_sum_k<nt, vt, real_t, out_t>,
          dim3((unsigned)plan.tiles, (unsigned)div_up(width, nt * vt)), nt,
          stream, grad, stride, width, keys[into], positions[into], count, rows,
          plan.tile_size, scale, (int)accumulate, output, parts, counters);
      };
      if(width <= 32 * vt) launch(std::integral_constant<int, 32>());
      else if(width <= 128 * vt) launch(std::integral_constant<int, 128>());
      else launch(std::integral_constant<int, 256>());
    });
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
