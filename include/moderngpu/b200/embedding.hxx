// Embedding rows by token, and the gradient of the table they come from.
//
//   lookup:    output[i] = scale * table[tokens[i]]
//   gradient:  output[r] = scale * sum of grad[i] over the i with tokens[i] = r
//
// The lookup is interval_gather with whole rows for elements. The gradient is
// a segmented reduction with whole rows for items: the positions are sorted by
// token (stable, so that equal tokens keep the order of their positions), each
// row of the table is a segment of the sorted positions, and a row that no
// token names is an empty segment. The work of both is cut as segreduce cuts
// it, by merge path over the sorted positions and the ends of the rows, so a
// token that fills half of the batch and a hundred thousand rows without a
// token cost every CTA the same.
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
// `rows` and end up behind all others.

enum { token_sort_nt = 256, token_sort_vt = 16,
  token_sort_nv = token_sort_nt * token_sort_vt, token_digit_bits = 9,
  token_digits = 1 << token_digit_bits };

inline int token_sort_passes(int rows) {
  int bits = 0;
  while(bits < 32 && ((uint64_t)rows >> bits)) ++bits;   // keys 0 .. rows
  return bits ? div_up(bits, (int)token_digit_bits) : 1;
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

////////////////////////////////////////////////////////////////////////////////
// Gradient.

// Where a tile starts: `entry` sorted positions and `row` rows are before it.
struct MGPU_ALIGN(8) embedding_cut_t { int entry, row; };

enum { embedding_tile = 64 };

// Tile t holds the elements [64 t, 64 t + 64) of the merge of the sorted keys
// with the ends of the rows 0, 1, ..., rows - 1 (the end of a row comes after
// its entries). keys[e] + e rises strictly, so the entries in front of the
// merged place d are those with keys[e] + e < d: one binary search for a tile.
// With `accumulate` rows without entries have nothing to write, and tiles are
// 64 entries each.
template<int nt>
__global__ void __launch_bounds__(nt)
embedding_cuts_k(const uint32_t* keys, int count, int rows, int accumulate,
  int tiles, embedding_cut_t* cuts) {
  int t = (int)(blockIdx.x * nt + threadIdx.x);
  if(t > tiles) return;
  int64_t place = (int64_t)t * embedding_tile;
  int lo = 0, hi = count;
  if(accumulate) {
    // Entries with a row of the table.
    while(lo < hi) {
      int mid = (int)(((int64_t)lo + hi) / 2);
      if(keys[mid] < (uint32_t)rows) lo = mid + 1; else hi = mid;
    }
    int entry = place < lo ? (int)place : lo;
    cuts[t] = embedding_cut_t { entry, entry < lo ? (int)keys[entry] : rows };
  } else {
    while(lo < hi) {
      int mid = (int)(((int64_t)lo + hi) / 2);
      if((int64_t)keys[mid] + mid < place && keys[mid] < (uint32_t)rows)
        lo = mid + 1;
      else
        hi = mid;
    }
    int64_t row = place - lo;
    cuts[t] = embedding_cut_t { lo, row < rows ? (int)row : rows };
  }
}

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

// One CTA per tile and slab of nt * pack columns; every thread walks the
// tile's entries for its own columns with the running sum in registers. A row
// that began in an earlier tile, and one that goes on in a later tile, leaves
// its sum in `head` and `tail` for embedding_join_k.
template<int nt, int pack, typename real_t, typename out_t>
__global__ void __launch_bounds__(nt)
embedding_sum_k(const real_t* grad, int64_t stride, int width,
  const uint32_t* keys, const int* positions, const embedding_cut_t* cuts,
  float scale, int accumulate, out_t* output, float* head, float* tail) {
  typedef pack_t<real_t, pack> word_t;
  __shared__ uint32_t tile_keys[embedding_tile];
  __shared__ int tile_positions[embedding_tile];
  __shared__ int carried;
  int tile = (int)blockIdx.x;
  embedding_cut_t from = cuts[tile], to = cuts[tile + 1];
  int entries = to.entry - from.entry;
  for(int e = threadIdx.x; e < entries; e += nt) {
    tile_keys[e] = keys[from.entry + e];
    tile_positions[e] = positions[from.entry + e];
  }
  if(!threadIdx.x)
    carried = from.entry > 0 && from.row < to.row &&
      keys[from.entry - 1] == (uint32_t)from.row;
  __syncthreads();
  int column = (int)(blockIdx.y * nt + threadIdx.x) * pack;
  if(column >= width) return;

  float sum[pack], zero[pack];
  #pragma unroll
  for(int j = 0; j < pack; ++j) sum[j] = zero[j] = 0;
  int row = from.row;
  bool first = carried, some = false;
  auto finish = [&]() {
    if(first) {
      #pragma unroll
      for(int j = 0; j < pack; ++j)
        head[(size_t)tile * width + column + j] = sum[j];
    } else if(some || !accumulate)
      store_row_part<out_t, pack>(output + (size_t)row * width + column, sum,
        scale, 0 != accumulate);
    first = some = false;
    #pragma unroll
    for(int j = 0; j < pack; ++j) sum[j] = 0;
  };
  auto skip_to = [&](int next) {
    if(!accumulate)
      for(int r = row + 1; r < next; ++r)
        store_row_part<out_t, pack>(output + (size_t)r * width + column, zero,
          scale, false);
    row = next;
  };
  for(int e = 0; e < entries; ++e) {
    int key = (int)tile_keys[e];
    if(key != row) {
      finish();
      skip_to(key);
    }
    word_t word = *(const word_t*)(grad + (int64_t)tile_positions[e] * stride +
      column);
    some = true;
    #pragma unroll
    for(int j = 0; j < pack; ++j) sum[j] += to_f32(word.v[j]);
  }
  if(row < to.row) {
    finish();
    skip_to(to.row);
  } else if(some) {
    #pragma unroll
    for(int j = 0; j < pack; ++j)
      tail[(size_t)tile * width + column + j] = sum[j];
  }
}

// The first row that ends in a tile, where it began in an earlier one: the
// sums of the tiles before it, in order, and its own.
template<int nt, typename out_t>
__global__ void __launch_bounds__(nt)
embedding_join_k(int width, const uint32_t* keys, const embedding_cut_t* cuts,
  float scale, int accumulate, out_t* output, const float* head,
  const float* tail) {
  int tile = (int)blockIdx.x;
  embedding_cut_t from = cuts[tile], to = cuts[tile + 1];
  if(!(from.entry > 0 && from.row < to.row &&
    keys[from.entry - 1] == (uint32_t)from.row)) return;
  // The earliest tile that holds an entry of the row: tiles between it and
  // this one hold nothing else.
  int lo = 0, hi = from.entry;
  while(lo < hi) {
    int mid = (int)(((int64_t)lo + hi) / 2);
    if(keys[mid] < (uint32_t)from.row) lo = mid + 1; else hi = mid;
  }
  int begin = tile - 1;
  int a = 0, b = tile;              // last cut with entry <= lo
  while(a < b) {
    int mid = (int)(((int64_t)a + b) / 2);
    if(cuts[mid + 1].entry <= lo) a = mid + 1; else b = mid;
  }
  begin = a;
  for(int c = blockIdx.y * nt + threadIdx.x; c < width; c += gridDim.y * nt) {
    float sum = 0;
    for(int t = begin; t < tile; ++t) sum += tail[(size_t)t * width + c];
    sum += head[(size_t)tile * width + c];
    float part[1] = { sum };
    store_row_part<out_t, 1>(output + (size_t)from.row * width + c, part, scale,
      0 != accumulate);
  }
}

// Scratch: the pairs of two passes, the digit counts with the scan's own
// scratch, the tiles' cuts and the sums of rows that cross tiles.
struct embedding_plan_t {
  int tiles, sort_tiles, passes;
  size_t keys[2], positions[2], counts, scan, cuts, head, tail, bytes;

  embedding_plan_t(int count, int rows, int width, bool accumulate) {
    int64_t merged = accumulate ? (int64_t)count : (int64_t)count + rows;
    tiles = (int)div_up(merged, (int64_t)embedding_tile);
    sort_tiles = (int)div_up((int64_t)count, (int64_t)token_sort_nv);
    passes = token_sort_passes(rows);
    size_t at = 0;
    auto take = [&](size_t n) {
      size_t here = at;
      at += (n + 127) / 128 * 128;
      return here;
    };
    for(int i = 0; i < 2; ++i) {
      keys[i] = take(4 * (size_t)count);
      positions[i] = take(4 * (size_t)count);
    }
    int cells = sort_tiles * token_digits;
    counts = take(4 * (size_t)cells);
    scan = take(scan_workspace_bytes<typename scan_default_tuning<int>::type,
      int>(cells));
    cuts = take(sizeof(embedding_cut_t) * ((size_t)tiles + 1));
    head = take(4 * (size_t)tiles * width);
    tail = take(4 * (size_t)tiles * width);
    bytes = at;
  }
};

template<typename real_t, typename out_t, typename token_t>
void embedding_gradient_enqueue(const real_t* grad, int64_t stride, int width,
  const token_t* tokens, int count, int rows, float scale, bool accumulate,
  out_t* output, void* workspace, cudaStream_t stream) {
  if(!rows || !width || (accumulate && !count)) return;
  embedding_plan_t plan(count, rows, width, accumulate);
  char* base = (char*)workspace;
  uint32_t* keys[2] = { (uint32_t*)(base + plan.keys[0]),
    (uint32_t*)(base + plan.keys[1]) };
  int* positions[2] = { (int*)(base + plan.positions[0]),
    (int*)(base + plan.positions[1]) };
  int* counts = (int*)(base + plan.counts);
  embedding_cut_t* cuts = (embedding_cut_t*)(base + plan.cuts);
  float* head = (float*)(base + plan.head);
  float* tail = (float*)(base + plan.tail);

  int into = 0;
  if(count) {
    typedef scan_route_t<empty_t, int, int*, int*> route_t;
    auto pass = [&](auto source, int shift, int to) {
      token_count_k<<<plan.sort_tiles, token_sort_nt, 0, stream>>>(source,
        count, shift, plan.sort_tiles, counts);
      scan_dispatch<route_t, scan_type_exc, int>(counts,
        plan.sort_tiles * token_digits, counts, plus_t<int>(),
        discard_iterator_t<int>(), base + plan.scan, stream);
      token_scatter_k<<<plan.sort_tiles, token_sort_nt, 0, stream>>>(source,
        count, shift, plan.sort_tiles, counts, keys[to], positions[to]);
    };
    pass(token_keys_t<token_t> { tokens, rows }, 0, 0);
    for(int p = 1; p < plan.passes; ++p, into ^= 1)
      pass(sorted_keys_t { keys[into], positions[into] },
        p * token_digit_bits, into ^ 1);
  }
  embedding_cuts_k<256><<<div_up(plan.tiles + 1, 256), 256, 0, stream>>>(
    keys[into], count, rows, accumulate, plan.tiles, cuts);
  // A pack of 8 columns is stored as two words where the sums are 32 bits wide.
  int out_pack = pack_limit(output, width, width, (int)sizeof(out_t));
  if(16 / (int)sizeof(out_t) == out_pack) out_pack = 8;
  int pack = min(pack_limit(grad, stride, width, (int)sizeof(real_t)),
    out_pack);
  auto launch = [&](auto tag) {
    enum { nt = 128 };
    enum { vt = decltype(tag)::value };
    dim3 grid((unsigned)plan.tiles, (unsigned)div_up(width, nt * vt));
    embedding_sum_k<nt, vt, real_t, out_t><<<grid, nt, 0, stream>>>(grad,
      stride, width, keys[into], positions[into], cuts, scale, accumulate,
      output, head, tail);
  };
  switch(pack) {
    case 8: launch(std::integral_constant<int,
      (sizeof(real_t) == 2 ? 8 : 4)>()); break;
    case 4: launch(std::integral_constant<int, 4>()); break;
    case 2: launch(std::integral_constant<int, 2>()); break;
    default: launch(std::integral_constant<int, 1>()); break;
  }
  embedding_join_k<256, out_t><<<dim3((unsigned)plan.tiles,
    (unsigned)min(div_up(width, 256), 64)), 256, 0, stream>>>(width, keys[into],
    cuts, scale, accumulate, output, head, tail);
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
  mem_t<char> workspace(detail::embedding_plan_t(count, rows, width,
    accumulate).bytes, context);
  detail::embedding_gradient_enqueue(grad, stride, width, tokens, count, rows,
    scale, accumulate, output, workspace.data(), context.stream());
}

#endif // __CUDACC__

END_MGPU_NAMESPACE
