// embedding.cu — embedding lookup with scaling, and its gradient by sorted tokens, for sm_100a.
//
//   lookup:    out[t, :] = scale * table[token[t], :]
//   gradient:  grad_table[v, :] (= or +=) scale * sum over t with token[t] = v of grad_out[t, :]
//
// Both are bound by HBM bytes: the lookup reads every named row once (repeats come from L2) and writes out once; the
// gradient reads grad_out once and writes the table once (or reads and writes the named rows, when added).  Sums are
// fp32 and run in an order that the token positions alone fix, so the same call gives the same bits; no floating-point
// atomics.  The gradient's steps:
//
//   1. a stable radix sort of (token, position) — one CTA in shared memory for up to 4096 tokens, else a histogram and
//      a scatter launch per digit;
//   2. segmented sums over equal chunks of the sorted positions, which balances frequent tokens by construction: a run
//      of one token inside a chunk is written straight to its row, a run that crosses a chunk's border leaves an fp32
//      partial row in the workspace;
//   3. the partial rows of every crossing run are joined, in chunk order, and written;
//   4. without `accumulate`, rows that no token names are filled with zeros.
//
// Tokens outside [0, vocabulary) read as zeros (lookup) or contribute nothing (gradient) and are recorded in the device
// status word.  A padding token and out-of-range tokens sort behind every row under the key `vocabulary`.
#include "bb200_elementwise.cuh"
#include "bb200_internal.h"

namespace bb200 {
namespace {

constexpr int kThreads = 256;

// The row vectors of one step: VEC elements, widened.
template <typename T, int VEC> __device__ __forceinline__ void widen(const Pack<T, VEC>& in, float (&out)[VEC]) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) out[e] = Conv<float, T>::widen(in.v[e]);
}

// ---- lookup -------------------------------------------------------------------------------------------------------
// `1 << lane_bits` neighbouring threads share a row; each moves two vectors of it per pass over the columns, so 2048
// threads per SM keep 64 KB of loads in flight.
template <typename T, typename O, typename Id, int VEC>
__global__ void __launch_bounds__(kThreads)
lookup_rows(const Id* __restrict__ tokens, const T* __restrict__ table, O* __restrict__ out, size_t count, size_t vocabulary, int steps,
            int lane_bits, float scale, int* status_word) {
  dependent_launch_prologue();
  const int lanes = 1 << lane_bits, lane = threadIdx.x & (lanes - 1);
  const size_t row = (size_t)blockIdx.x * (kThreads >> lane_bits) + (threadIdx.x >> lane_bits);
  if (row >= count) return;
  const long long token = (long long)tokens[row];
  const bool inside = token >= 0 && (unsigned long long)token < vocabulary;
  if (!inside && lane == 0 && blockIdx.y == 0 && status_word) atomicExch(status_word, BB200_TOKEN_OUT_OF_RANGE);
  const T* __restrict__ source = table + (inside ? (size_t)token : 0) * ((size_t)steps * VEC);
  O* __restrict__ target = out + row * ((size_t)steps * VEC);
  for (int step = blockIdx.y * 2 * lanes + lane; step < steps; step += gridDim.y * 2 * lanes) {
    const int other = step + lanes;
    Pack<T, VEC> a, b;
    a = load_shared_operand<T, VEC>(source + (size_t)step * VEC);
    if (other < steps) b = load_shared_operand<T, VEC>(source + (size_t)other * VEC);
    Pack<O, VEC> r;
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.v[e] = Conv<float, O>::narrow(inside ? Conv<float, T>::widen(a.v[e]) * scale : 0.0f);
    store_stream<O, VEC>(target + (size_t)step * VEC, r);
    if (other < steps) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) r.v[e] = Conv<float, O>::narrow(inside ? Conv<float, T>::widen(b.v[e]) * scale : 0.0f);
      store_stream<O, VEC>(target + (size_t)other * VEC, r);
    }
  }
}

template <typename T, typename O, typename Id, int VEC>
int launch_lookup(const void* tokens, const void* table, void* out, size_t count, size_t vocabulary, size_t hidden, float scale,
                  cudaStream_t stream) {
  const int steps = (int)(hidden / VEC);
  int lane_bits = 2;
  while (lane_bits < 8 && (2 << lane_bits) < steps) ++lane_bits;
  const size_t rows_per_block = kThreads >> lane_bits;
  const size_t blocks = (count + rows_per_block - 1) / rows_per_block;
  const size_t columns = ((size_t)steps + (2u << lane_bits) - 1) >> (lane_bits + 1);
  launch_dependent(lookup_rows<T, O, Id, VEC>, dim3((unsigned)blocks, (unsigned)(columns < 65535 ? columns : 65535)), dim3(kThreads), 0, stream,
                   static_cast<const Id*>(tokens), static_cast<const T*>(table), static_cast<O*>(out), count, vocabulary, steps, lane_bits,
                   scale, device_status_word());
  return check_launch("embedding kernel launch");
}

// ---- sorting the tokens ---------------------------------------------------------------------------------------------
// Least-significant-digit radix sort of (token, position), stable, digits of at most 9 bits.  A CTA ranks a tile of
// 4096: warp w holds the tile's elements [256 w, 256 w + 256), 32 at a time in order; within 32 the rank among equal
// digits comes from __match_any_sync, earlier 32s of the warp are counted in the warp's own shared-memory counters,
// and earlier warps by a prefix over the sixteen counters of a digit.
constexpr int kSortThreads = 512, kSortRounds = 8, kSortWarps = kSortThreads / 32, kTile = kSortThreads * kSortRounds, kDigitBits = 9,
              kBins = 1 << kDigitBits;

template <typename Id> __device__ __forceinline__ uint32_t key_of(Id raw, uint32_t vocabulary, long long padding, int* status_word) {
  const long long token = (long long)raw;
  if (token < 0 || token >= (long long)vocabulary) {
    if (status_word) atomicExch(status_word, BB200_TOKEN_OUT_OF_RANGE);
    return vocabulary;
  }
  return token == padding ? vocabulary : (uint32_t)token;
}

// Stable rank of each of a thread's eight elements among the tile's elements of the same digit; on return counters[d]
// of warp 0 hold how many elements of the tile have digit d.  `counters`: [kSortWarps + 1][kBins].
__device__ __forceinline__ void rank_tile(const uint32_t (&digit)[kSortRounds], uint32_t (&rank)[kSortRounds], uint32_t* counters) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t* mine = counters + warp * kBins;
  for (int bin = lane; bin < kBins; bin += 32) mine[bin] = 0;
  __syncwarp();
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const uint32_t same = __match_any_sync(0xffffffffu, digit[r]);
    const uint32_t before = __popc(same & ((1u << lane) - 1));
    rank[r] = mine[digit[r]] + before;
    __syncwarp();
    if (before == 0) mine[digit[r]] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  uint32_t total = 0;  // one thread per digit: exclusive prefix over the warps
  if (threadIdx.x < kBins) {
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t n = counters[w * kBins + threadIdx.x];
      counters[w * kBins + threadIdx.x] = total;
      total += n;
    }
    counters[kSortWarps * kBins + threadIdx.x] = total;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) rank[r] += mine[digit[r]];
}

// Exclusive prefix sum over kBins values, one per thread (kBins == kSortThreads).
__device__ __forceinline__ uint32_t exclusive_over_bins(uint32_t value, uint32_t* warp_totals) {
  static_assert(kBins == kSortThreads, "one bin per thread");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t inclusive = value;
#pragma unroll
  for (int offset = 1; offset < 32; offset <<= 1) {
    const uint32_t below = __shfl_up_sync(0xffffffffu, inclusive, offset);
    if (lane >= offset) inclusive += below;
  }
  if (lane == 31) warp_totals[warp] = inclusive;
  __syncthreads();
  uint32_t base = 0;
  for (int w = 0; w < warp; ++w) base += warp_totals[w];
  __syncthreads();
  return base + inclusive - value;
}

// Up to kTile tokens in one CTA: all digits in shared memory, one launch.
template <typename Id>
__global__ void __launch_bounds__(kSortThreads)
sort_tokens_small(const Id* __restrict__ tokens, uint32_t count, uint32_t vocabulary, long long padding, int passes, int digit_bits,
                  uint32_t* __restrict__ keys_out, uint32_t* __restrict__ order_out, uint8_t* __restrict__ named, int* status_word) {
  extern __shared__ uint32_t shared[];
  uint32_t* keys = shared;
  uint32_t* order = keys + kTile;
  uint32_t* counters = order + kTile;  // [kSortWarps + 1][kBins]
  uint32_t* starts = counters + (kSortWarps + 1) * kBins;
  __shared__ uint32_t warp_totals[kSortWarps];
  dependent_launch_prologue();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t key[kSortRounds], position[kSortRounds];
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    position[r] = warp * (32 * kSortRounds) + r * 32 + lane;
    key[r] = position[r] < count ? key_of(tokens[position[r]], vocabulary, padding, status_word) : vocabulary;
    if (named && key[r] < vocabulary) named[key[r]] = 1;
  }
  for (int pass = 0; pass < passes; ++pass) {
    uint32_t digit[kSortRounds], rank[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) digit[r] = (key[r] >> (pass * digit_bits)) & (kBins - 1) & ((1u << digit_bits) - 1);
    rank_tile(digit, rank, counters);
    starts[threadIdx.x] = exclusive_over_bins(counters[kSortWarps * kBins + threadIdx.x], warp_totals);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      const uint32_t at = starts[digit[r]] + rank[r];
      keys[at] = key[r];
      order[at] = position[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      const uint32_t at = warp * (32 * kSortRounds) + r * 32 + lane;
      key[r] = keys[at];
      position[r] = order[at];
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {  // the fill beyond `count` carries the last key and the last positions: it sorted behind
    const uint32_t at = warp * (32 * kSortRounds) + r * 32 + lane;
    if (at < count) {
      keys_out[at] = key[r];
      order_out[at] = position[r];
    }
  }
}

// counts[tile][digit] of one digit.  The first pass reads the tokens themselves and marks the rows they name.
template <typename Id, bool FIRST>
__global__ void __launch_bounds__(kSortThreads)
count_digits(const Id* __restrict__ tokens, const uint32_t* __restrict__ keys, uint32_t count, uint32_t vocabulary, long long padding,
             int shift, uint32_t mask, uint32_t* __restrict__ counts, uint8_t* __restrict__ named, int* status_word) {
  __shared__ uint32_t local[kBins];
  dependent_launch_prologue();
  local[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const size_t at = (size_t)blockIdx.x * kTile + r * kSortThreads + threadIdx.x;
    if (at < count) {
      uint32_t key;
      if constexpr (FIRST) {
        key = key_of(tokens[at], vocabulary, padding, status_word);
        if (named && key < vocabulary) named[key] = 1;
      } else {
        key = keys[at];
      }
      atomicAdd(&local[(key >> shift) & mask], 1u);
    }
  }
  __syncthreads();
  counts[(size_t)blockIdx.x * kBins + threadIdx.x] = local[threadIdx.x];
}

// Moves every element of the tile to its place by one digit.  The place of the tile's first element of a digit is the
// number of elements with smaller digits plus those of the same digit in earlier tiles, which every CTA adds up from
// the counts itself (512 coalesced columns, `tiles` rows from L2).
template <typename Id, bool FIRST>
__global__ void __launch_bounds__(kSortThreads)
scatter_digits(const Id* __restrict__ tokens, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ order, uint32_t count,
               uint32_t vocabulary, long long padding, int shift, uint32_t mask, const uint32_t* __restrict__ counts, int tiles,
               uint32_t* __restrict__ keys_out, uint32_t* __restrict__ order_out) {
  __shared__ uint32_t counters[(kSortWarps + 1) * kBins];
  __shared__ uint32_t starts[kBins];
  __shared__ uint32_t warp_totals[kSortWarps];
  dependent_launch_prologue();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t total = 0, earlier = 0;
#pragma unroll 8
  for (int tile = 0; tile < tiles; ++tile) {
    const uint32_t n = counts[(size_t)tile * kBins + threadIdx.x];
    if (tile < (int)blockIdx.x) earlier += n;
    total += n;
  }
  starts[threadIdx.x] = exclusive_over_bins(total, warp_totals) + earlier;
  uint32_t key[kSortRounds], position[kSortRounds], digit[kSortRounds], rank[kSortRounds];
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const size_t at = (size_t)blockIdx.x * kTile + warp * (32 * kSortRounds) + r * 32 + lane;
    const bool valid = at < count;  // only the last tile has elements that are not, and they rank behind its others
    if constexpr (FIRST) {
      key[r] = valid ? key_of(tokens[at], vocabulary, padding, static_cast<int*>(nullptr)) : vocabulary;
      position[r] = (uint32_t)at;
    } else {
      key[r] = valid ? keys[at] : vocabulary;
      position[r] = valid ? order[at] : 0;
    }
    digit[r] = valid ? (key[r] >> shift) & mask : kBins - 1;
  }
  rank_tile(digit, rank, counters);
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const size_t at = (size_t)blockIdx.x * kTile + warp * (32 * kSortRounds) + r * 32 + lane;
    if (at < count) {
      const uint32_t to = starts[digit[r]] + rank[r];
      keys_out[to] = key[r];
      order_out[to] = position[r];
    }
  }
}

// ---- segmented sums ---------------------------------------------------------------------------------------------------
constexpr int kBatch = 8;  // rows of grad_out a thread has in flight

template <typename W, int VEC> __device__ __forceinline__ void write_row(W* __restrict__ row, const float (&sum)[VEC], float scale, bool accumulate) {
  Pack<W, VEC> r;
  if (accumulate) {
    const Pack<W, VEC> old = load_stream<W, VEC>(row);
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.v[e] = Conv<float, W>::narrow(fmaf(sum[e], scale, Conv<float, W>::widen(old.v[e])));
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.v[e] = Conv<float, W>::narrow(sum[e] * scale);
  }
  store_stream<W, VEC>(row, r);
}

struct Segments {
  const uint32_t* keys;   // sorted tokens
  const uint32_t* order;  // their positions
  float* partial;         // [chunks][2][hidden]: the sums of a chunk's first run (it began before) and of its last (it goes on)
  uint32_t count, vocabulary, chunk_length, chunks;
  int steps, lane_bits;
};

// One group of `1 << lane_bits` threads per chunk; a thread owns one vector column of it.
template <typename G, typename W, int VEC>
__global__ void __launch_bounds__(kThreads)
sum_chunks(const __grid_constant__ Segments s, const G* __restrict__ grad_out, W* __restrict__ grad_table, float scale, int accumulate) {
  dependent_launch_prologue();
  const size_t chunk = (size_t)blockIdx.x * (kThreads >> s.lane_bits) + (threadIdx.x >> s.lane_bits);
  if (chunk >= s.chunks) return;
  const size_t hidden = (size_t)s.steps * VEC;
  const uint32_t first = (uint32_t)(chunk * s.chunk_length);
  const uint32_t end = s.count - first < s.chunk_length ? s.count : first + s.chunk_length;
  if (s.keys[first] >= s.vocabulary) return;  // only dropped tokens from here on
  for (int step = (blockIdx.y << s.lane_bits) + (threadIdx.x & ((1 << s.lane_bits) - 1)); step < s.steps; step += gridDim.y << s.lane_bits) {
    const size_t column = (size_t)step * VEC;
    uint32_t current = s.keys[first];
    bool began_before = first > 0 && s.keys[first - 1] == current;
    float sum[VEC] = {};
    bool live = true;
    for (uint32_t at = first; at < end && live; at += kBatch) {
      uint32_t key[kBatch];
      Pack<G, VEC> rows[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        key[j] = at + j < end ? s.keys[at + j] : s.vocabulary;
        if (key[j] < s.vocabulary) rows[j] = load_stream<G, VEC>(grad_out + (size_t)s.order[at + j] * hidden + column);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (key[j] >= s.vocabulary) {  // behind the chunk's end, or dropped tokens: nothing follows
          live = false;
        } else {
          if (key[j] != current) {
            if (began_before) {
              float* to = s.partial + (chunk * 2) * hidden + column;
#pragma unroll
              for (int e = 0; e < VEC; ++e) to[e] = sum[e];
            } else {
              write_row<W, VEC>(grad_table + (size_t)current * hidden + column, sum, scale, accumulate != 0);
            }
            current = key[j];
            began_before = false;
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[e] = 0.0f;
          }
          float value[VEC];
          widen<G, VEC>(rows[j], value);
#pragma unroll
          for (int e = 0; e < VEC; ++e) sum[e] += value[e];
        }
      }
    }
    const bool goes_on = end < s.count && s.keys[end] == current;
    if (began_before || goes_on) {
      float* to = s.partial + (chunk * 2 + (began_before ? 0 : 1)) * hidden + column;
#pragma unroll
      for (int e = 0; e < VEC; ++e) to[e] = sum[e];
    } else {
      write_row<W, VEC>(grad_table + (size_t)current * hidden + column, sum, scale, accumulate != 0);
    }
  }
}

// Joins the partial sums of every run that crosses a chunk's border; the chunk where the run begins does it.
template <typename W, int VEC>
__global__ void __launch_bounds__(kThreads)
join_chunks(const __grid_constant__ Segments s, W* __restrict__ grad_table, float scale, int accumulate) {
  dependent_launch_prologue();
  const size_t chunk = (size_t)blockIdx.x * (kThreads >> s.lane_bits) + (threadIdx.x >> s.lane_bits);
  if (chunk + 1 >= s.chunks) return;  // the last chunk's last run ends with it
  const size_t hidden = (size_t)s.steps * VEC;
  const uint32_t first = (uint32_t)(chunk * s.chunk_length), next = first + s.chunk_length;
  const uint32_t key = s.keys[next - 1];
  if (key >= s.vocabulary || s.keys[next] != key) return;
  if (first > 0 && s.keys[first] == key && s.keys[first - 1] == key) return;  // began in an earlier chunk
  // the last chunk that the run reaches into
  size_t last = chunk + 1;
  while (last + 1 < s.chunks && s.keys[(last + 1) * s.chunk_length] == key) ++last;
  for (int step = (blockIdx.y << s.lane_bits) + (threadIdx.x & ((1 << s.lane_bits) - 1)); step < s.steps; step += gridDim.y << s.lane_bits) {
    const size_t column = (size_t)step * VEC;
    float sum[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = s.partial[(chunk * 2 + 1) * hidden + column + e];
    for (size_t c = chunk + 1; c <= last; ++c) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] += s.partial[c * 2 * hidden + column + e];
    }
    write_row<W, VEC>(grad_table + (size_t)key * hidden + column, sum, scale, accumulate != 0);
  }
}

// Zeros for every row that no token names.
template <typename W, int VEC>
__global__ void __launch_bounds__(kThreads)
zero_unnamed(const uint8_t* __restrict__ named, W* __restrict__ grad_table, uint32_t vocabulary, int steps, int lane_bits) {
  dependent_launch_prologue();
  const size_t row = (size_t)blockIdx.x * (kThreads >> lane_bits) + (threadIdx.x >> lane_bits);
  if (row >= vocabulary || named[row]) return;
  Pack<W, VEC> zero;
#pragma unroll
  for (int e = 0; e < VEC; ++e) zero.v[e] = Conv<float, W>::narrow(0.0f);
  const int lanes = 1 << lane_bits;
  for (int step = threadIdx.x & (lanes - 1); step < steps; step += lanes)
    store_stream<W, VEC>(grad_table + (row * steps + step) * VEC, zero);
}

struct GradientCall {
  const void* grad_out;
  const void* tokens;
  void* grad_table;
  size_t count, vocabulary, hidden;
  float scale;
  long long padding;
  int accumulate;
};

inline size_t round_up(size_t n) { return (n + 255) & ~(size_t)255; }

// Sorts the call's tokens; `keys` and `order` receive them.  `spare_*`: as much again, for the passes between.
template <typename Id>
int sort_tokens(const GradientCall& call, uint32_t* keys, uint32_t* order, uint32_t* spare_keys, uint32_t* spare_order, uint32_t* counts,
                uint8_t* named, cudaStream_t stream) {
  const uint32_t count = (uint32_t)call.count, vocabulary = (uint32_t)call.vocabulary;
  int bits = 1;  // of the keys 0 .. vocabulary
  while (((unsigned long long)call.vocabulary >> bits) != 0) ++bits;
  const int passes = (bits + kDigitBits - 1) / kDigitBits, digit_bits = (bits + passes - 1) / passes;
  const Id* tokens = static_cast<const Id*>(call.tokens);
  if (call.count <= (size_t)kTile) {
    constexpr int kSmem = (2 * kTile + (kSortWarps + 2) * kBins) * (int)sizeof(uint32_t);
    if (int status = check_runtime(cudaFuncSetAttribute(sort_tokens_small<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem),
                                   "cudaFuncSetAttribute(embedding_backward sort)"))
      return status;
    launch_dependent(sort_tokens_small<Id>, dim3(1), dim3(kSortThreads), kSmem, stream, tokens, count, vocabulary, call.padding, passes,
                     digit_bits, keys, order, named, device_status_word());
    return check_launch("embedding_backward sort launch");
  }
  const int tiles = (int)((call.count + kTile - 1) / kTile);
  const uint32_t mask = (1u << digit_bits) - 1;
  // the last pass writes `keys` and `order`: with an even number of passes the first one writes the spare pair
  for (int pass = 0; pass < passes; ++pass) {
    const bool to_result = (passes - 1 - pass) % 2 == 0;
    uint32_t *keys_to = to_result ? keys : spare_keys, *order_to = to_result ? order : spare_order;
    const uint32_t *keys_from = to_result ? spare_keys : keys, *order_from = to_result ? spare_order : order;
    const int shift = pass * digit_bits;
    if (pass == 0) {
      launch_dependent(count_digits<Id, true>, dim3(tiles), dim3(kSortThreads), 0, stream, tokens, keys_from, count, vocabulary, call.padding,
                       shift, mask, counts, named, device_status_word());
      if (int status = check_launch("embedding_backward count launch")) return status;
      launch_dependent(scatter_digits<Id, true>, dim3(tiles), dim3(kSortThreads), 0, stream, tokens, keys_from, order_from, count, vocabulary,
                       call.padding, shift, mask, static_cast<const uint32_t*>(counts), tiles, keys_to, order_to);
    } else {
      launch_dependent(count_digits<Id, false>, dim3(tiles), dim3(kSortThreads), 0, stream, tokens, keys_from, count, vocabulary, call.padding,
                       shift, mask, counts, static_cast<uint8_t*>(nullptr), static_cast<int*>(nullptr));
      if (int status = check_launch("embedding_backward count launch")) return status;
      launch_dependent(scatter_digits<Id, false>, dim3(tiles), dim3(kSortThreads), 0, stream, tokens, keys_from, order_from, count, vocabulary,
                       call.padding, shift, mask, static_cast<const uint32_t*>(counts), tiles, keys_to, order_to);
    }
    if (int status = check_launch("embedding_backward scatter launch")) return status;
  }
  return BB200_OK;
}

template <typename G, typename W, int VEC> int gradient(const GradientCall& call, bool wide_tokens, cudaStream_t stream) {
  const size_t count = call.count, steps = call.hidden / VEC;
  const size_t tiles = (count + kTile - 1) / kTile;
  const uint32_t chunk_length = count <= (1u << 16) ? 32 : count <= (1u << 19) ? 128 : 512;
  const size_t chunks = (count + chunk_length - 1) / chunk_length;
  const size_t list = round_up(count * 4), counts_bytes = round_up(tiles * kBins * 4), partial = round_up(chunks * 2 * call.hidden * 4);
  const size_t named_bytes = call.accumulate ? 0 : round_up(call.vocabulary);
  Workspace workspace(stream);
  if (int status = workspace.take(4 * list + counts_bytes + partial + named_bytes, "embedding_backward workspace")) return status;
  char* at = workspace.data();
  uint32_t* lists[4];
  for (uint32_t*& one : lists) {
    one = reinterpret_cast<uint32_t*>(at);
    at += list;
  }
  uint32_t* counts = reinterpret_cast<uint32_t*>(at);
  float* partials = reinterpret_cast<float*>(at + counts_bytes);
  uint8_t* named = call.accumulate ? nullptr : reinterpret_cast<uint8_t*>(at + counts_bytes + partial);
  if (named) {
    if (int status = check_runtime(cudaMemsetAsync(named, 0, call.vocabulary, stream), "cudaMemsetAsync(embedding_backward)")) return status;
  }
  if (int status = wide_tokens ? sort_tokens<int64_t>(call, lists[0], lists[1], lists[2], lists[3], counts, named, stream)
                               : sort_tokens<int32_t>(call, lists[0], lists[1], lists[2], lists[3], counts, named, stream))
    return status;
  Segments s = {};
  s.keys = lists[0];
  s.order = lists[1];
  s.partial = partials;
  s.count = (uint32_t)count;
  s.vocabulary = (uint32_t)call.vocabulary;
  s.chunk_length = chunk_length;
  s.chunks = (uint32_t)chunks;
  s.steps = (int)steps;
  s.lane_bits = 5;
  while (s.lane_bits < 8 && ((size_t)1 << s.lane_bits) < steps) ++s.lane_bits;
  const size_t groups = kThreads >> s.lane_bits, columns = (steps + ((size_t)1 << s.lane_bits) - 1) >> s.lane_bits;
  const dim3 grid((unsigned)((chunks + groups - 1) / groups), (unsigned)(columns < 65535 ? columns : 65535));
  W* table = static_cast<W*>(call.grad_table);
  launch_dependent(sum_chunks<G, W, VEC>, grid, dim3(kThreads), 0, stream, s, static_cast<const G*>(call.grad_out), table, call.scale, call.accumulate);
  if (int status = check_launch("embedding_backward sum launch")) return status;
  if (chunks > 1) {
    launch_dependent(join_chunks<W, VEC>, grid, dim3(kThreads), 0, stream, s, table, call.scale, call.accumulate);
    if (int status = check_launch("embedding_backward join launch")) return status;
  }
  if (named) {
    launch_dependent(zero_unnamed<W, VEC>, dim3((unsigned)((call.vocabulary + groups - 1) / groups)), dim3(kThreads), 0, stream,
                     static_cast<const uint8_t*>(named), table, s.vocabulary, s.steps, s.lane_bits);
    if (int status = check_launch("embedding_backward zero launch")) return status;
  }
  return workspace.release("cudaFreeAsync(embedding_backward workspace)");
}

bool is_float(bb200_dtype t) { return t == BB200_F32 || t == BB200_BF16 || t == BB200_F16; }

int check_extents(const char* what, size_t count, size_t vocabulary, size_t hidden, bb200_dtype token_dtype, bb200_dtype table_dtype,
                  bb200_dtype rows_dtype) {
  if (!is_float(table_dtype) || !is_float(rows_dtype))
    return fail(BB200_E_INVALID_ARGUMENT, "%s: dtypes %d and %d must be bf16/f16/f32", what, (int)table_dtype, (int)rows_dtype);
  if (token_dtype != BB200_I32 && token_dtype != BB200_I64)
    return fail(BB200_E_INVALID_ARGUMENT, "%s: token dtype %d is not i32/i64", what, (int)token_dtype);
  if (count == 0 || vocabulary == 0 || hidden == 0) return fail(BB200_E_INVALID_ARGUMENT, "%s: count, vocabulary and hidden must be > 0", what);
  if (count >= 0x7fffffffu || vocabulary >= 0x7fffffffu || hidden >= 0x7fffffffu)
    return fail(BB200_E_UNSUPPORTED_SHAPE, "%s: extents must be below 2^31 - 1", what);
  return BB200_OK;
}

bool misaligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

// Calls `f.run<T, O, VEC>()` for the two dtypes: whole 16-byte vectors of the narrower type where rows and pointers allow
// it, single elements otherwise.
template <typename F> int over_dtypes(bb200_dtype a, bb200_dtype b, size_t hidden, bool aligned, const F& f) {
#define BB200_PAIR(CODE_A, A, CODE_B, B)                                                     \
  if (a == CODE_A && b == CODE_B) {                                                          \
    constexpr int kVec = sizeof(A) == 4 && sizeof(B) == 4 ? 4 : 8;                           \
    return aligned && hidden % kVec == 0 ? f.template run<A, B, kVec>() : f.template run<A, B, 1>(); \
  }
  BB200_PAIR(BB200_F32, float, BB200_F32, float)
  BB200_PAIR(BB200_F32, float, BB200_BF16, __nv_bfloat16)
  BB200_PAIR(BB200_F32, float, BB200_F16, __half)
  BB200_PAIR(BB200_BF16, __nv_bfloat16, BB200_F32, float)
  BB200_PAIR(BB200_BF16, __nv_bfloat16, BB200_BF16, __nv_bfloat16)
  BB200_PAIR(BB200_BF16, __nv_bfloat16, BB200_F16, __half)
  BB200_PAIR(BB200_F16, __half, BB200_F32, float)
  BB200_PAIR(BB200_F16, __half, BB200_BF16, __nv_bfloat16)
  BB200_PAIR(BB200_F16, __half, BB200_F16, __half)
#undef BB200_PAIR
  return BB200_E_INVALID_ARGUMENT;
}

struct LookupCall {
  const void *tokens, *table;
  void* out;
  size_t count, vocabulary, hidden;
  float scale;
  bool wide_tokens;
  cudaStream_t stream;
  template <typename T, typename O, int VEC> int run() const {
    return wide_tokens ? launch_lookup<T, O, int64_t, VEC>(tokens, table, out, count, vocabulary, hidden, scale, stream)
                       : launch_lookup<T, O, int32_t, VEC>(tokens, table, out, count, vocabulary, hidden, scale, stream);
  }
};

struct GradientRun {
  GradientCall call;
  bool wide_tokens;
  cudaStream_t stream;
  template <typename G, typename W, int VEC> int run() const { return gradient<G, W, VEC>(call, wide_tokens, stream); }
};

}  // namespace
}  // namespace bb200

using namespace bb200;

extern "C" int bb200_embedding(bb200_dtype table_dtype, bb200_dtype out_dtype, bb200_dtype token_dtype, const void* tokens, const void* table,
                               void* out, size_t count, size_t vocabulary, size_t hidden, float scale, void* stream) {
  if (!tokens || !table || !out) return fail(BB200_E_INVALID_ARGUMENT, "embedding: null tensor pointer");
  if (int status = check_extents("embedding", count, vocabulary, hidden, token_dtype, table_dtype, out_dtype)) return status;
  if (misaligned(tokens, dtype_bytes(token_dtype)) || misaligned(table, dtype_bytes(table_dtype)) || misaligned(out, dtype_bytes(out_dtype)))
    return fail(BB200_E_MISALIGNED, "embedding: a tensor is not aligned to its element size");
  const size_t out_bytes = count * hidden * dtype_bytes(out_dtype);
  if (overlap(out, out_bytes, table, vocabulary * hidden * dtype_bytes(table_dtype)) || overlap(out, out_bytes, tokens, count * dtype_bytes(token_dtype)))
    return fail(BB200_E_INVALID_ARGUMENT, "embedding: out shares memory with an input");
  const LookupCall call = {tokens, table, out, count, vocabulary, hidden, scale, token_dtype == BB200_I64, static_cast<cudaStream_t>(stream)};
  return over_dtypes(table_dtype, out_dtype, hidden, aligned16(table) && aligned16(out), call);
}

extern "C" int bb200_embedding_backward(bb200_dtype grad_dtype, bb200_dtype table_dtype, bb200_dtype token_dtype, const void* grad_out,
                                        const void* tokens, void* grad_table, size_t count, size_t vocabulary, size_t hidden, float scale,
                                        int64_t padding_token, int accumulate, void* stream) {
  if (!grad_out || !tokens || !grad_table) return fail(BB200_E_INVALID_ARGUMENT, "embedding_backward: null tensor pointer");
  if (int status = check_extents("embedding_backward", count, vocabulary, hidden, token_dtype, table_dtype, grad_dtype)) return status;
  if (misaligned(tokens, dtype_bytes(token_dtype)) || misaligned(grad_out, dtype_bytes(grad_dtype)) || misaligned(grad_table, dtype_bytes(table_dtype)))
    return fail(BB200_E_MISALIGNED, "embedding_backward: a tensor is not aligned to its element size");
  const size_t table_bytes = vocabulary * hidden * dtype_bytes(table_dtype);
  if (overlap(grad_table, table_bytes, grad_out, count * hidden * dtype_bytes(grad_dtype)) ||
      overlap(grad_table, table_bytes, tokens, count * dtype_bytes(token_dtype)))
    return fail(BB200_E_INVALID_ARGUMENT, "embedding_backward: grad_table shares memory with an input");
  GradientRun run = {{grad_out, tokens, grad_table, count, vocabulary, hidden, scale, (long long)padding_token, accumulate},
                     token_dtype == BB200_I64, static_cast<cudaStream_t>(stream)};
  return over_dtypes(grad_dtype, table_dtype, hidden, aligned16(grad_out) && aligned16(grad_table), run);
}
