// embedding.cu — embedding lookup with scaling, and its gradient by sorted tokens, for sm_100a.
//
//   lookup:    out[t, :] = scale * table[token[t], :]
//   gradient:  grad_table[v, :] (= or +=) scale * sum over t with token[t] = v of grad_out[t, :]
//
// Both are bound by HBM bytes: the lookup reads every named row and writes out once, repeats from L2 while they are still
// there (65536 tokens: 1.3 to 1.6 times the distinct rows' bytes from DRAM); the gradient reads grad_out once and writes the
// table once (or reads and writes the named rows, when added).  Sums are fp32 and run in an order that the token positions
// alone fix, so the same call gives the same bits; no floating-point atomics.  Few tokens of few columns take one launch
// that finds the places of every token by comparing (sum_few); the gradient's steps otherwise:
//
//   1. a stable radix sort of (token, position) — one launch for up to 65536 tokens, held in the shared memory of a cluster
//      of CTAs, else a histogram and a scatter launch per digit;
//   2. segmented sums over equal chunks of the sorted positions, which balances frequent tokens by construction: a run
//      of one token inside a chunk is written straight to its row, a run that crosses a chunk's border leaves an fp32
//      partial row in the workspace;
//   3. one launch that joins the partial rows of every crossing run and, without `accumulate`, fills the rows that no
//      token names with zeros.
//
// Widths that are no whole 16-byte vectors, and tensors not aligned to them, move element by element: 65536 rows of 1004 bf16 take
// the lookup 89 us (1024: 29 us) and the gradient, written to 50257 rows, 122 us (75 us).
//
// Tokens outside [0, vocabulary) read as zeros (lookup) or contribute nothing (gradient) and are recorded in the device
// status word.  A padding token and out-of-range tokens sort behind every row under the key `vocabulary`.
#include "bb200_internal.h"
#include "bb200_rows.cuh"

namespace bb200 {
namespace {

constexpr int kThreads = 256;

// The fp32 sum of some rows' vectors: VEC elements, in pairs where there are any.
template <int VEC> struct Sum {
  F2 pair[VEC / 2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) pair[i] = both(0.0f);
  }
  template <typename T> __device__ __forceinline__ void add(const Pack<T, VEC>& v) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) pair[i] = pair[i] + Pairs<T>::get(v, i);
  }
  // the sum times `scale` (and plus `old`), rounded once
  template <typename T> __device__ __forceinline__ Pack<T, VEC> times(float scale) const {
    Pack<T, VEC> r;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) Pairs<T>::set(r, i, pair[i] * both(scale));
    return r;
  }
  template <typename T> __device__ __forceinline__ Pack<T, VEC> times_plus(float scale, const Pack<T, VEC>& old) const {
    Pack<T, VEC> r;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) Pairs<T>::set(r, i, fma2(pair[i], both(scale), Pairs<T>::get(old, i)));
    return r;
  }
  __device__ __forceinline__ Pack<float, VEC> values() const { return times<float>(1.0f); }
};
template <> struct Sum<1> {
  float value;
  __device__ __forceinline__ void clear() { value = 0.0f; }
  template <typename T> __device__ __forceinline__ void add(const Pack<T, 1>& v) { value += Conv<float, T>::widen(v.v[0]); }
  template <typename T> __device__ __forceinline__ Pack<T, 1> times(float scale) const { return {{Conv<float, T>::narrow(value * scale)}}; }
  template <typename T> __device__ __forceinline__ Pack<T, 1> times_plus(float scale, const Pack<T, 1>& old) const {
    return {{Conv<float, T>::narrow(fmaf(value, scale, Conv<float, T>::widen(old.v[0])))}};
  }
  __device__ __forceinline__ Pack<float, 1> values() const { return {{value}}; }
};

// A token outside the table is recorded only where nothing else is: the code of a wait that gave up, which means that some
// output is incomplete, stays.
__device__ __forceinline__ void record_bad_token(int* status_word) {
  if (status_word) atomicCAS(status_word, 0, BB200_TOKEN_OUT_OF_RANGE);
}

// ---- lookup -------------------------------------------------------------------------------------------------------
// `1 << lane_bits` neighbouring threads share a row; each has four vectors of it on their way at once.  Up to 64 threads a
// row: 65536 rows of 4096 bf16 114 us, 124 us with two vectors a thread; f32 to bf16 156 us, 160 us with 256 threads a row.
constexpr int kUnroll = 4, kMostLaneBits = 6;

template <typename O, typename T, int VEC> __device__ __forceinline__ Pack<O, VEC> scaled(const Pack<T, VEC>& v, float scale) {
  Pack<O, VEC> r;
  if constexpr (VEC == 1) {
    r.v[0] = Conv<float, O>::narrow(Conv<float, T>::widen(v.v[0]) * scale);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) Pairs<O>::set(r, i, Pairs<T>::get(v, i) * both(scale));
  }
  return r;
}

template <typename T, typename O, typename Id, int VEC>
__global__ void __launch_bounds__(kThreads)
lookup_rows(const Id* __restrict__ tokens, const T* __restrict__ table, O* __restrict__ out, size_t count, size_t vocabulary, int steps,
            int lane_bits, float scale, bool wide, int* status_word) {
  dependent_launch_prologue();
  const int lanes = 1 << lane_bits, lane = threadIdx.x & (lanes - 1);
  const size_t row = (size_t)blockIdx.x * (kThreads >> lane_bits) + (threadIdx.x >> lane_bits);
  if (row >= count) return;
  const long long token = (long long)tokens[row];
  const bool inside = token >= 0 && (unsigned long long)token < vocabulary;
  if (!inside && lane == 0 && blockIdx.y == 0) record_bad_token(status_word);
  const T* __restrict__ source = table + (inside ? (size_t)token : 0) * ((size_t)steps * VEC);
  O* __restrict__ target = out + row * ((size_t)steps * VEC);
  for (int step = blockIdx.y * kUnroll * lanes + lane; step < steps; step += gridDim.y * kUnroll * lanes) {
    Pack<T, VEC> a[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (step + u * lanes < steps) a[u] = load_stream_32<T, VEC>(source + (size_t)(step + u * lanes) * VEC, wide);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (step + u * lanes < steps) {
        Pack<O, VEC> r;
        if (inside) {
          r = scaled<O>(a[u], scale);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) r.v[e] = Conv<float, O>::narrow(0.0f);
        }
        store_stream_32<O, VEC>(target + (size_t)(step + u * lanes) * VEC, r, wide);
      }
    }
  }
}

template <typename T, typename O, typename Id, int VEC>
int launch_lookup(const void* tokens, const void* table, void* out, size_t count, size_t vocabulary, size_t hidden, float scale,
                  cudaStream_t stream) {
  const int steps = (int)(hidden / VEC);
  int lane_bits = 2;
  while (lane_bits < kMostLaneBits && (kUnroll << lane_bits) < steps) ++lane_bits;
  const size_t rows_per_block = kThreads >> lane_bits;
  const size_t blocks = (count + rows_per_block - 1) / rows_per_block;
  const size_t columns = ((size_t)steps + ((size_t)kUnroll << lane_bits) - 1) / ((size_t)kUnroll << lane_bits);
  launch_dependent(lookup_rows<T, O, Id, VEC>, dim3((unsigned)blocks, (unsigned)(columns < 65535 ? columns : 65535)), dim3(kThreads), 0, stream,
                   static_cast<const Id*>(tokens), static_cast<const T*>(table), static_cast<O*>(out), count, vocabulary, steps, lane_bits,
                   scale, aligned32(table) && aligned32(out), device_status_word());
  return check_launch("embedding kernel launch");
}

// ---- sorting the tokens ---------------------------------------------------------------------------------------------
// Least-significant-digit radix sort of (token, position), stable, digits of at most 9 bits.  A CTA ranks 1024 * R elements:
// warp w holds elements [32 R w, 32 R (w + 1)), 32 at a time in order; within 32 the rank among equal digits comes from
// a ballot per bit, earlier 32s of the warp are counted in the warp's own shared-memory counters, and earlier warps by a
// prefix over the 32 counters of a digit.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kDigitBits = 9, kBins = 1 << kDigitBits;
// 16-bit counters, two digits to a word; rows of 257 words keep the prefix over warps free of bank conflicts.
constexpr int kCounterWords = kBins / 2 + 1;

template <typename Id> __device__ __forceinline__ uint32_t key_of(Id raw, uint32_t vocabulary, long long padding, int* status_word) {
  const long long token = (long long)raw;
  if (token < 0 || token >= (long long)vocabulary) {
    record_bad_token(status_word);
    return vocabulary;
  }
  return token == padding ? vocabulary : (uint32_t)token;
}

// Stable rank of each of a thread's R elements among the CTA's elements of the same digit; totals[d] = how many there are.
template <int R>
__device__ __forceinline__ void rank_digits(const uint32_t (&digit)[R], uint32_t (&rank)[R], int digit_bits, uint32_t (*counters)[kCounterWords], uint32_t* totals) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int word = lane; word < kCounterWords; word += 32) counters[warp][word] = 0;
  uint16_t* mine = reinterpret_cast<uint16_t*>(counters[warp]);
  __syncwarp();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    uint32_t same = 0xffffffffu;
    for (int bit = 0; bit < digit_bits; ++bit) {
      const bool set = (digit[r] >> bit) & 1;
      const uint32_t vote = __ballot_sync(0xffffffffu, set);
      same &= set ? vote : ~vote;
    }
    const uint32_t before = __popc(same & ((1u << lane) - 1));
    rank[r] = mine[digit[r]] + before;
    __syncwarp();
    if (before == 0) mine[digit[r]] = (uint16_t)(rank[r] + __popc(same));
    __syncwarp();
  }
  __syncthreads();
  {  // four threads to a word, eight warps to a thread: exclusive prefix over the warps, both halves of the word at once
    const int word = threadIdx.x >> 2, part = threadIdx.x & 3;
    static_assert(kSortThreads == kBins * 2 && kSortWarps == 32, "four threads to a word, eight warps each");
    uint32_t n[8], sum = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) n[w] = counters[part * 8 + w][word];
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const uint32_t own = n[w];
      n[w] = sum;
      sum += own;  // the halves stay below 8192
    }
    uint32_t inclusive = sum;
#pragma unroll
    for (int offset = 1; offset < 4; offset <<= 1) {
      const uint32_t below = __shfl_up_sync(0xffffffffu, inclusive, offset, 4);
      if (part >= offset) inclusive += below;
    }
    const uint32_t base = inclusive - sum;
#pragma unroll
    for (int w = 0; w < 8; ++w) counters[part * 8 + w][word] = base + n[w];
    if (part == 3) {
      totals[2 * word] = inclusive & 0xffffu;
      totals[2 * word + 1] = inclusive >> 16;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) rank[r] += mine[digit[r]];
}

// Exclusive prefix sum over kBins values, one to a thread (threads past them bring 0 and are ignored).
__device__ __forceinline__ uint32_t exclusive_over_bins(uint32_t value, uint32_t* warp_totals) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t inclusive = value;
#pragma unroll
  for (int offset = 1; offset < 32; offset <<= 1) {
    const uint32_t below = __shfl_up_sync(0xffffffffu, inclusive, offset);
    if (lane >= offset) inclusive += below;
  }
  if (lane == 31) warp_totals[warp] = inclusive;
  __syncthreads();
  uint32_t others = lane < warp ? warp_totals[lane] : 0;
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) others += __shfl_xor_sync(0xffffffffu, others, offset);
  __syncthreads();
  return others + inclusive - value;
}

struct SortedList {
  uint32_t* keys;
  uint32_t* order;
  uint32_t* crossings;  // see Segments; the two counts are set to 0 here
};

// Up to 65536 tokens in one launch: one cluster of up to 16 CTAs holds them all in shared memory.  Every pass ranks in
// each CTA, adds up the CTAs' digit counts through distributed shared memory and sends every element to its place there;
// nobody touches another CTA's memory after the last pass's barrier.  A sort keeps few SMs busy, so where the whole table is
// written the launch has more clusters, which meanwhile fill the table's first rows with zeros (the sums overwrite those
// that tokens name).
constexpr uint32_t kMostCtas = 16;

template <int R> struct ClusterSort {
  uint2 pairs[kSortThreads * R];
  uint32_t counters[kSortWarps][kCounterWords];
  uint32_t totals[kBins];
  uint32_t starts[kBins];
  uint32_t warp_totals[kSortWarps];
};

template <typename Id, int R>
__global__ void __launch_bounds__(kSortThreads, 1)
sort_in_cluster(const Id* __restrict__ tokens, uint32_t count, uint32_t vocabulary, long long padding, int passes, int digit_bits, uint32_t ctas,
                const __grid_constant__ SortedList list, uint8_t* __restrict__ named, uint4* __restrict__ zeros, size_t zero_vectors, int* status_word) {
  constexpr uint32_t kEach = kSortThreads * R;
  extern __shared__ __align__(16) unsigned char shared[];
  ClusterSort<R>& s = *reinterpret_cast<ClusterSort<R>*>(shared);
  dependent_launch_prologue();
  if (blockIdx.x >= ctas) {  // the other clusters
    const size_t stride = (size_t)(gridDim.x - ctas) * kSortThreads;
    for (size_t i = (size_t)(blockIdx.x - ctas) * kSortThreads + threadIdx.x; i < zero_vectors; i += stride) __stcs(zeros + i, make_uint4(0, 0, 0, 0));
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank_of_cta = cluster_rank();
  uint32_t key[R], position[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    position[r] = rank_of_cta * kEach + warp * (32 * R) + r * 32 + lane;
    // the fill beyond `count` sorts behind every token, dropped ones included, because it comes after them
    key[r] = position[r] < count ? key_of(tokens[position[r]], vocabulary, padding, status_word) : vocabulary;
    if (named && key[r] < vocabulary) named[key[r]] = 1;
  }
  if (blockIdx.x == 0 && threadIdx.x < 2) list.crossings[threadIdx.x] = 0;
  for (int pass = 0; pass < passes; ++pass) {
    uint32_t digit[R], rank[R];
#pragma unroll
    for (int r = 0; r < R; ++r) digit[r] = (key[r] >> (pass * digit_bits)) & ((1u << digit_bits) - 1);
    rank_digits<R>(digit, rank, digit_bits, s.counters, s.totals);
    uint32_t total = 0, earlier = 0;
    if (ctas > 1) cluster_barrier();  // every CTA's totals stand
    if (threadIdx.x < kBins) {
      uint32_t n[kMostCtas];  // all of them on their way at once
#pragma unroll
      for (uint32_t c = 0; c < kMostCtas; ++c) {
        n[c] = 0;
        if (c < ctas) asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(n[c]) : "r"(in_cta(&s.totals[threadIdx.x], c)) : "memory");
      }
#pragma unroll
      for (uint32_t c = 0; c < kMostCtas; ++c) {
        if (c < rank_of_cta) earlier += n[c];
        total += n[c];
      }
    }
    const uint32_t start = exclusive_over_bins(total, s.warp_totals) + earlier;
    if (threadIdx.x < kBins) s.starts[threadIdx.x] = start;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t to = s.starts[digit[r]] + rank[r];
      asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(in_cta(&s.pairs[to % kEach], to / kEach)), "r"(key[r]), "r"(position[r]) : "memory");
    }
    if (ctas > 1) cluster_barrier();  // everything has arrived, and every CTA has read the totals
    else __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint2 pair = s.pairs[warp * (32 * R) + r * 32 + lane];
      key[r] = pair.x;
      position[r] = pair.y;
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint32_t at = rank_of_cta * kEach + warp * (32 * R) + r * 32 + lane;
    if (at < count) {
      list.keys[at] = key[r];
      list.order[at] = position[r];
    }
  }
}

// More tokens: per digit a launch that counts and a launch that scatters, a tile of 8192 to a CTA.
constexpr int kTileRounds = 8, kTile = kSortThreads * kTileRounds;

// counts[tile][digit] of one digit.  The first pass reads the tokens themselves and marks the rows they name.
template <typename Id, bool FIRST>
__global__ void __launch_bounds__(kSortThreads)
count_digits(const Id* __restrict__ tokens, const uint32_t* __restrict__ keys, uint32_t count, uint32_t vocabulary, long long padding,
             int shift, uint32_t mask, uint32_t* __restrict__ counts, uint8_t* __restrict__ named, int* status_word) {
  __shared__ uint32_t local[kBins];
  dependent_launch_prologue();
  if (threadIdx.x < kBins) local[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
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
  if (threadIdx.x < kBins) counts[(size_t)blockIdx.x * kBins + threadIdx.x] = local[threadIdx.x];
}

// Moves every element of the tile to its place by one digit.  The place of the tile's first element of a digit is the
// number of elements with smaller digits plus those of the same digit in earlier tiles, which every CTA adds up from
// the counts itself (512 coalesced columns, `tiles` rows from L2).
template <typename Id, bool FIRST>
__global__ void __launch_bounds__(kSortThreads)
scatter_digits(const Id* __restrict__ tokens, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ order, uint32_t count,
               uint32_t vocabulary, long long padding, int shift, uint32_t mask, const uint32_t* __restrict__ counts, int tiles,
               const __grid_constant__ SortedList list, int last) {
  __shared__ uint32_t counters[kSortWarps][kCounterWords];
  __shared__ uint32_t totals[kBins];
  __shared__ uint32_t starts[kBins];
  __shared__ uint32_t warp_totals[kSortWarps];
  dependent_launch_prologue();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t total = 0, earlier = 0;
  if (threadIdx.x < kBins) {
#pragma unroll 8
    for (int tile = 0; tile < tiles; ++tile) {
      const uint32_t n = counts[(size_t)tile * kBins + threadIdx.x];
      if (tile < (int)blockIdx.x) earlier += n;
      total += n;
    }
  }
  const uint32_t start = exclusive_over_bins(total, warp_totals) + earlier;
  if (threadIdx.x < kBins) starts[threadIdx.x] = start;
  uint32_t key[kTileRounds], position[kTileRounds], digit[kTileRounds], rank[kTileRounds];
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const size_t at = (size_t)blockIdx.x * kTile + warp * (32 * kTileRounds) + r * 32 + lane;
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
  rank_digits<kTileRounds>(digit, rank, kDigitBits, counters, totals);
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const size_t at = (size_t)blockIdx.x * kTile + warp * (32 * kTileRounds) + r * 32 + lane;
    if (at < count) {
      const uint32_t to = starts[digit[r]] + rank[r];
      list.keys[to] = key[r];
      list.order[to] = position[r];
    }
  }
  if (last && blockIdx.x == 0 && threadIdx.x < 2) list.crossings[threadIdx.x] = 0;
}

// ---- segmented sums ---------------------------------------------------------------------------------------------------
constexpr uint32_t kShortSpan = 8;

struct Segments {
  const uint32_t* keys;   // sorted tokens
  const uint32_t* order;  // their positions
  // the runs that cross a chunk's border, by the chunk where they begin: [0] how many reach into fewer than kShortSpan further
  // chunks, [1] how many into more, then room for all of them, the short ones from the front and the long ones from the back
  uint32_t* crossings;
  float* partial;  // [chunks][2][hidden]: the sums of a chunk's first run (it began before) and of its last (it goes on)
  uint32_t count, vocabulary, chunk_length, chunks;
  uint32_t fill_from;  // the first row that may still need zeros
  int steps, lane_bits;
  bool wide;  // table and gradient are aligned to 32 bytes
};

// One group of `1 << lane_bits` threads per chunk; a thread owns one vector column of it and has a batch of rows in
// flight, with the table's rows that the batch completes where they are added to.  The chunks' keys and positions are
// staged in shared memory first, so that only the rows themselves are waited for.
constexpr int kStagedList = 4096;  // entries for all chunks of a CTA

template <typename G, typename W, int VEC, bool ADD>
__global__ void __launch_bounds__(kThreads, 3)
sum_chunks(const __grid_constant__ Segments s, const G* __restrict__ grad_out, W* __restrict__ grad_table, float scale) {
  constexpr int kBatch = (int)sizeof(G) * VEC + (ADD ? (int)sizeof(W) * VEC : 0) <= 16 ? 8 : 4;
  extern __shared__ uint32_t staged[];  // keys of the CTA's chunks and one behind them, then their positions
  dependent_launch_prologue();
  const uint32_t groups = kThreads >> s.lane_bits, group = threadIdx.x >> s.lane_bits, entries = groups * s.chunk_length;
  {
    const size_t from = (size_t)blockIdx.x * entries;
    for (uint32_t i = threadIdx.x; i <= entries; i += kThreads) {
      const bool inside = from + i < s.count;
      staged[i] = inside ? s.keys[from + i] : s.vocabulary;
      if (i < entries) staged[entries + 1 + i] = inside ? s.order[from + i] : 0;
    }
  }
  __syncthreads();
  const size_t chunk = (size_t)blockIdx.x * groups + group;
  if (chunk >= s.chunks) return;
  const uint32_t* keys = staged + group * s.chunk_length;
  const uint32_t* order = staged + entries + 1 + group * s.chunk_length;
  const int lane = threadIdx.x & ((1 << s.lane_bits) - 1);
  const size_t hidden = (size_t)s.steps * VEC, first = chunk * s.chunk_length;
  const bool first_began_before = first > 0 && s.keys[first - 1] == keys[0];
  for (int step = (blockIdx.y << s.lane_bits) + lane; step < s.steps; step += gridDim.y << s.lane_bits) {
    const size_t column = (size_t)step * VEC;
    const G* from = grad_out + column;
    bool began_before = first_began_before, open = false;
    Sum<VEC> sum;
    sum.clear();
    for (uint32_t at = 0; at < s.chunk_length; at += kBatch) {
      uint32_t key[kBatch + 1];
#pragma unroll
      for (int j = 0; j <= kBatch; ++j) key[j] = keys[at + j];
      if (key[0] >= s.vocabulary) break;  // dropped tokens, or behind the list: nothing follows
      Pack<G, VEC> rows[kBatch];
      Pack<W, VEC> old[ADD ? kBatch : 1];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (key[j] < s.vocabulary) {
          rows[j] = load_stream_32<G, VEC>(from + (size_t)order[at + j] * hidden, s.wide);
          if constexpr (ADD) {
            if (key[j] != key[j + 1]) old[j] = load_stream_32<W, VEC>(grad_table + (size_t)key[j] * hidden + column, s.wide);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (key[j] < s.vocabulary) {
          sum.add(rows[j]);
          open = key[j] == key[j + 1];
          if (!open) {
            W* row = grad_table + (size_t)key[j] * hidden + column;
            if (began_before) store_stream_32<float, VEC>(s.partial + chunk * 2 * hidden + column, sum.values(), true);
            else if constexpr (ADD) store_stream_32<W, VEC>(row, sum.times_plus(scale, old[j]), s.wide);
            else store_stream_32<W, VEC>(row, sum.template times<W>(scale), s.wide);
            began_before = false;
            sum.clear();
          }
        }
      }
    }
    if (open) {
      store_stream_32<float, VEC>(s.partial + (chunk * 2 + (began_before ? 0 : 1)) * hidden + column, sum.values(), true);
      if (!began_before && step == 0) {
        const size_t probe = chunk + kShortSpan;
        const bool is_long = probe < s.chunks && s.keys[probe * s.chunk_length] == keys[s.chunk_length - 1];
        const uint32_t at = atomicAdd(s.crossings + is_long, 1u);
        s.crossings[is_long ? 1 + s.chunks - at : 2 + at] = (uint32_t)chunk;
      }
    }
  }
}

// Two jobs in one launch.  The first `join_blocks` CTAs join the partial sums of the runs that cross a chunk's border, 32
// vector columns of one run at a time and in a fixed order: a warp for a run of a few chunks, the CTA's eight warps over the
// chunks of a long one.  The other CTAs, where the whole table is written, fill the rows that no token names with zeros; the
// joins hide behind them.
constexpr int kFillRows = 4;  // rows that a group looks at together

template <typename W, int VEC, bool ADD>
__global__ void __launch_bounds__(kThreads, ADD ? 4 : 6)
join_and_fill(const __grid_constant__ Segments s, W* __restrict__ grad_table, float scale, unsigned join_blocks, const uint8_t* __restrict__ named) {
  __shared__ Pack<float, VEC> parts[kThreads / 32][32];
  dependent_launch_prologue();
  const size_t hidden = (size_t)s.steps * VEC;
  if (blockIdx.x >= join_blocks) {
    const int lanes = 1 << s.lane_bits, groups = kThreads >> s.lane_bits;
    const size_t first = s.fill_from + (size_t)(blockIdx.x - join_blocks) * groups * kFillRows + (threadIdx.x >> s.lane_bits);
    bool empty[kFillRows];
#pragma unroll
    for (int r = 0; r < kFillRows; ++r) empty[r] = first + r * groups < s.vocabulary && !named[first + r * groups];
    Pack<W, VEC> zero;
#pragma unroll
    for (int e = 0; e < VEC; ++e) zero.v[e] = Conv<float, W>::narrow(0.0f);
#pragma unroll
    for (int r = 0; r < kFillRows; ++r) {
      if (empty[r]) {
        W* row = grad_table + (first + r * groups) * ((size_t)s.steps * VEC);
        for (int step = threadIdx.x & (lanes - 1); step < s.steps; step += lanes) store_stream_32<W, VEC>(row + (size_t)step * VEC, zero, s.wide);
      }
    }
    return;
  }
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const uint32_t tiles = (uint32_t)(s.steps + 31) / 32;
  const unsigned long long short_items = (unsigned long long)s.crossings[0] * tiles, items = (unsigned long long)s.crossings[1] * tiles;
  for (unsigned long long item = (unsigned long long)blockIdx.x * (kThreads / 32) + slice; item < short_items; item += (unsigned long long)join_blocks * (kThreads / 32)) {
    const size_t chunk = s.crossings[2 + item / tiles], probe = chunk + 1 + lane;
    const int step = (int)(item % tiles) * 32 + lane;
    const uint32_t key = s.keys[(chunk + 1) * s.chunk_length - 1];
    const int further = __popc(__ballot_sync(0xffffffffu, probe < s.chunks && s.keys[probe * s.chunk_length] == key));
    if (step < s.steps) {
      const float* from = s.partial + (chunk * 2 + 1) * hidden + (size_t)step * VEC;
      Sum<VEC> sum;
      sum.clear();
      sum.add(load_stream_32<float, VEC>(from, true));
      from += hidden;
#pragma unroll 4
      for (int c = 0; c < further; ++c) sum.add(load_stream_32<float, VEC>(from + (size_t)c * 2 * hidden, true));
      W* row = grad_table + (size_t)key * hidden + (size_t)step * VEC;
      if constexpr (ADD) store_stream_32<W, VEC>(row, sum.times_plus(scale, load_stream_32<W, VEC>(row, s.wide)), s.wide);
      else store_stream_32<W, VEC>(row, sum.template times<W>(scale), s.wide);
    }
  }
  for (unsigned long long item = blockIdx.x; item < items; item += join_blocks) {
    const size_t chunk = s.crossings[1 + s.chunks - item / tiles];
    const int step = (int)(item % tiles) * 32 + lane;
    const size_t column = (size_t)step * VEC;
    const uint32_t key = s.keys[(chunk + 1) * s.chunk_length - 1];
    size_t end = chunk + 1;  // one past the last chunk that the run reaches into: the chunks it does begin with the key
    for (bool more = true; more; ) {
      const size_t probe = end + threadIdx.x;
      const int found = __syncthreads_count(probe < s.chunks && s.keys[probe * s.chunk_length] == key);
      end += found;
      more = found == kThreads;
    }
    Sum<VEC> sum;
    sum.clear();
    if (step < s.steps) {
#pragma unroll 8
      for (size_t c = chunk + slice; c < end; c += kThreads / 32)
        sum.add(load_stream_32<float, VEC>(s.partial + (c * 2 + (c == chunk ? 1 : 0)) * hidden + column, true));
    }
    parts[slice][lane] = sum.values();
    __syncthreads();
    if (slice == 0 && step < s.steps) {
#pragma unroll
      for (int w = 1; w < kThreads / 32; ++w) sum.add(parts[w][lane]);
      W* row = grad_table + (size_t)key * hidden + column;
      if constexpr (ADD) store_stream_32<W, VEC>(row, sum.times_plus(scale, load_stream_32<W, VEC>(row, s.wide)), s.wide);
      else store_stream_32<W, VEC>(row, sum.template times<W>(scale), s.wide);
    }
    __syncthreads();
  }
}

// ---- few tokens -------------------------------------------------------------------------------------------------------
// Up to 1024 tokens need no sort, workspace or second launch: a CTA holds all keys, and a warp finds the places of its token by
// comparing it with all of them.  The token's first place does the work: the warp sums the rows of a short run, the CTA's eight
// warps those of a long one, slice by slice in a fixed order.  CTAs of 8 tokens by 32 vector columns.  Where the whole
// table is written, further CTAs fill the rows that no token names, which they find in the keys as well.
constexpr uint32_t kMostDirect = 1024;
constexpr int kDirectTokens = kThreads / 32, kShortRun = 16;

struct Direct {
  const void* tokens;
  uint32_t count, vocabulary, sum_blocks, column_tiles, fill_rows;
  long long padding;
  int steps;
  bool wide_tokens, wide;  // i64 tokens; gradient and table aligned to 32 bytes
  int* status_word;
};

__device__ __forceinline__ uint32_t direct_key(const Direct& d, uint32_t at, int* status_word) {
  return d.wide_tokens ? key_of(static_cast<const int64_t*>(d.tokens)[at], d.vocabulary, d.padding, status_word)
                       : key_of(static_cast<const int32_t*>(d.tokens)[at], d.vocabulary, d.padding, status_word);
}

template <typename G, typename W, int VEC, bool ADD>
__global__ void __launch_bounds__(kThreads)
sum_few(const __grid_constant__ Direct d, const G* __restrict__ grad_out, W* __restrict__ grad_table, float scale) {
  constexpr int kBatch = (int)sizeof(G) * VEC <= 16 ? 8 : 4;
  __shared__ uint4 all[kMostDirect / 4];
  __shared__ uint16_t places[kMostDirect];  // of the CTA's tokens, run after run: distinct tokens, so there is room
  __shared__ uint32_t lengths[kDirectTokens];
  __shared__ Pack<float, VEC> parts[kDirectTokens][32];
  dependent_launch_prologue();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t hidden = (size_t)d.steps * VEC;
  if (blockIdx.x >= d.sum_blocks) {
    uint8_t* named = reinterpret_cast<uint8_t*>(all);  // at most kMostFillRows of them
    const uint32_t first = (blockIdx.x - d.sum_blocks) * d.fill_rows;
    const uint32_t rows = d.vocabulary - first < d.fill_rows ? d.vocabulary - first : d.fill_rows;
    for (uint32_t r = threadIdx.x; r < rows; r += kThreads) named[r] = 0;
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < d.count; at += kThreads) {
      const uint32_t key = direct_key(d, at, nullptr);
      if (key - first < rows) named[key - first] = 1;
    }
    __syncthreads();
    Pack<W, VEC> zero;
#pragma unroll
    for (int e = 0; e < VEC; ++e) zero.v[e] = Conv<float, W>::narrow(0.0f);
    for (uint32_t r = warp; r < rows; r += kThreads / 32) {
      if (named[r]) continue;
      W* row = grad_table + (size_t)(first + r) * hidden;
      for (int step = lane; step < d.steps; step += 32) store_stream_32<W, VEC>(row + (size_t)step * VEC, zero, d.wide);
    }
    return;
  }
  const uint32_t tile = blockIdx.x % d.column_tiles, group = blockIdx.x / d.column_tiles * kDirectTokens;
  uint32_t* keys = reinterpret_cast<uint32_t*>(all);
  const uint32_t padded = (d.count + 127) & ~127u;
#pragma unroll
  for (uint32_t k = 0; k < kMostDirect; k += kThreads) {
    const uint32_t at = k + threadIdx.x;
    if (at < padded) keys[at] = at < d.count ? direct_key(d, at, tile == 0 && at - group < (uint32_t)kDirectTokens ? d.status_word : nullptr) : 0xffffffffu;
  }
  __syncthreads();
  const uint32_t mine = group + warp;
  const uint32_t key = mine < d.count ? keys[mine] : d.vocabulary;
  uint32_t found = 0, earlier = 0;  // four bits for each of up to eight vectors of keys
  if (key < d.vocabulary) {
#pragma unroll
    for (uint32_t i = 0; i < kMostDirect / 128; ++i) {
      if (i * 128 < padded) {
        const uint4 four = all[i * 32 + lane];
        const uint32_t equal = (four.x == key) | (four.y == key) << 1 | (four.z == key) << 2 | (four.w == key) << 3;
        const uint32_t at = (i * 32 + lane) * 4;
        earlier |= at + 4 <= mine ? equal : at < mine ? equal & ((1u << (mine - at)) - 1) : 0;
        found |= equal << (4 * i);
      }
    }
  }
  const uint32_t length = __any_sync(0xffffffffu, earlier != 0) ? 0 : __reduce_add_sync(0xffffffffu, __popc(found));
  if (lane == 0) lengths[warp] = length;
  __syncthreads();
  uint32_t start = 0;
  for (int w = 0; w < warp; ++w) start += lengths[w];
  if (length) {
    uint32_t to = start;
#pragma unroll
    for (uint32_t i = 0; i < kMostDirect / 128; ++i) {
      if (i * 128 < padded) {
        const uint32_t bits = found >> (4 * i) & 15u;
        uint32_t below = __popc(bits), total;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
          const uint32_t other = __shfl_up_sync(0xffffffffu, below, offset);
          if (lane >= offset) below += other;
        }
        total = __shfl_sync(0xffffffffu, below, 31);
        below -= __popc(bits);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (bits >> e & 1) places[to + below++] = (uint16_t)((i * 32 + lane) * 4 + e);
        to += total;
      }
    }
  }
  __syncthreads();
  const auto add_rows = [&](Sum<VEC>& sum, const G* from, uint32_t begin, uint32_t end) {
    for (uint32_t at = begin; at < end; at += kBatch) {
      Pack<G, VEC> rows[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (at + j < end) rows[j] = load_stream_32<G, VEC>(from + (size_t)places[at + j] * hidden, d.wide);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (at + j < end) sum.add(rows[j]);
    }
  };
  const auto store = [&](const Sum<VEC>& sum, W* row, const Pack<W, VEC>& old) {
    if constexpr (ADD) store_stream_32<W, VEC>(row, sum.times_plus(scale, old), d.wide);
    else store_stream_32<W, VEC>(row, sum.template times<W>(scale), d.wide);
  };
  const int step = (int)tile * 32 + lane;
  const bool inside = step < d.steps;
  const G* from = grad_out + (size_t)step * VEC;
  if (length && length <= kShortRun && inside) {
    W* row = grad_table + (size_t)key * hidden + (size_t)step * VEC;
    Pack<W, VEC> old;
    if constexpr (ADD) old = load_stream_32<W, VEC>(row, d.wide);
    Sum<VEC> sum;
    sum.clear();
    add_rows(sum, from, start, start + length);
    store(sum, row, old);
  }
  uint32_t begin = 0;
  for (int run = 0; run < kDirectTokens; ++run) {  // the same for the whole CTA
    const uint32_t all_of_it = lengths[run], slice = (all_of_it + kDirectTokens - 1) / kDirectTokens;
    if (all_of_it > kShortRun) {
      const uint32_t low = warp * slice < all_of_it ? warp * slice : all_of_it, high = low + slice < all_of_it ? low + slice : all_of_it;
      W* row = grad_table + (size_t)keys[group + run] * hidden + (size_t)step * VEC;
      Pack<W, VEC> old;
      if constexpr (ADD) {
        if (warp == 0 && inside) old = load_stream_32<W, VEC>(row, d.wide);
      }
      Sum<VEC> sum;
      sum.clear();
      if (inside) add_rows(sum, from, begin + low, begin + high);
      parts[warp][lane] = sum.values();
      __syncthreads();
      if (warp == 0 && inside) {
#pragma unroll
        for (int w = 1; w < kDirectTokens; ++w) sum.add(parts[w][lane]);
        store(sum, row, old);
      }
      __syncthreads();
    }
    begin += all_of_it;
  }
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

template <typename Id, int R>
int launch_cluster_sort(const GradientCall& call, unsigned ctas, int passes, int digit_bits, const SortedList& list, uint8_t* named, size_t zero_bytes,
                        cudaStream_t stream) {
  const unsigned fill = zero_bytes ? ((unsigned)multiprocessor_count() + ctas - 1) / ctas * ctas : 0;  // whole clusters
  if (int status = allow_shared_memory<sort_in_cluster<Id, R>>((int)sizeof(ClusterSort<R>), "cudaFuncSetAttribute(embedding_backward sort)")) return status;
  launch_dependent_cluster(sort_in_cluster<Id, R>, dim3(ctas + fill), dim3(kSortThreads), ctas, sizeof(ClusterSort<R>), stream,
                           static_cast<const Id*>(call.tokens), (uint32_t)call.count, (uint32_t)call.vocabulary, call.padding, passes, digit_bits,
                           (uint32_t)ctas, list, named, static_cast<uint4*>(call.grad_table), zero_bytes / 16, device_status_word());
  return check_launch("embedding_backward sort launch");
}

struct ClusterShape {
  unsigned ctas = 0;  // 0: no cluster holds the tokens
  int rounds = 0;     // elements a thread
};

// The cluster that sorts `count` tokens: few elements a thread and many CTAs (65536 tokens: 24 us with 16 CTAs, 35 us with eight of
// twice the elements).  65536 tokens at most, half as many on a device that cannot hold clusters of 16.
template <typename Id> ClusterShape cluster_for(uint32_t count) {
  const auto ctas = [count](uint32_t rounds) {  // a power of two
    unsigned n = 1;
    while (n < 32 && n * rounds * kSortThreads < count) n *= 2;
    return n;
  };
  const unsigned one = ctas(1), two = ctas(2), four = ctas(4);
  if (one <= 8 || (one == 16 && sixteen_fit<sort_in_cluster<Id, 1>>(kSortThreads, sizeof(ClusterSort<1>)))) return {one, 1};
  if (two <= 8 || (two == 16 && sixteen_fit<sort_in_cluster<Id, 2>>(kSortThreads, sizeof(ClusterSort<2>)))) return {two, 2};
  if (four <= 8 || (four == 16 && sixteen_fit<sort_in_cluster<Id, 4>>(kSortThreads, sizeof(ClusterSort<4>)))) return {four, 4};
  return {};
}

// Sorts the call's tokens into `list`, in `cluster` where there is one.  `spare`: as much again, for the passes between, and
// `counts`, where there is none.
template <typename Id>
int sort_tokens(const GradientCall& call, const ClusterShape& cluster, const SortedList& list, const SortedList& spare, uint32_t* counts,
                uint8_t* named, size_t zero_bytes, cudaStream_t stream) {
  const uint32_t count = (uint32_t)call.count, vocabulary = (uint32_t)call.vocabulary;
  int bits = 1;  // of the keys 0 .. vocabulary
  while (((unsigned long long)call.vocabulary >> bits) != 0) ++bits;
  const int passes = (bits + kDigitBits - 1) / kDigitBits, digit_bits = (bits + passes - 1) / passes;
  if (cluster.rounds == 1) return launch_cluster_sort<Id, 1>(call, cluster.ctas, passes, digit_bits, list, named, zero_bytes, stream);
  if (cluster.rounds == 2) return launch_cluster_sort<Id, 2>(call, cluster.ctas, passes, digit_bits, list, named, zero_bytes, stream);
  if (cluster.rounds == 4) return launch_cluster_sort<Id, 4>(call, cluster.ctas, passes, digit_bits, list, named, zero_bytes, stream);
  const Id* tokens = static_cast<const Id*>(call.tokens);
  const int tiles = (int)((call.count + kTile - 1) / kTile);
  const uint32_t mask = (1u << digit_bits) - 1;
  // the last pass writes `list`: with an even number of passes the first one writes the spare one
  for (int pass = 0; pass < passes; ++pass) {
    const bool to_list = (passes - 1 - pass) % 2 == 0;
    const SortedList &to = to_list ? list : spare, &from = to_list ? spare : list;
    const uint32_t *keys_from = from.keys, *order_from = from.order;
    const int shift = pass * digit_bits, last = pass + 1 == passes;
    if (pass == 0) {
      launch_dependent(count_digits<Id, true>, dim3(tiles), dim3(kSortThreads), 0, stream, tokens, keys_from, count, vocabulary, call.padding,
                       shift, mask, counts, named, device_status_word());
      if (int status = check_launch("embedding_backward count launch")) return status;
      launch_dependent(scatter_digits<Id, true>, dim3(tiles), dim3(kSortThreads), 0, stream, tokens, keys_from, order_from, count, vocabulary,
                       call.padding, shift, mask, static_cast<const uint32_t*>(counts), tiles, to, last);
    } else {
      launch_dependent(count_digits<Id, false>, dim3(tiles), dim3(kSortThreads), 0, stream, tokens, keys_from, count, vocabulary, call.padding,
                       shift, mask, counts, static_cast<uint8_t*>(nullptr), static_cast<int*>(nullptr));
      if (int status = check_launch("embedding_backward count launch")) return status;
      launch_dependent(scatter_digits<Id, false>, dim3(tiles), dim3(kSortThreads), 0, stream, tokens, keys_from, order_from, count, vocabulary,
                       call.padding, shift, mask, static_cast<const uint32_t*>(counts), tiles, to, last);
    }
    if (int status = check_launch("embedding_backward scatter launch")) return status;
  }
  return BB200_OK;
}

constexpr size_t kMostFillRows = 256, kFillBytes = 65536;  // rows, and about as many bytes, for a CTA to fill

// CTAs of sum_few that do not only fill.
template <int VEC> size_t few_sum_blocks(const GradientCall& call) {
  return (call.count + kDirectTokens - 1) / kDirectTokens * ((call.hidden / VEC + 31) / 32);
}

template <typename G, typename W, int VEC, bool ADD> int few(const GradientCall& call, bool wide_tokens, cudaStream_t stream) {
  Direct d = {};
  d.tokens = call.tokens;
  d.count = (uint32_t)call.count;
  d.vocabulary = (uint32_t)call.vocabulary;
  d.padding = call.padding;
  d.steps = (int)(call.hidden / VEC);
  d.wide_tokens = wide_tokens;
  d.wide = aligned32(call.grad_out) && aligned32(call.grad_table);
  d.status_word = device_status_word();
  d.sum_blocks = (uint32_t)few_sum_blocks<VEC>(call);
  d.column_tiles = d.sum_blocks / ((d.count + kDirectTokens - 1) / kDirectTokens);
  const size_t fill_rows = kFillBytes / (call.hidden * sizeof(W));
  d.fill_rows = (uint32_t)(fill_rows < 1 ? 1 : fill_rows > kMostFillRows ? kMostFillRows : fill_rows);
  const uint32_t fill_blocks = ADD ? 0 : (d.vocabulary + d.fill_rows - 1) / d.fill_rows;
  launch_dependent(sum_few<G, W, VEC, ADD>, dim3(d.sum_blocks + fill_blocks), dim3(kThreads), 0, stream, d, static_cast<const G*>(call.grad_out),
                   static_cast<W*>(call.grad_table), call.scale);
  return check_launch("embedding_backward launch");
}

template <typename G, typename W, int VEC, bool ADD> int gradient(const GradientCall& call, bool wide_tokens, cudaStream_t stream) {
  const size_t count = call.count, steps = call.hidden / VEC;
  // Few tokens of few columns: as long as the CTAs, each of which looks through all tokens, are on the SMs at once (16 to 1024
  // tokens, up to 1024 columns: 6.2 to 10.6 us against 10.3 to 16.9 us with the steps below; 1024 tokens of 2048 columns, 1024 CTAs, 18.2
  // against 14.6 us).  Its worst case loses by it: 1024 times the same token, 1024 columns, 14.3 against 11.5 us.  That shows only in the
  // tokens' values, which the host does not look at.
  if (count <= kMostDirect && few_sum_blocks<VEC>(call) <= 4 * (size_t)multiprocessor_count() && call.vocabulary <= (size_t)1 << 30)
    return few<G, W, VEC, ADD>(call, wide_tokens, stream);
  Segments s = {};
  s.count = (uint32_t)count;
  s.vocabulary = (uint32_t)call.vocabulary;
  s.steps = (int)steps;
  s.wide = aligned32(call.grad_out) && aligned32(call.grad_table);
  s.lane_bits = 2;
  while (s.lane_bits < 8 && ((size_t)1 << s.lane_bits) < steps) ++s.lane_bits;
  const size_t groups = kThreads >> s.lane_bits, columns = (steps + ((size_t)1 << s.lane_bits) - 1) >> s.lane_bits;
  // Short chunks while there are few tokens, so that the SMs have groups to run (2000 tokens of 1024 columns 17.1 us in chunks of 8, 21.1 in
  // chunks of 16; 4000 of 256 18.2 and 18.8); with more tokens long runs cross too many borders of short chunks (three rows in turn, 64
  // columns, 8192 tokens: 19.1 and 16.2 us; one row, 256 columns, 65536 tokens: 138 and 82 us), though up to 8192 spread ones would
  // still take up to 1.8 us less in chunks of 8.  About four waves of groups otherwise, and no more of them than a CTA can stage.
  const size_t resident = ((size_t)multiprocessor_count() * 1024) >> s.lane_bits;
  s.chunk_length = count <= 4096 ? 8 : 16;
  while (2 * s.chunk_length * groups <= (size_t)kStagedList && s.chunk_length < 512 && count * columns > (size_t)s.chunk_length * resident * 4)
    s.chunk_length *= 2;
  s.chunks = (uint32_t)((count + s.chunk_length - 1) / s.chunk_length);
  const ClusterShape cluster = wide_tokens ? cluster_for<int64_t>(s.count) : cluster_for<int32_t>(s.count);
  const bool spare = !cluster.ctas;
  const size_t list = round_up(count * 4), crossings = round_up((2 + (size_t)s.chunks) * 4);
  const size_t counts_bytes = spare ? round_up((count + kTile - 1) / kTile * kBins * 4) : 0, partial = round_up((size_t)s.chunks * 2 * call.hidden * 4);
  const size_t named_bytes = ADD ? 0 : round_up(call.vocabulary);
  Workspace workspace(stream);
  if (int status = workspace.take((spare ? 4 : 2) * list + crossings + counts_bytes + partial + named_bytes, "embedding_backward workspace")) return status;
  char* at = workspace.data();
  const auto next = [&at](size_t bytes) {
    char* here = at;
    at += bytes;
    return here;
  };
  SortedList sorted = {}, other = {};
  sorted.keys = reinterpret_cast<uint32_t*>(next(list));
  sorted.order = reinterpret_cast<uint32_t*>(next(list));
  sorted.crossings = other.crossings = reinterpret_cast<uint32_t*>(next(crossings));
  if (spare) {
    other.keys = reinterpret_cast<uint32_t*>(next(list));
    other.order = reinterpret_cast<uint32_t*>(next(list));
  }
  uint32_t* counts = reinterpret_cast<uint32_t*>(next(counts_bytes));
  s.partial = reinterpret_cast<float*>(next(partial));
  uint8_t* named = ADD ? nullptr : reinterpret_cast<uint8_t*>(next(named_bytes));
  if (named) {
    if (int status = check_runtime(cudaMemsetAsync(named, 0, call.vocabulary, stream), "cudaMemsetAsync(embedding_backward)")) return status;
  }
  // Rows that are filled with zeros during the sort: whole sixteens, for about as many bytes as the idle SMs write meanwhile
  // (65536 tokens take 24 us); the rows from there on are filled behind the sums.
  size_t early_rows = 0;
  if (named && !spare && aligned16(call.grad_table)) {
    const size_t most = count * 1536 / (call.hidden * sizeof(W)) / 16 * 16, all = call.vocabulary / 16 * 16;
    early_rows = most < all ? most : all;
  }
  const size_t zero_bytes = early_rows * call.hidden * sizeof(W);
  if (int status = wide_tokens ? sort_tokens<int64_t>(call, cluster, sorted, other, counts, named, zero_bytes, stream)
                               : sort_tokens<int32_t>(call, cluster, sorted, other, counts, named, zero_bytes, stream))
    return status;
  s.fill_from = (uint32_t)early_rows;
  s.keys = sorted.keys;
  s.order = sorted.order;
  s.crossings = sorted.crossings;
  W* table = static_cast<W*>(call.grad_table);
  launch_dependent(sum_chunks<G, W, VEC, ADD>, dim3((unsigned)((s.chunks + groups - 1) / groups), (unsigned)(columns < 65535 ? columns : 65535)),
                   dim3(kThreads), (2 * groups * s.chunk_length + 1) * sizeof(uint32_t), stream, s, static_cast<const G*>(call.grad_out), table,
                   call.scale);
  if (int status = check_launch("embedding_backward sum launch")) return status;
  // at most one run crosses each border between two chunks
  const size_t most_items = (size_t)(s.chunks - 1) * ((steps + 31) / 32), join_most = (size_t)multiprocessor_count() * 8;
  const unsigned join_blocks = (unsigned)(most_items < join_most ? most_items : join_most);
  const unsigned fill_blocks = named ? (unsigned)((call.vocabulary - early_rows + groups * kFillRows - 1) / (groups * kFillRows)) : 0;
  if (join_blocks + fill_blocks > 0) {
    launch_dependent(join_and_fill<W, VEC, ADD>, dim3(join_blocks + fill_blocks), dim3(kThreads), 0, stream, s, table, call.scale, join_blocks,
                     static_cast<const uint8_t*>(named));
    if (int status = check_launch("embedding_backward join launch")) return status;
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
  // columns are counted in an int that runs past the row by up to a grid's stride, 65535 * 256 steps
  if (count >= 0x7fffffffu || vocabulary >= 0x7fffffffu || hidden > (1u << 30))
    return fail(BB200_E_UNSUPPORTED_SHAPE, "%s: count and vocabulary must be below 2^31 - 1 and hidden at most 2^30", what);
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
  template <typename G, typename W, int VEC> int run() const {
    return call.accumulate ? gradient<G, W, VEC, true>(call, wide_tokens, stream) : gradient<G, W, VEC, false>(call, wide_tokens, stream);
  }
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
