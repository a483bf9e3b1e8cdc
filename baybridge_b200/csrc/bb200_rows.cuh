// bb200_rows.cuh — building blocks of the kernels that walk the rows of a matrix: pairs of f32, copies ahead into
// shared memory, sums over the threads that share a row.
#pragma once
#include <stdint.h>

#include "bb200_elementwise.cuh"

namespace bb200 {

// ---- two f32 at a time ------------------------------------------------------------------------------------------
// sm_100a adds, multiplies and fuses two f32 held in a register pair with one instruction.  The row kernels are bound by
// instruction issue before they are bound by memory when written element by element (LayerNorm backward: 31 warp
// instructions per element-and-lane, 4.4 TB/s, issue slots 68 % used), so their arithmetic runs in pairs.
struct F2 {
  unsigned long long bits;
};
__device__ __forceinline__ F2 make_f2(float low, float high) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.bits) : "f"(low), "f"(high));
  return r;
}
__device__ __forceinline__ F2 both(float v) { return make_f2(v, v); }
__device__ __forceinline__ void split(F2 v, float& low, float& high) { asm("mov.b64 {%0, %1}, %2;" : "=f"(low), "=f"(high) : "l"(v.bits)); }
__device__ __forceinline__ float total(F2 v) {
  float low, high;
  split(v, low, high);
  return low + high;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return r;
}

// Elements 2 i and 2 i + 1 of a vector, widened exactly; and back, one rounding each.
template <typename T> struct Pairs;
template <> struct Pairs<float> {
  template <int VEC> static __device__ __forceinline__ F2 get(const Pack<float, VEC>& p, int i) { return make_f2(p.v[2 * i], p.v[2 * i + 1]); }
  template <int VEC> static __device__ __forceinline__ void set(Pack<float, VEC>& p, int i, F2 v) { split(v, p.v[2 * i], p.v[2 * i + 1]); }
};
template <> struct Pairs<__nv_bfloat16> {
  template <int VEC> static __device__ __forceinline__ F2 get(const Pack<__nv_bfloat16, VEC>& p, int i) {
    const uint32_t word = reinterpret_cast<const uint32_t*>(&p)[i];  // a bf16 is the upper half of the f32 of its value
    return make_f2(__uint_as_float(word << 16), __uint_as_float(word & 0xffff0000u));
  }
  template <int VEC> static __device__ __forceinline__ void set(Pack<__nv_bfloat16, VEC>& p, int i, F2 v) {
    float low, high;
    split(v, low, high);
    reinterpret_cast<__nv_bfloat162*>(&p)[i] = __floats2bfloat162_rn(low, high);
  }
};
template <> struct Pairs<__half> {
  template <int VEC> static __device__ __forceinline__ F2 get(const Pack<__half, VEC>& p, int i) {
    const float2 v = __half22float2(reinterpret_cast<const __half2*>(&p)[i]);
    return make_f2(v.x, v.y);
  }
  template <int VEC> static __device__ __forceinline__ void set(Pack<__half, VEC>& p, int i, F2 v) {
    float low, high;
    split(v, low, high);
    reinterpret_cast<__half2*>(&p)[i] = __floats2half2_rn(low, high);
  }
};

// ---- 32 bytes a thread ---------------------------------------------------------------------------------------------
// Vectors of 32 bytes (eight f32 beside eight 16-bit values) as one access where `aligned` (to 32 bytes) says so, as two of
// 16 otherwise.  Two 16-byte accesses 32 bytes apart from the neighbouring thread's touch every sector twice: AdamW over
// 400 M parameters with masters 1912 us with them, 1639 us with these.
template <typename T, int VEC> __device__ __forceinline__ Pack<T, VEC> load_stream_32(const T* p, bool aligned) {
  if constexpr (sizeof(T) * VEC == 32) {
    if (aligned) {
      Pack<T, VEC> r;
      uint32_t* w = reinterpret_cast<uint32_t*>(&r);
      asm volatile("ld.global.cs.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(p)
                   : "memory");
      return r;
    }
  }
  return load_stream<T, VEC>(p);
}
template <typename T, int VEC> __device__ __forceinline__ void store_stream_32(T* p, const Pack<T, VEC>& v, bool aligned) {
  if constexpr (sizeof(T) * VEC == 32) {
    if (aligned) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
      asm volatile("st.global.cs.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                   "r"(w[6]), "r"(w[7]), "l"(p)
                   : "memory");
      return;
    }
  }
  store_stream<T, VEC>(p, v);
}

// ---- clusters ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// The address of CTA `rank`'s copy of a shared variable of this CTA.
__device__ __forceinline__ uint32_t in_cta(const void* shared, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(shared)), "r"(rank));
  return a;
}

// ---- copies ahead ------------------------------------------------------------------------------------------------
// 16 bytes from global to shared memory, both 16-byte aligned, of which `bytes` are read and the rest become zeros.
__device__ __forceinline__ void copy_async_16(void* shared, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(shared)), "l"(global) : "memory");
}
__device__ __forceinline__ void copy_async_part(void* shared, const void* global, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(shared)), "l"(global), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ---- sums over the LANES threads that share a row ---------------------------------------------------------------------
// LANES is a power of two; up to 32 they are neighbours in a warp, above they are whole warps that meet at named barrier
// `barrier`.  Every thread of the group receives the sums, the same bits in each.  `scratch`: the group's own, two
// buffers of COUNT floats per warp, used in turn (`turn` = 0 or 1): a warp can write a buffer again only after every warp
// has passed the barrier of the other one and so has read this one.
template <int LANES, int COUNT> struct alignas(16) RowSums {
  static constexpr int kWarps = LANES <= 32 ? 1 : LANES / 32;
  float buffer[2][kWarps][COUNT];
};

template <int LANES> __device__ __forceinline__ void row_barrier(int barrier) {
  if constexpr (LANES <= 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(LANES) : "memory");
}

// COUNT (1, 2 or 4) sums at once.  In a whole warp the first exchanges leave a part of the sums to each half or quarter
// of the lanes, so four sums cost six shuffles and not twenty.
template <int LANES, int COUNT>
__device__ __forceinline__ void row_sums(float (&v)[COUNT], RowSums<LANES, COUNT>* scratch, int& turn, int barrier) {
  if constexpr (LANES < 32) {
#pragma unroll
    for (int offset = LANES / 2; offset > 0; offset >>= 1) {
#pragma unroll
      for (int k = 0; k < COUNT; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], offset);
    }
  } else {
    const int lane = threadIdx.x & 31;
    float kept[COUNT];
#pragma unroll
    for (int k = 0; k < COUNT; ++k) kept[k] = v[k];
    int offset = 16;
#pragma unroll
    for (int n = COUNT; n > 1; n >>= 1, offset >>= 1) {
      const bool upper = lane & offset;
#pragma unroll
      for (int k = 0; k < n / 2; ++k) {
        const float sent = upper ? kept[k] : kept[k + n / 2];
        kept[k] = (upper ? kept[k + n / 2] : kept[k]) + __shfl_xor_sync(0xffffffffu, sent, offset);
      }
    }
    float sum = kept[0];
#pragma unroll
    for (int o = 32 / COUNT / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    // lane k * (32 / COUNT) now holds sum k
    constexpr int kEach = 32 / COUNT;
    if constexpr (LANES == 32) {
#pragma unroll
      for (int k = 0; k < COUNT; ++k) v[k] = COUNT == 1 ? sum : __shfl_sync(0xffffffffu, sum, k * kEach);
    } else {
      constexpr int WARPS = LANES / 32;
      float(&buffer)[WARPS][COUNT] = scratch->buffer[turn];
      if (lane % kEach == 0) buffer[(threadIdx.x / 32) % WARPS][lane / kEach] = sum;
      row_barrier<LANES>(barrier);
      static_assert(WARPS * COUNT <= 32, "one value to a lane");
      sum = lane < WARPS * COUNT ? (&buffer[0][0])[lane] : 0.0f;  // lane w * COUNT + k: warp w's part of sum k
#pragma unroll
      for (int o = WARPS * COUNT / 2; o >= COUNT; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
      for (int k = 0; k < COUNT; ++k) v[k] = __shfl_sync(0xffffffffu, sum, k);
      turn ^= 1;
    }
  }
}

// ---- the rows of TENSORS matrices, copied ahead --------------------------------------------------------------------------
// THREADS threads in groups of LANES; a group walks its rows, and the next rows' bytes are on their way to shared memory
// while it works on one.  Both forms give a thread the same columns of every row, as PAIRS pairs, so it can keep what
// belongs to columns (weights, sums over rows) in registers.  Bytes in flight per SM decide the depth:
// about 56 KB cover the latency of HBM3e at its bandwidth (44 B/ns per SM, 1.3 us).  More only lengthens the queues: with
// 80 KB the gradient of 65536 x 4096 took 275 us instead of 261, the forward of 65536 x 8192 371 instead of 344.
template <int STAGE_BYTES, int MOST_BYTES> constexpr int stages_for() {
  constexpr int wanted = 1 + (56 * 1024 + STAGE_BYTES - 1) / STAGE_BYTES, most = MOST_BYTES / STAGE_BYTES, within = wanted > 6 ? 6 : wanted < 3 ? 3 : wanted;
  static_assert(most >= 2, "two stages have to fit");
  return within < most ? within : most;
}

// Rows of whole 16-byte vectors, 16-byte aligned.  Thread `lane` of a group owns the vectors lane, lane + LANES, ...; it
// copies and reads them itself, so it waits for nothing but its own copies.  FULL: the rows fill all of them.
template <typename T, int THREADS_, int LANES_, int VPT, int TENSORS, int MOST_BYTES, bool FULL = false> struct VectorRows {
  static constexpr int THREADS = THREADS_, LANES = LANES_, VEC = 16 / sizeof(T), PAIRS = VPT * VEC / 2, GROUPS = THREADS / LANES;
  static constexpr int kSlot = THREADS * VPT * 16, kStage = kSlot * TENSORS, STAGES = stages_for<kStage, MOST_BYTES>(), kBytes = kStage * STAGES;

  unsigned char* shared;
  const T* tensors[TENSORS];
  size_t rows;
  int hidden, lane, stage;

  __device__ __forceinline__ VectorRows(unsigned char* memory, const T* const (&sources)[TENSORS], size_t rows_, int hidden_, int lane_, int)
      : shared(memory), rows(rows_), hidden(hidden_), lane(lane_), stage(0) {
#pragma unroll
    for (int t = 0; t < TENSORS; ++t) tensors[t] = sources[t];
  }
  __device__ __forceinline__ unsigned char* slot(int at, int tensor, int j) const {
    return shared + at * kStage + tensor * kSlot + (j * THREADS + threadIdx.x) * 16;
  }
  __device__ __forceinline__ int vector(int j) const { return lane + j * LANES; }
  __device__ __forceinline__ bool has(int j) const { return vector(j) * VEC < hidden; }
  __device__ __forceinline__ void fetch(size_t row, int at) {
    if (row < rows) {
      const size_t offset = row * (size_t)hidden;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        if (has(j)) {
#pragma unroll
          for (int t = 0; t < TENSORS; ++t) copy_async_16(slot(at, t, j), tensors[t] + offset + vector(j) * VEC);
        }
      }
    }
    copy_async_commit();
  }
  __device__ __forceinline__ void start(size_t row, size_t stride, int) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      if (!has(j)) {  // slots past the row's end are never copied to: zeros, so rows are read without a question
        for (int at = 0; at < STAGES * TENSORS; ++at)
          *reinterpret_cast<uint4*>(shared + at * kSlot + (j * THREADS + threadIdx.x) * 16) = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int at = 0; at < STAGES - 1; ++at) fetch(row + at * stride, at);
  }
  // The row has arrived, and a later one is on its way into the slots of the row before it.
  __device__ __forceinline__ void arrive(size_t row, size_t stride) {
    fetch(row + (STAGES - 1) * stride, stage == 0 ? STAGES - 1 : stage - 1);
    copy_async_wait<STAGES - 1>();
  }
  __device__ __forceinline__ void before_sums() {}
  __device__ __forceinline__ void after_sums(size_t, size_t) {}
  __device__ __forceinline__ void next() { stage = stage + 1 == STAGES ? 0 : stage + 1; }

  // The row's pairs of one tensor; zeros past the row's end.
  __device__ __forceinline__ void get(int tensor, F2 (&out)[PAIRS]) const {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const Pack<T, VEC> v = *reinterpret_cast<const Pack<T, VEC>*>(slot(stage, tensor, j));
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) out[j * (VEC / 2) + i] = Pairs<T>::get(v, i);
    }
  }
  __device__ __forceinline__ void put(T* row, const F2 (&in)[PAIRS]) const {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      if (has(j)) {
        Pack<T, VEC> v;
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) Pairs<T>::set(v, i, in[j * (VEC / 2) + i]);
        store_stream<T, VEC>(row + vector(j) * VEC, v);
      }
    }
  }
  __device__ __forceinline__ int column(int pair, int half) const { return vector(pair / (VEC / 2)) * VEC + pair % (VEC / 2) * 2 + half; }
  // `v` with what lies past the row's end left out
  __device__ __forceinline__ F2 inside(int pair, F2 v) const { return F2{has(pair / (VEC / 2)) ? v.bits : 0ull}; }
  // `v`, which all columns of a row share, or zero past the row's end: one question a vector
  static constexpr bool kMasked = true;
  __device__ __forceinline__ F2 where_inside(int pair, float v) const { return both(FULL || has(pair / (VEC / 2)) ? v : 0.0f); }
};

// Rows of any width in tensors whose first element is 16-byte aligned: the group copies the 16-byte windows that cover the
// row (the last one of a tensor only as far as the tensor goes), and thread `lane` owns the columns lane, lane + LANES, ...
// The copies are other threads' too.  One barrier a row does for that: a thread waits for its copies of the next row before
// it meets the others at the barrier of the row's (first) sums, and copies into the slots of the row before after it.
// SURE: so many of a thread's columns lie inside every row that this form is used for (LANES * SURE <= hidden), and are
// not asked about.
template <typename T, int THREADS_, int LANES_, int COLUMNS, int SURE, int TENSORS, int MOST_BYTES> struct ShiftedRows {
  static constexpr int THREADS = THREADS_, LANES = LANES_, PAIRS = COLUMNS / 2, GROUPS = THREADS / LANES;
  static constexpr int kSlot = LANES * COLUMNS * (int)sizeof(T) + 32, kGroup = kSlot * TENSORS, kStage = kGroup * GROUPS,
                       STAGES = stages_for<kStage, MOST_BYTES>(), kBytes = kStage * STAGES, kWindows = COLUMNS * (int)sizeof(T) / 16 + 1;
  static_assert(STAGES >= 3, "the next row's copies are waited for a row ahead");

  unsigned char* shared;
  const unsigned char* tensors[TENSORS];
  size_t rows;
  int hidden, lane, stage;
  uint32_t shift;  // bytes from the window's start to the row's, of the row at hand

  __device__ __forceinline__ ShiftedRows(unsigned char* memory, const T* const (&sources)[TENSORS], size_t rows_, int hidden_, int lane_, int group)
      : shared(memory + group * kGroup), rows(rows_), hidden(hidden_), lane(lane_), stage(0), shift(0) {
#pragma unroll
    for (int t = 0; t < TENSORS; ++t) tensors[t] = reinterpret_cast<const unsigned char*>(sources[t]);
  }
  __device__ __forceinline__ void fetch(size_t row, int at) {
    if (row < rows) {
      const uint32_t row_bytes = (uint32_t)hidden * (uint32_t)sizeof(T);
      const size_t begin = row * row_bytes;
      const uint32_t inside = (uint32_t)begin & 15u, bytes = inside + row_bytes, windows = (bytes + 15) / 16;
      const size_t window_end = begin - inside + windows * 16u, end = rows * row_bytes;
      const uint32_t tail = window_end > end ? 16u - (uint32_t)(window_end - end) : 16u;  // of the last window, nothing behind the tensor
      const size_t from = begin - inside + (size_t)lane * 16;
      unsigned char* to = shared + at * kStage + lane * 16;
#pragma unroll
      for (int w = 0; w < kWindows; ++w) {
        const uint32_t v = lane + w * LANES;
        if (v < windows) {
          const uint32_t size = v + 1 == windows ? tail : 16u;
#pragma unroll
          for (int t = 0; t < TENSORS; ++t) copy_async_part(to + t * kSlot + w * (LANES * 16), tensors[t] + from + w * (LANES * 16), size);
        }
      }
    }
    copy_async_commit();
  }
  __device__ __forceinline__ void start(size_t row, size_t stride, int barrier) {
#pragma unroll
    for (int at = 0; at < STAGES - 1; ++at) fetch(row + at * stride, at);
    copy_async_wait<STAGES - 2>();
    row_barrier<LANES>(barrier);
  }
  __device__ __forceinline__ void arrive(size_t row, size_t) { shift = (uint32_t)(row * ((uint32_t)hidden * (uint32_t)sizeof(T))) & 15u; }
  __device__ __forceinline__ void before_sums() {
    copy_async_wait<STAGES - 3>();
    if constexpr (LANES <= 32) __syncwarp();  // otherwise the sums' own barrier
  }
  __device__ __forceinline__ void after_sums(size_t row, size_t stride) { fetch(row + (STAGES - 1) * stride, stage == 0 ? STAGES - 1 : stage - 1); }
  __device__ __forceinline__ void next() { stage = stage + 1 == STAGES ? 0 : stage + 1; }

  __device__ __forceinline__ void get(int tensor, F2 (&out)[PAIRS]) const {
    const T* row = reinterpret_cast<const T*>(shared + stage * kStage + tensor * kSlot + shift) + lane;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
      out[i] = make_f2(has(2 * i) ? Conv<float, T>::widen(row[2 * i * LANES]) : 0.0f, has(2 * i + 1) ? Conv<float, T>::widen(row[(2 * i + 1) * LANES]) : 0.0f);
  }
  __device__ __forceinline__ void put(T* row, const F2 (&in)[PAIRS]) const {
    row += lane;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      Pack<T, 2> v;  // rounded in pairs: one instruction
      Pairs<T>::set(v, 0, in[i]);
      if (has(2 * i)) row[2 * i * LANES] = v.v[0];
      if (has(2 * i + 1)) row[(2 * i + 1) * LANES] = v.v[1];
    }
  }
  __device__ __forceinline__ int column(int pair, int half) const { return lane + (2 * pair + half) * LANES; }
  __device__ __forceinline__ bool has(int k) const { return k < SURE || lane + k * LANES < hidden; }
  // `v` with what lies past the row's end left out
  __device__ __forceinline__ F2 inside(int pair, F2 v) const {
    if (2 * pair + 1 < SURE) return v;
    float low, high;
    split(v, low, high);
    return make_f2(has(2 * pair) ? low : 0.0f, has(2 * pair + 1) ? high : 0.0f);
  }
  // would be a question for every column here (8191 x 1001: 3 % of the gradient's time): `v` stays as it is
  static constexpr bool kMasked = false;
  __device__ __forceinline__ F2 where_inside(int, float v) const { return both(v); }
};

// A vector over the columns, of the rows' type or f32: its pairs for this thread, zeros past the row's end.
template <typename T, typename Rows>
__device__ __forceinline__ void column_pairs(const Rows& rows, const void* vector, bool wide, F2 (&out)[Rows::PAIRS]) {
#pragma unroll
  for (int i = 0; i < Rows::PAIRS; ++i) {
    float v[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int c = rows.column(i, half);
      v[half] = !vector || c >= rows.hidden ? 0.0f : wide ? static_cast<const float*>(vector)[c] : Conv<float, T>::widen(static_cast<const T*>(vector)[c]);
    }
    out[i] = make_f2(v[0], v[1]);
  }
}

}  // namespace bb200
