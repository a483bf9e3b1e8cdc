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
// buffers of one F2 per warp, used in turn (`turn` = 0 or 1): a warp can write a buffer again only after every warp has
// passed the barrier of the other one and so has read this one.
template <int LANES> struct RowSums {
  static constexpr int kWarps = LANES <= 32 ? 1 : LANES / 32;
  F2 buffer[2][kWarps < 2 ? 2 : kWarps];
};

template <int LANES> __device__ __forceinline__ void row_barrier(int barrier) {
  if constexpr (LANES <= 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(LANES) : "memory");
}

template <int LANES> __device__ __forceinline__ float row_sum(float a, RowSums<LANES>* scratch, int& turn, int barrier) {
#pragma unroll
  for (int offset = (LANES < 32 ? LANES : 32) / 2; offset > 0; offset >>= 1) a += __shfl_xor_sync(0xffffffffu, a, offset);
  if constexpr (LANES > 32) {
    constexpr int WARPS = LANES / 32;
    float* buffer = reinterpret_cast<float*>(scratch->buffer[turn]);
    if ((threadIdx.x & 31) == 0) buffer[(threadIdx.x / 32) % WARPS] = a;
    row_barrier<LANES>(barrier);
    a = buffer[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) a += buffer[w];
    turn ^= 1;
  }
  return a;
}

// Two sums at once.  In a whole warp the first exchange leaves one sum in each half-warp, which halves the shuffles.
template <int LANES> __device__ __forceinline__ void row_sums(float& a, float& b, RowSums<LANES>* scratch, int& turn, int barrier) {
  if constexpr (LANES < 32) {
#pragma unroll
    for (int offset = LANES / 2; offset > 0; offset >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, offset);
      b += __shfl_xor_sync(0xffffffffu, b, offset);
    }
  } else {
    const int lane = threadIdx.x & 31;
    const bool upper = lane & 16;
    float kept = upper ? b : a;
    kept += __shfl_xor_sync(0xffffffffu, upper ? a : b, 16);
#pragma unroll
    for (int offset = 8; offset > 0; offset >>= 1) kept += __shfl_xor_sync(0xffffffffu, kept, offset);
    if constexpr (LANES == 32) {
      a = __shfl_sync(0xffffffffu, kept, 0);
      b = __shfl_sync(0xffffffffu, kept, 16);
    } else {
      constexpr int WARPS = LANES / 32;
      F2* buffer = scratch->buffer[turn];
      if ((lane & 15) == 0) reinterpret_cast<float*>(buffer + (threadIdx.x / 32) % WARPS)[lane >> 4] = kept;
      row_barrier<LANES>(barrier);
      F2 sum = buffer[0];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) sum = sum + buffer[w];
      split(sum, a, b);
      turn ^= 1;
    }
  }
}

// ---- the rows of TENSORS matrices, copied ahead --------------------------------------------------------------------------
// THREADS threads in groups of LANES; a group walks its rows, and the next rows' bytes are on their way to shared memory
// while one is worked on.  Both forms give a thread the same columns of every row, as PAIRS pairs, so it can keep what
// belongs to columns (weights, sums over rows) in registers.  Bytes in flight per SM decide the depth: about 80 KB cover
// the latency of HBM3e at its bandwidth (44 B/ns per SM, 1 to 2 us under load).
constexpr int kRowThreads = 512;

template <int STAGE_BYTES> constexpr int stages_for() {
  constexpr int wanted = 1 + (80 * 1024 + STAGE_BYTES - 1) / STAGE_BYTES;
  constexpr int most = 200 * 1024 / STAGE_BYTES;
  return wanted > 6 ? 6 : wanted < 3 ? (most < 3 ? most : 3) : (wanted > most ? most : wanted);
}

// Rows of whole 16-byte vectors, 16-byte aligned.  Thread `lane` of a group owns the vectors lane, lane + LANES, ...; it
// copies and reads them itself, so it waits for nothing but its own copies.
template <typename T, int LANES_, int VPT, int TENSORS> struct VectorRows {
  static constexpr bool kWholePairs = true;  // a pair is inside the row or past its end, never half
  static constexpr int LANES = LANES_, VEC = 16 / sizeof(T), PAIRS = VPT * VEC / 2, GROUPS = kRowThreads / LANES;
  static constexpr int kSlot = kRowThreads * VPT * 16, kStage = kSlot * TENSORS, STAGES = stages_for<kStage>(), kBytes = kStage * STAGES;

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
    return shared + at * kStage + tensor * kSlot + (j * kRowThreads + threadIdx.x) * 16;
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
  __device__ __forceinline__ void start(size_t row, size_t stride) {
#pragma unroll
    for (int at = 0; at < STAGES - 1; ++at) fetch(row + at * stride, at);
  }
  // The row at hand has arrived, and a later one is on its way into the slots of the row before it.
  __device__ __forceinline__ void arrive(size_t row, size_t stride) {
    fetch(row + (STAGES - 1) * stride, stage == 0 ? STAGES - 1 : stage - 1);
    copy_async_wait<STAGES - 1>();
  }
  __device__ __forceinline__ void next() { stage = stage + 1 == STAGES ? 0 : stage + 1; }

  // The row's pairs of one tensor; zeros past the row's end.
  __device__ __forceinline__ void get(int tensor, F2 (&out)[PAIRS]) const {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      if (has(j)) {
        const Pack<T, VEC> v = *reinterpret_cast<const Pack<T, VEC>*>(slot(stage, tensor, j));
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) out[j * (VEC / 2) + i] = Pairs<T>::get(v, i);
      } else {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) out[j * (VEC / 2) + i] = both(0.0f);
      }
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
};

// Rows of any width in tensors whose first element is 16-byte aligned: the group copies the 16-byte windows that cover the
// row (the last one of a tensor only as far as the tensor goes), and thread `lane` owns the columns lane, lane + LANES, ...
// The copies are other threads' too, so the group meets at its barrier before it reads a row.
template <typename T, int LANES_, int COLUMNS, int TENSORS> struct ShiftedRows {
  static constexpr bool kWholePairs = false;
  static constexpr int LANES = LANES_, PAIRS = COLUMNS / 2, GROUPS = kRowThreads / LANES;
  static constexpr int kSlot = LANES * COLUMNS * (int)sizeof(T) + 32, kStage = kSlot * GROUPS * TENSORS, STAGES = stages_for<kStage>(),
                       kBytes = kStage * STAGES;

  unsigned char* shared;
  const T* tensors[TENSORS];
  size_t rows;
  int hidden, lane, barrier, stage, shift;

  __device__ __forceinline__ ShiftedRows(unsigned char* memory, const T* const (&sources)[TENSORS], size_t rows_, int hidden_, int lane_, int group)
      : shared(memory + group * (kSlot * TENSORS)), rows(rows_), hidden(hidden_), lane(lane_), barrier(group + 1), stage(0), shift(0) {
#pragma unroll
    for (int t = 0; t < TENSORS; ++t) tensors[t] = sources[t];
  }
  __device__ __forceinline__ unsigned char* slot(int at, int tensor) const { return shared + at * kStage + tensor * kSlot; }
  __device__ __forceinline__ void fetch(size_t row, int at) {
    if (row < rows) {
      const size_t begin = row * (size_t)hidden * sizeof(T), window = begin & ~(size_t)15, end = rows * (size_t)hidden * sizeof(T);
      const int vectors = (int)((begin - window + (size_t)hidden * sizeof(T) + 15) / 16);
      for (int v = lane; v < vectors; v += LANES) {
        const size_t from = window + (size_t)v * 16;
        const uint32_t bytes = end - from < 16 ? (uint32_t)(end - from) : 16;
#pragma unroll
        for (int t = 0; t < TENSORS; ++t) copy_async_part(slot(at, t) + v * 16, reinterpret_cast<const unsigned char*>(tensors[t]) + from, bytes);
      }
    }
    copy_async_commit();
  }
  __device__ __forceinline__ void start(size_t row, size_t stride) {
#pragma unroll
    for (int at = 0; at < STAGES - 1; ++at) fetch(row + at * stride, at);
  }
  __device__ __forceinline__ void arrive(size_t row, size_t stride) {
    copy_async_wait<STAGES - 2>();
    row_barrier<LANES>(barrier);  // everyone's copies have landed, and everyone is done with the row before
    fetch(row + (STAGES - 1) * stride, stage == 0 ? STAGES - 1 : stage - 1);
    shift = (int)((row * (size_t)hidden * sizeof(T)) & 15) / (int)sizeof(T);
  }
  __device__ __forceinline__ void next() { stage = stage + 1 == STAGES ? 0 : stage + 1; }

  __device__ __forceinline__ void get(int tensor, F2 (&out)[PAIRS]) const {
    const T* row = reinterpret_cast<const T*>(slot(stage, tensor)) + shift;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      const int low = column(i, 0), high = column(i, 1);
      out[i] = make_f2(low < hidden ? Conv<float, T>::widen(row[low]) : 0.0f, high < hidden ? Conv<float, T>::widen(row[high]) : 0.0f);
    }
  }
  __device__ __forceinline__ void put(T* row, const F2 (&in)[PAIRS]) const {
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      float low, high;
      split(in[i], low, high);
      if (column(i, 0) < hidden) row[column(i, 0)] = Conv<float, T>::narrow(low);
      if (column(i, 1) < hidden) row[column(i, 1)] = Conv<float, T>::narrow(high);
    }
  }
  __device__ __forceinline__ int column(int pair, int half) const { return lane + (2 * pair + half) * LANES; }
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
