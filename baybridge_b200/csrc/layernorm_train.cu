// layernorm_train.cu — LayerNorm for training, sm_100a: the forward pass that keeps its statistics, and the backward pass.
//
//   forward:   s = x (+ residual);  out = (s - mean) * rstd * weight + bias;  mean, rstd = 1 / sqrt(variance + eps) per row
//   backward:  n = (x - mean) * rstd;  g = grad_out * weight
//              grad_x      = rstd * (g - mean(g) - n * mean(g * n))  (+ grad_resid)
//              grad_weight = sum over rows of grad_out * n,   grad_bias = sum over rows of grad_out
//
// Both are bound by HBM bytes: forward reads x (and residual) once and writes out (and out_resid) once, backward reads
// grad_out and x (and grad_resid) once and writes grad_x once; weights, statistics and the two column sums are small.
// Everything is computed in fp32 and rounded once per output; the variance is the mean of squared differences from the
// mean (two passes over registers), so a large mean costs no precision.  The column sums are split over CTAs, each of
// which keeps its share in registers over all its rows, and joined by a second kernel in a fixed order: no atomics, the
// same call gives the same bits.
#include "bb200_elementwise.cuh"
#include "bb200_internal.h"

namespace bb200 {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) v += __shfl_xor_sync(0xffffffffu, v, offset);
  return v;
}

// Sum over the WARPS warps that share a row; every thread receives it.  `scratch`: one float per warp of the CTA.
template <int WARPS> __device__ __forceinline__ float row_sum(float v, float* scratch) {
  v = warp_sum(v);
  if constexpr (WARPS == 1) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();  // scratch may still be read from the previous sum
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  return warp_sum(lane < WARPS ? scratch[lane] : 0.0f);
}

template <typename T, int VEC> __device__ __forceinline__ void widen(const Pack<T, VEC>& in, float (&out)[VEC]) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) out[e] = Conv<float, T>::widen(in.v[e]);
}

// ---- forward ---------------------------------------------------------------------------------------------------------
template <typename T, typename W> struct Forward {
  const T* x;
  const T* residual;  // null: none, and out_resid is null too
  const W* weight;
  const W* bias;  // null: none
  T* out;
  T* out_resid;
  float* mean;
  float* rstd;
  size_t rows;
  int hidden;
  float epsilon;
};

// WARPS warps own a row, ROWS rows to a CTA (ROWS > 1 only with WARPS = 1); the row stays in registers.
template <typename T, typename W, int WARPS, int ROWS, int VPT, bool RESIDUAL>
__global__ void __launch_bounds__(WARPS * ROWS * 32)
norm_rows(const __grid_constant__ Forward<T, W> p) {
  static_assert(WARPS == 1 || ROWS == 1, "one row to a CTA where several warps share it");
  constexpr int VEC = 16 / sizeof(T), LANES = WARPS * 32;
  __shared__ float scratch[32];
  dependent_launch_prologue();
  const int lane = WARPS == 1 ? threadIdx.x & 31 : threadIdx.x;
  const size_t row = (size_t)blockIdx.x * ROWS + (ROWS == 1 ? 0 : threadIdx.x >> 5);
  if (row >= p.rows) return;
  const size_t offset = row * (size_t)p.hidden;
  const int nvec = p.hidden / VEC;
  float s[VPT][VEC];
  float sum = 0.0f;
  {
    Pack<T, VEC> a[VPT], b[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int v = lane + j * LANES;
      if (v < nvec) {
        a[j] = load_stream<T, VEC>(p.x + offset + (size_t)v * VEC);
        if constexpr (RESIDUAL) b[j] = load_stream<T, VEC>(p.residual + offset + (size_t)v * VEC);
      }
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int v = lane + j * LANES;
      if (v < nvec) {
        widen<T, VEC>(a[j], s[j]);
        if constexpr (RESIDUAL) {
          Pack<T, VEC> r;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            s[j][e] += Conv<float, T>::widen(b[j].v[e]);
            r.v[e] = Conv<float, T>::narrow(s[j][e]);
          }
          store_stream<T, VEC>(p.out_resid + offset + (size_t)v * VEC, r);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum += s[j][e];
      }
    }
  }
  const float mean = row_sum<WARPS>(sum, scratch) / (float)p.hidden;
  float centred = 0.0f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    if (lane + j * LANES < nvec) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = s[j][e] - mean;
        centred = fmaf(d, d, centred);
      }
    }
  }
  const float rstd = 1.0f / sqrtf(row_sum<WARPS>(centred, scratch) / (float)p.hidden + p.epsilon);
  if (lane == 0) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int v = lane + j * LANES;
    if (v < nvec) {
      const Pack<W, VEC> w = load_shared_operand<W, VEC>(p.weight + (size_t)v * VEC);
      Pack<W, VEC> b;
      if (p.bias) b = load_shared_operand<W, VEC>(p.bias + (size_t)v * VEC);
      Pack<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        o.v[e] = Conv<float, T>::narrow(fmaf((s[j][e] - mean) * rstd, Conv<float, W>::widen(w.v[e]), p.bias ? Conv<float, W>::widen(b.v[e]) : 0.0f));
      store_stream<T, VEC>(p.out + offset + (size_t)v * VEC, o);
    }
  }
}

// Rows that are no whole number of vectors, or tensors that are not 16-byte aligned: element by element, the row kept in
// shared memory as fp32.
constexpr int kElementThreads = 256;
template <typename T, typename W>
__global__ void __launch_bounds__(kElementThreads)
norm_rows_by_element(const __grid_constant__ Forward<T, W> p) {
  extern __shared__ float row_values[];
  __shared__ float scratch[32];
  dependent_launch_prologue();
  const size_t row = blockIdx.x, offset = row * (size_t)p.hidden;
  float sum = 0.0f;
#pragma unroll 4
  for (int c = threadIdx.x; c < p.hidden; c += kElementThreads) {
    float v = Conv<float, T>::widen(p.x[offset + c]);
    if (p.residual) {
      v += Conv<float, T>::widen(p.residual[offset + c]);
      p.out_resid[offset + c] = Conv<float, T>::narrow(v);
    }
    row_values[c] = v;
    sum += v;
  }
  const float mean = row_sum<kElementThreads / 32>(sum, scratch) / (float)p.hidden;
  float centred = 0.0f;
  for (int c = threadIdx.x; c < p.hidden; c += kElementThreads) {
    const float d = row_values[c] - mean;
    centred = fmaf(d, d, centred);
  }
  const float rstd = 1.0f / sqrtf(row_sum<kElementThreads / 32>(centred, scratch) / (float)p.hidden + p.epsilon);
  if (threadIdx.x == 0) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
  for (int c = threadIdx.x; c < p.hidden; c += kElementThreads)
    p.out[offset + c] = Conv<float, T>::narrow(
        fmaf((row_values[c] - mean) * rstd, Conv<float, W>::widen(p.weight[c]), p.bias ? Conv<float, W>::widen(p.bias[c]) : 0.0f));
}

template <typename T, typename W, int WARPS, int ROWS, int VPT> int launch_norm(const Forward<T, W>& p, cudaStream_t stream) {
  const dim3 grid((unsigned)((p.rows + ROWS - 1) / ROWS)), block(WARPS * ROWS * 32);
  if (p.residual) launch_dependent(norm_rows<T, W, WARPS, ROWS, VPT, true>, grid, block, 0, stream, p);
  else launch_dependent(norm_rows<T, W, WARPS, ROWS, VPT, false>, grid, block, 0, stream, p);
  return check_launch("layernorm_forward kernel launch");
}

template <typename T, typename W> int forward(const Forward<T, W>& p, bool aligned, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  if (!aligned || p.hidden % VEC) {
    const int smem = p.hidden * (int)sizeof(float);
    if (smem > 48 * 1024) {
      if (int status = check_runtime(cudaFuncSetAttribute(norm_rows_by_element<T, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, 32768 * 4),
                                     "cudaFuncSetAttribute(layernorm_forward)"))
        return status;
    }
    launch_dependent(norm_rows_by_element<T, W>, dim3((unsigned)p.rows), dim3(kElementThreads), (size_t)smem, stream, p);
    return check_launch("layernorm_forward kernel launch");
  }
  const int nvec = p.hidden / VEC;
  // up to 128 vectors a warp holds the row by itself and no CTA-wide sum is needed; above, about two vectors a thread
  if (nvec <= 32) return launch_norm<T, W, 1, 8, 1>(p, stream);
  if (nvec <= 64) return launch_norm<T, W, 1, 8, 2>(p, stream);
  if (nvec <= 128) return launch_norm<T, W, 1, 8, 4>(p, stream);
  if (nvec <= 256) return launch_norm<T, W, 8, 1, 1>(p, stream);
  if (nvec <= 512) return launch_norm<T, W, 8, 1, 2>(p, stream);
  if (nvec <= 1024) return launch_norm<T, W, 16, 1, 2>(p, stream);
  if (nvec <= 2048) return launch_norm<T, W, 32, 1, 2>(p, stream);
  return launch_norm<T, W, 32, 1, 4>(p, stream);
}

// ---- backward --------------------------------------------------------------------------------------------------------
template <typename T, typename W> struct Backward {
  const T* grad_out;
  const T* x;
  const float* mean;
  const float* rstd;
  const W* weight;
  const T* grad_resid;  // null: none
  T* grad_x;
  float* partial;  // [CTAs][2][hidden]: the CTA's share of grad_weight and grad_bias
  size_t rows;
  int hidden;
};

__device__ __forceinline__ void copy_async_16(void* shared, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(shared)), "l"(global) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// WARPS warps own a row, GROUPS such groups to a CTA; a group walks rows `group, group + all groups, ...`.  Thread t of a
// group owns the vectors t, t + LANES, ... of every row: it copies them into its own shared-memory slots STAGES - 1 rows
// ahead (so it waits for its own copies only, no barrier), and keeps the weight's and bias's gradients of its columns
// in registers over all rows.
template <typename T, int WARPS, int GROUPS, int VPT, bool RESIDUAL> struct BackwardShape {
  static constexpr int kThreads = WARPS * GROUPS * 32, kTensors = RESIDUAL ? 3 : 2;
  static constexpr int kSlot = kThreads * VPT * 16;          // bytes of one tensor in one stage
  static constexpr int kStage = kSlot * kTensors;
  static constexpr int kStages = kStage * 4 <= 98304 ? 4 : 3;
  static constexpr int kSmem = kStage * kStages;
};

template <typename T, typename W, int WARPS, int GROUPS, int VPT, bool RESIDUAL>
__global__ void __launch_bounds__(WARPS * GROUPS * 32, WARPS * GROUPS <= 8 ? 2 : 1)
norm_backward_rows(const __grid_constant__ Backward<T, W> p) {
  using Shape = BackwardShape<T, WARPS, GROUPS, VPT, RESIDUAL>;
  constexpr int VEC = 16 / sizeof(T), LANES = WARPS * 32, STAGES = Shape::kStages;
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ float2 sums[2][GROUPS][WARPS];
  dependent_launch_prologue();
  const int group = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const int nvec = p.hidden / VEC;
  const size_t all = (size_t)gridDim.x * GROUPS;
  const float scale = 1.0f / (float)p.hidden;

  auto slot = [&](int stage, int tensor, int j) { return shared + stage * Shape::kStage + tensor * Shape::kSlot + (j * Shape::kThreads + threadIdx.x) * 16; };
  auto fetch = [&](size_t row, int stage) {
    if (row < p.rows) {
      const size_t offset = row * (size_t)p.hidden;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const int v = lane + j * LANES;
        if (v < nvec) {
          copy_async_16(slot(stage, 0, j), p.grad_out + offset + (size_t)v * VEC);
          copy_async_16(slot(stage, 1, j), p.x + offset + (size_t)v * VEC);
          if constexpr (RESIDUAL) copy_async_16(slot(stage, 2, j), p.grad_resid + offset + (size_t)v * VEC);
        }
      }
    }
    copy_async_commit();
  };

  const size_t start = (size_t)blockIdx.x * GROUPS + group;
#pragma unroll
  for (int stage = 0; stage < STAGES - 1; ++stage) fetch(start + stage * all, stage);
  float weight[VPT][VEC], grad_weight[VPT][VEC], grad_bias[VPT][VEC];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int v = lane + j * LANES;
#pragma unroll
    for (int e = 0; e < VEC; ++e) weight[j][e] = grad_weight[j][e] = grad_bias[j][e] = 0.0f;
    if (v < nvec) widen<W, VEC>(load_shared_operand<W, VEC>(p.weight + (size_t)v * VEC), weight[j]);
  }
  float mean = start < p.rows ? p.mean[start] : 0.0f, rstd = start < p.rows ? p.rstd[start] : 0.0f;
  int stage = 0, parity = 0;
  for (size_t row = start; row < p.rows; row += all) {
    fetch(row + (STAGES - 1) * all, stage == 0 ? STAGES - 1 : stage - 1);
    const size_t after = row + all;
    const float next_mean = after < p.rows ? p.mean[after] : 0.0f, next_rstd = after < p.rows ? p.rstd[after] : 0.0f;
    copy_async_wait<STAGES - 1>();
    Pack<T, VEC> given[VPT], x[VPT];
    float sum_g = 0.0f, sum_gn = 0.0f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      if (lane + j * LANES < nvec) {
        given[j] = *reinterpret_cast<const Pack<T, VEC>*>(slot(stage, 0, j));
        x[j] = *reinterpret_cast<const Pack<T, VEC>*>(slot(stage, 1, j));
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float d = Conv<float, T>::widen(given[j].v[e]), n = (Conv<float, T>::widen(x[j].v[e]) - mean) * rstd;
          const float g = d * weight[j][e];
          sum_g += g;
          sum_gn = fmaf(g, n, sum_gn);
          grad_weight[j][e] = fmaf(d, n, grad_weight[j][e]);
          grad_bias[j][e] += d;
        }
      }
    }
    sum_g = warp_sum(sum_g);
    sum_gn = warp_sum(sum_gn);
    if constexpr (WARPS > 1) {
      // two buffers, so one barrier a row: a warp can write the other buffer only after every warp has read this one
      if ((threadIdx.x & 31) == 0) sums[parity][group][lane >> 5] = make_float2(sum_g, sum_gn);
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(LANES) : "memory");
      const float2 part = (threadIdx.x & 31) < WARPS ? sums[parity][group][threadIdx.x & 31] : make_float2(0.0f, 0.0f);
      sum_g = warp_sum(part.x);
      sum_gn = warp_sum(part.y);
      parity ^= 1;
    }
    const float mean_g = sum_g * scale, mean_gn = sum_gn * scale;
    T* __restrict__ to = p.grad_x + row * (size_t)p.hidden;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int v = lane + j * LANES;
      if (v < nvec) {
        Pack<T, VEC> resid, r;
        if constexpr (RESIDUAL) resid = *reinterpret_cast<const Pack<T, VEC>*>(slot(stage, 2, j));
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float n = (Conv<float, T>::widen(x[j].v[e]) - mean) * rstd;
          const float inner = fmaf(-n, mean_gn, fmaf(Conv<float, T>::widen(given[j].v[e]), weight[j][e], -mean_g));
          r.v[e] = Conv<float, T>::narrow(RESIDUAL ? fmaf(rstd, inner, Conv<float, T>::widen(resid.v[e])) : rstd * inner);
        }
        store_stream<T, VEC>(to + (size_t)v * VEC, r);
      }
    }
    mean = next_mean;
    rstd = next_rstd;
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  copy_async_wait<0>();
  // the CTA's share of the column sums: its groups add up in shared memory, one after the other
  float* columns = reinterpret_cast<float*>(shared);  // [2][hidden], over the row slots, which nobody reads any more
  float* mine = p.partial + (size_t)blockIdx.x * 2 * p.hidden;
  if constexpr (GROUPS > 1) {
    for (int g = 0; g < GROUPS; ++g) {
      __syncthreads();
      if (g == group) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
          const int v = lane + j * LANES;
          if (v < nvec) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const int c = v * VEC + e;
              columns[c] = g ? columns[c] + grad_weight[j][e] : grad_weight[j][e];
              columns[p.hidden + c] = g ? columns[p.hidden + c] + grad_bias[j][e] : grad_bias[j][e];
            }
          }
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * p.hidden; c += Shape::kThreads) mine[c] = columns[c];
  } else {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int v = lane + j * LANES;
      if (v < nvec) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
          *reinterpret_cast<float4*>(mine + v * VEC + e) = make_float4(grad_weight[j][e], grad_weight[j][e + 1], grad_weight[j][e + 2], grad_weight[j][e + 3]);
          *reinterpret_cast<float4*>(mine + p.hidden + v * VEC + e) = make_float4(grad_bias[j][e], grad_bias[j][e + 1], grad_bias[j][e + 2], grad_bias[j][e + 3]);
        }
      }
    }
  }
}

// Any width and alignment: grad_x of one row per CTA, element by element, reading the row twice (the second time from L2).
template <typename T, typename W>
__global__ void __launch_bounds__(kElementThreads)
norm_backward_by_element(const __grid_constant__ Backward<T, W> p) {
  __shared__ float scratch[32];
  dependent_launch_prologue();
  const size_t row = blockIdx.x, offset = row * (size_t)p.hidden;
  const float mean = p.mean[row], rstd = p.rstd[row];
  float sum_g = 0.0f, sum_gn = 0.0f;
#pragma unroll 4
  for (int c = threadIdx.x; c < p.hidden; c += kElementThreads) {
    const float g = Conv<float, T>::widen(p.grad_out[offset + c]) * Conv<float, W>::widen(p.weight[c]);
    sum_g += g;
    sum_gn = fmaf(g, (Conv<float, T>::widen(p.x[offset + c]) - mean) * rstd, sum_gn);
  }
  const float mean_g = row_sum<kElementThreads / 32>(sum_g, scratch) / (float)p.hidden;
  const float mean_gn = row_sum<kElementThreads / 32>(sum_gn, scratch) / (float)p.hidden;
#pragma unroll 4
  for (int c = threadIdx.x; c < p.hidden; c += kElementThreads) {
    const float g = Conv<float, T>::widen(p.grad_out[offset + c]) * Conv<float, W>::widen(p.weight[c]);
    const float n = (Conv<float, T>::widen(p.x[offset + c]) - mean) * rstd;
    const float inner = rstd * fmaf(-n, mean_gn, g - mean_g);
    p.grad_x[offset + c] = Conv<float, T>::narrow(p.grad_resid ? inner + Conv<float, T>::widen(p.grad_resid[offset + c]) : inner);
  }
}

// The column sums that go with it: thread per column, CTA per slab of rows.
template <typename T, typename W>
__global__ void __launch_bounds__(kElementThreads)
norm_backward_columns(const __grid_constant__ Backward<T, W> p, size_t slab_rows) {
  dependent_launch_prologue();
  const int c = blockIdx.x * kElementThreads + threadIdx.x;
  if (c >= p.hidden) return;
  const size_t first = (size_t)blockIdx.y * slab_rows;
  const size_t end = p.rows - first < slab_rows ? p.rows : first + slab_rows;
  float grad_weight = 0.0f, grad_bias = 0.0f;
#pragma unroll 4
  for (size_t row = first; row < end; ++row) {
    const float d = Conv<float, T>::widen(p.grad_out[row * p.hidden + c]);
    grad_weight = fmaf(d, (Conv<float, T>::widen(p.x[row * p.hidden + c]) - p.mean[row]) * p.rstd[row], grad_weight);
    grad_bias += d;
  }
  float* mine = p.partial + (size_t)blockIdx.y * 2 * p.hidden;
  mine[c] = grad_weight;
  mine[p.hidden + c] = grad_bias;
}

// grad_weight and grad_bias from the shares: 32 columns to a CTA, eight warps over the shares.
constexpr int kJoinSlices = 8;
template <typename W>
__global__ void __launch_bounds__(32 * kJoinSlices)
join_columns(const float* __restrict__ partial, int shares, int hidden, W* __restrict__ grad_weight, W* __restrict__ grad_bias) {
  __shared__ float2 parts[kJoinSlices][32];
  dependent_launch_prologue();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  const int each = (shares + kJoinSlices - 1) / kJoinSlices, first = slice * each;
  const int end = first + each < shares ? first + each : shares;
  float2 sum = make_float2(0.0f, 0.0f);
  if (c < hidden) {
#pragma unroll 8
    for (int s = first; s < end; ++s) {
      sum.x += partial[(size_t)s * 2 * hidden + c];
      sum.y += partial[(size_t)s * 2 * hidden + hidden + c];
    }
  }
  parts[slice][lane] = sum;
  __syncthreads();
  if (slice == 0 && c < hidden) {
#pragma unroll
    for (int s = 1; s < kJoinSlices; ++s) {
      sum.x += parts[s][lane].x;
      sum.y += parts[s][lane].y;
    }
    grad_weight[c] = Conv<float, W>::narrow(sum.x);
    if (grad_bias) grad_bias[c] = Conv<float, W>::narrow(sum.y);
  }
}

template <typename W> int join(const float* partial, int shares, int hidden, void* grad_weight, void* grad_bias, cudaStream_t stream) {
  launch_dependent(join_columns<W>, dim3((hidden + 31) / 32), dim3(32 * kJoinSlices), 0, stream, partial, shares, hidden,
                   static_cast<W*>(grad_weight), static_cast<W*>(grad_bias));
  return check_launch("layernorm_backward join launch");
}

template <typename T, typename W, int WARPS, int GROUPS, int VPT, bool RESIDUAL>
int launch_backward(Backward<T, W> p, void* grad_weight, void* grad_bias, cudaStream_t stream) {
  using Shape = BackwardShape<T, WARPS, GROUPS, VPT, RESIDUAL>;
  const auto kernel = norm_backward_rows<T, W, WARPS, GROUPS, VPT, RESIDUAL>;
  constexpr int resident = WARPS * GROUPS <= 8 ? 2 : 1;
  const size_t wanted = (p.rows + GROUPS - 1) / GROUPS, most = (size_t)multiprocessor_count() * resident;
  const int blocks = (int)(wanted < most ? wanted : most);
  Workspace workspace(stream);
  if (int status = workspace.take((size_t)blocks * 2 * p.hidden * sizeof(float), "layernorm_backward workspace")) return status;
  p.partial = reinterpret_cast<float*>(workspace.data());
  if (int status = check_runtime(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem),
                                 "cudaFuncSetAttribute(layernorm_backward)"))
    return status;
  launch_dependent(kernel, dim3(blocks), dim3(Shape::kThreads), (size_t)Shape::kSmem, stream, p);
  if (int status = check_launch("layernorm_backward kernel launch")) return status;
  if (int status = join<W>(p.partial, blocks, p.hidden, grad_weight, grad_bias, stream)) return status;
  return workspace.release("cudaFreeAsync(layernorm_backward workspace)");
}

template <typename T, typename W> int backward(Backward<T, W> p, bool aligned, void* grad_weight, void* grad_bias, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  const int nvec = p.hidden / VEC;
  if (aligned && p.hidden % VEC == 0 && nvec <= 1024) {
#define BB200_LN_BACKWARD(WARPS, GROUPS, VPT)                                                                             \
  if (nvec <= (WARPS) * 32 * (VPT))                                                                                       \
    return p.grad_resid ? launch_backward<T, W, WARPS, GROUPS, VPT, true>(p, grad_weight, grad_bias, stream)             \
                        : launch_backward<T, W, WARPS, GROUPS, VPT, false>(p, grad_weight, grad_bias, stream)
    BB200_LN_BACKWARD(1, 8, 1);
    BB200_LN_BACKWARD(1, 8, 2);
    BB200_LN_BACKWARD(2, 4, 2);
    BB200_LN_BACKWARD(4, 2, 2);
    BB200_LN_BACKWARD(8, 1, 2);
    BB200_LN_BACKWARD(16, 1, 2);
#undef BB200_LN_BACKWARD
  }
  const size_t blocks = (p.hidden + kElementThreads - 1) / kElementThreads;
  size_t slabs = ((size_t)multiprocessor_count() * 8 + blocks - 1) / blocks;
  if (slabs > (p.rows + 7) / 8) slabs = (p.rows + 7) / 8;
  if (slabs > 1024) slabs = 1024;
  const size_t slab_rows = (p.rows + slabs - 1) / slabs;
  slabs = (p.rows + slab_rows - 1) / slab_rows;
  Workspace workspace(stream);
  if (int status = workspace.take(slabs * 2 * p.hidden * sizeof(float), "layernorm_backward workspace")) return status;
  p.partial = reinterpret_cast<float*>(workspace.data());
  launch_dependent(norm_backward_by_element<T, W>, dim3((unsigned)p.rows), dim3(kElementThreads), 0, stream, p);
  if (int status = check_launch("layernorm_backward kernel launch")) return status;
  launch_dependent(norm_backward_columns<T, W>, dim3((unsigned)blocks, (unsigned)slabs), dim3(kElementThreads), 0, stream, p, slab_rows);
  if (int status = check_launch("layernorm_backward columns launch")) return status;
  if (int status = join<W>(p.partial, (int)slabs, p.hidden, grad_weight, grad_bias, stream)) return status;
  return workspace.release("cudaFreeAsync(layernorm_backward workspace)");
}

int check_norm(const char* what, bb200_dtype dtype, bb200_dtype weight_dtype, size_t rows, size_t hidden) {
  if (dtype != BB200_F32 && dtype != BB200_BF16 && dtype != BB200_F16)
    return fail(BB200_E_INVALID_ARGUMENT, "%s: dtype %d is not bf16/f16/f32", what, (int)dtype);
  if (weight_dtype != dtype && weight_dtype != BB200_F32)
    return fail(BB200_E_INVALID_ARGUMENT, "%s: weight dtype %d must be the rows' dtype or f32", what, (int)weight_dtype);
  if (rows == 0 || hidden == 0) return fail(BB200_E_INVALID_ARGUMENT, "%s: rows and hidden must be > 0", what);
  const size_t limit = dtype == BB200_F32 ? 16384 : 32768;
  if (rows >= 0x7fffffffu || hidden > limit)
    return fail(BB200_E_UNSUPPORTED_SHAPE, "%s: rows must be below 2^31 - 1 and hidden at most %zu (got %zu)", what, limit, hidden);
  return BB200_OK;
}

bool misaligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

struct Range {
  const void* p;
  size_t bytes;
};

// Whether any of `written` shares memory with another of `written` or with one of `read`.
template <size_t N, size_t M> bool clash(const Range (&written)[N], const Range (&read)[M]) {
  for (size_t i = 0; i < N; ++i) {
    for (size_t j = i + 1; j < N; ++j)
      if (overlap(written[i].p, written[i].bytes, written[j].p, written[j].bytes)) return true;
    for (size_t j = 0; j < M; ++j)
      if (overlap(written[i].p, written[i].bytes, read[j].p, read[j].bytes)) return true;
  }
  return false;
}

}  // namespace
}  // namespace bb200

using namespace bb200;

#define BB200_NORM_DTYPES(CALL)                                                                                          \
  switch (dtype) {                                                                                                       \
    case BB200_BF16: return weight_dtype == BB200_F32 ? CALL(__nv_bfloat16, float) : CALL(__nv_bfloat16, __nv_bfloat16); \
    case BB200_F16: return weight_dtype == BB200_F32 ? CALL(__half, float) : CALL(__half, __half);                       \
    default: return CALL(float, float);                                                                                  \
  }

extern "C" int bb200_layernorm_forward(bb200_dtype dtype, bb200_dtype weight_dtype, const void* x, const void* residual, const void* weight,
                                       const void* bias, void* out, void* out_resid, float* mean, float* rstd, size_t rows, size_t hidden,
                                       float epsilon, void* stream) {
  if (!x || !weight || !out || !mean || !rstd) return fail(BB200_E_INVALID_ARGUMENT, "layernorm_forward: null tensor pointer");
  if (!residual != !out_resid) return fail(BB200_E_INVALID_ARGUMENT, "layernorm_forward: residual and out_resid go together");
  if (int status = check_norm("layernorm_forward", dtype, weight_dtype, rows, hidden)) return status;
  const size_t size = dtype_bytes(dtype), weight_size = dtype_bytes(weight_dtype), row_bytes = rows * hidden * size;
  bool aligned = true;
  for (const void* p : {x, residual, static_cast<const void*>(out), static_cast<const void*>(out_resid)}) {
    if (misaligned(p, size)) return fail(BB200_E_MISALIGNED, "layernorm_forward: a tensor is not aligned to its element size");
    aligned = aligned && aligned16(p);
  }
  for (const void* p : {weight, bias}) {
    if (misaligned(p, weight_size)) return fail(BB200_E_MISALIGNED, "layernorm_forward: a tensor is not aligned to its element size");
    aligned = aligned && aligned16(p);
  }
  if (misaligned(mean, 4) || misaligned(rstd, 4)) return fail(BB200_E_MISALIGNED, "layernorm_forward: a tensor is not aligned to its element size");
  // out_resid may be x or residual itself: every element is read by the thread that writes it
  const Range written[] = {{out, row_bytes}, {mean, rows * 4}, {rstd, rows * 4}, {out_resid, row_bytes}};
  const Range read[] = {{x == out_resid ? nullptr : x, row_bytes}, {residual == out_resid ? nullptr : residual, row_bytes},
                        {weight, hidden * weight_size}, {bias, hidden * weight_size}};
  if (clash(written, read) || overlap(out, row_bytes, x, row_bytes) || overlap(out, row_bytes, residual, row_bytes))
    return fail(BB200_E_INVALID_ARGUMENT, "layernorm_forward: an output shares memory with another tensor");
#define BB200_CALL(T, W)                                                                                                              \
  forward<T, W>({static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const W*>(weight), static_cast<const W*>(bias), \
                 static_cast<T*>(out), static_cast<T*>(out_resid), mean, rstd, rows, (int)hidden, epsilon},                            \
                aligned, static_cast<cudaStream_t>(stream))
  BB200_NORM_DTYPES(BB200_CALL)
#undef BB200_CALL
}

extern "C" int bb200_layernorm_backward(bb200_dtype dtype, bb200_dtype weight_dtype, const void* grad_out, const void* x, const float* mean,
                                        const float* rstd, const void* weight, const void* grad_resid, void* grad_x, void* grad_weight,
                                        void* grad_bias, size_t rows, size_t hidden, void* stream) {
  if (!grad_out || !x || !mean || !rstd || !weight || !grad_x || !grad_weight)
    return fail(BB200_E_INVALID_ARGUMENT, "layernorm_backward: null tensor pointer");
  if (int status = check_norm("layernorm_backward", dtype, weight_dtype, rows, hidden)) return status;
  const size_t size = dtype_bytes(dtype), weight_size = dtype_bytes(weight_dtype), row_bytes = rows * hidden * size;
  bool aligned = aligned16(weight);
  for (const void* p : {grad_out, x, grad_resid, static_cast<const void*>(grad_x)}) {
    if (misaligned(p, size)) return fail(BB200_E_MISALIGNED, "layernorm_backward: a tensor is not aligned to its element size");
    aligned = aligned && aligned16(p);
  }
  for (const void* p : {weight, static_cast<const void*>(grad_weight), static_cast<const void*>(grad_bias)})
    if (misaligned(p, weight_size)) return fail(BB200_E_MISALIGNED, "layernorm_backward: a tensor is not aligned to its element size");
  if (misaligned(mean, 4) || misaligned(rstd, 4)) return fail(BB200_E_MISALIGNED, "layernorm_backward: a tensor is not aligned to its element size");
  const Range written[] = {{grad_x, row_bytes}, {grad_weight, hidden * weight_size}, {grad_bias, hidden * weight_size}};
  const Range read[] = {{grad_out, row_bytes}, {x, row_bytes}, {grad_resid, row_bytes}, {mean, rows * 4}, {rstd, rows * 4}, {weight, hidden * weight_size}};
  if (clash(written, read)) return fail(BB200_E_INVALID_ARGUMENT, "layernorm_backward: an output shares memory with another tensor");
#define BB200_CALL(T, W)                                                                                                                \
  backward<T, W>({static_cast<const T*>(grad_out), static_cast<const T*>(x), mean, rstd, static_cast<const W*>(weight),                  \
                  static_cast<const T*>(grad_resid), static_cast<T*>(grad_x), nullptr, rows, (int)hidden},                              \
                 aligned, grad_weight, grad_bias, static_cast<cudaStream_t>(stream))
  BB200_NORM_DTYPES(BB200_CALL)
#undef BB200_CALL
}
