// layernorm_backward.cu — the gradients of LayerNorm, sm_100a.  With n = (x - mean) * rstd and g = grad_out * weight:
//
//   grad_x      = rstd * (g - mean(g) - n * mean(g * n))  (+ grad_resid)
//   grad_weight = sum over rows of grad_out * n,   grad_bias = sum over rows of grad_out
//
// Bound by HBM bytes: grad_out and x (and grad_resid) are read once, grad_x written once.  fp32 throughout, one rounding per
// output.  A persistent CTA per SM walks groups of rows (bb200_rows.cuh); a thread keeps the two column sums of its columns
// in registers over all its rows, and a second kernel joins the CTAs' shares in a fixed order: no atomics, the same call
// gives the same bits.
#include <float.h>

#include "bb200_rows.cuh"
#include "layernorm_train.h"

namespace bb200 {
namespace {

template <typename T> struct Backward {
  const T* grad_out;
  const T* x;
  const float* mean;
  const float* rstd;
  const void* weight;
  const T* grad_resid;  // null: none
  T* grad_x;
  float* partial;  // [shares][2][hidden]: grad_weight and grad_bias over some of the rows
  void* grad_weight;
  void* grad_bias;  // null: none
  size_t rows;
  int hidden;
  bool wide;  // weight and the column sums are f32 beside 16-bit rows
};

constexpr int kRowThreads = 512, kMostSmem = 204800;

// CLUSTER: the grid is one cluster, and its CTAs join the column sums by themselves.
template <typename T, typename Rows, bool RESIDUAL, bool CLUSTER>
__global__ void __launch_bounds__(kRowThreads, 1)
norm_backward_rows(const __grid_constant__ Backward<T> p) {
  constexpr int PAIRS = Rows::PAIRS, LANES = Rows::LANES, GROUPS = Rows::GROUPS;
  static_assert(LANES <= 32 || GROUPS <= 15, "a barrier for every group beside __syncthreads");
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ RowSums<LANES, 2> scratch[GROUPS];
  dependent_launch_prologue();
  const int group = threadIdx.x / LANES, lane = threadIdx.x % LANES, barrier = group + 1;
  const T* sources[RESIDUAL ? 3 : 2];
  sources[0] = p.grad_out;
  sources[1] = p.x;
  if constexpr (RESIDUAL) sources[2] = p.grad_resid;
  Rows rows(shared, sources, p.rows, p.hidden, lane, group);
  const size_t stride = (size_t)gridDim.x * GROUPS;
  size_t row = (size_t)blockIdx.x * GROUPS + group;
  rows.start(row, stride, barrier);
  F2 weight[PAIRS], grad_weight[PAIRS], grad_bias[PAIRS];
  column_pairs<T>(rows, p.weight, p.wide, weight);
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) grad_weight[i] = grad_bias[i] = both(0.0f);
  const float scale = 1.0f / (float)p.hidden;
  float mean = row < p.rows ? p.mean[row] : 0.0f, rstd = row < p.rows ? p.rstd[row] : 0.0f;
  int turn = 0;
  // all groups of the CTA take the same number of turns, so every thread of a warp is there for the exchanges
  for (size_t first = (size_t)blockIdx.x * GROUPS; first < p.rows; first += stride, row += stride, rows.next()) {
    const bool active = row < p.rows;
    const size_t after = row + stride;
    const float next_mean = after < p.rows ? p.mean[after] : 0.0f, next_rstd = after < p.rows ? p.rstd[after] : 0.0f;
    rows.arrive(row, stride);
    F2 g[PAIRS], n[PAIRS];
    F2 sum_g = both(0.0f), sum_gn = both(0.0f);
    const F2 factor = both(rstd);
    if (active) {
      rows.get(0, g);
      rows.get(1, n);
      const F2 minus_mean = both(-mean);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        n[i] = (n[i] + minus_mean) * rows.where_inside(i, rstd);
        grad_weight[i] = fma2(g[i], n[i], grad_weight[i]);
        grad_bias[i] = grad_bias[i] + g[i];
        g[i] = g[i] * weight[i];
        sum_g = sum_g + g[i];
        sum_gn = fma2(g[i], n[i], sum_gn);
      }
      // past the row's end x and g are 0 and n, left alone, is -mean * rstd: where that overflows, 0 * n makes the sum NaN
      if constexpr (!Rows::kMasked) {
        if (!(fabsf(mean * rstd) <= FLT_MAX)) {
          sum_gn = both(0.0f);
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) sum_gn = fma2(g[i], rows.inside(i, n[i]), sum_gn);
        }
      }
    }
    float sums[2] = {total(sum_g), total(sum_gn)};
    rows.before_sums();
    row_sums<LANES>(sums, &scratch[group], turn, barrier);
    rows.after_sums(row, stride);
    if (active) {
      const F2 minus_mean_g = both(-sums[0] * scale), minus_mean_gn = both(-sums[1] * scale);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) g[i] = fma2(n[i], minus_mean_gn, g[i] + minus_mean_g);
      if constexpr (RESIDUAL) {
        rows.get(2, n);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) g[i] = fma2(g[i], factor, n[i]);
      } else {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) g[i] = g[i] * factor;
      }
      rows.put(p.grad_x + row * (size_t)p.hidden, g);
    }
    mean = next_mean;
    rstd = next_rstd;
  }
  copy_async_wait<0>();
  // the CTA's share of the column sums: groups inside a warp join by exchanges, warps (or groups) lay theirs out beside each
  // other in shared memory, over row slots that nobody reads any more, and every thread adds up some columns
  if constexpr (LANES < 32) {
#pragma unroll
    for (int offset = LANES; offset < 32; offset <<= 1) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        float a, b, c, d;
        split(grad_weight[i], a, b);
        split(grad_bias[i], c, d);
        a += __shfl_xor_sync(0xffffffffu, a, offset);
        b += __shfl_xor_sync(0xffffffffu, b, offset);
        c += __shfl_xor_sync(0xffffffffu, c, offset);
        d += __shfl_xor_sync(0xffffffffu, d, offset);
        grad_weight[i] = make_f2(a, b);
        grad_bias[i] = make_f2(c, d);
      }
    }
  }
  constexpr int SET = LANES < 32 ? 32 : LANES, SETS = kRowThreads / SET;
  constexpr bool STAGED = SETS > 1 || CLUSTER;
  static_assert(!STAGED || Rows::kBytes >= SETS * LANES * PAIRS * 2 * 2 * (int)sizeof(float), "the sets have to fit");
  float* share = p.partial + (size_t)blockIdx.x * 2 * p.hidden;
  float* columns = STAGED ? reinterpret_cast<float*>(shared) : share;  // [sets][2][hidden]
  if constexpr (STAGED) __syncthreads();
  if ((threadIdx.x & 31) % SET < LANES) {
    float* mine = columns + (threadIdx.x / SET) * 2 * p.hidden;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      float w[2], b[2];
      split(grad_weight[i], w[0], w[1]);
      split(grad_bias[i], b[0], b[1]);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int c = rows.column(i, half);
        if (c < p.hidden) {
          mine[c] = w[half];
          mine[p.hidden + c] = b[half];
        }
      }
    }
  }
  if constexpr (STAGED) {
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * p.hidden; c += kRowThreads) {
      float sum = columns[c];
#pragma unroll
      for (int set = 1; set < SETS; ++set) sum += columns[set * 2 * p.hidden + c];
      (CLUSTER ? columns : share)[c] = sum;
    }
    if constexpr (CLUSTER) __syncthreads();
  }
  if constexpr (CLUSTER) {
    cluster_barrier();
    for (int c = blockIdx.x * kRowThreads + threadIdx.x; c < 2 * p.hidden; c += gridDim.x * kRowThreads) {
      float sum = 0.0f;
#pragma unroll 4
      for (uint32_t cta = 0; cta < gridDim.x; ++cta) {
        float part;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part) : "r"(in_cta(columns + c, cta)) : "memory");
        sum += part;
      }
      const bool bias = c >= p.hidden;
      void* to = bias ? p.grad_bias : p.grad_weight;
      const int at = bias ? c - p.hidden : c;
      if (to && p.wide) static_cast<float*>(to)[at] = sum;
      else if (to) static_cast<T*>(to)[at] = Conv<float, T>::narrow(sum);
    }
    cluster_barrier();  // nobody leaves while another CTA still reads its share
  }
}

// Any width and alignment (rows of more than 8192 columns, of more than 4096 in f32 where they are no whole vectors): grad_x of one
// row per CTA, element by element, reading the row twice (the second time from L2); 16384 x 12288 bf16 767 us, 16384 x 8192 above 156 us.
constexpr int kElementThreads = 256;
template <typename T> __device__ __forceinline__ float weight_at(const Backward<T>& p, int c) {
  return p.wide ? static_cast<const float*>(p.weight)[c] : Conv<float, T>::widen(static_cast<const T*>(p.weight)[c]);
}

template <typename T>
__global__ void __launch_bounds__(kElementThreads)
norm_backward_by_element(const __grid_constant__ Backward<T> p) {
  __shared__ RowSums<kElementThreads, 2> scratch;
  dependent_launch_prologue();
  const size_t row = blockIdx.x, offset = row * (size_t)p.hidden;
  const float mean = p.mean[row], rstd = p.rstd[row], scale = 1.0f / (float)p.hidden;
  float sum_g = 0.0f, sum_gn = 0.0f;
#pragma unroll 4
  for (int c = threadIdx.x; c < p.hidden; c += kElementThreads) {
    const float g = Conv<float, T>::widen(p.grad_out[offset + c]) * weight_at(p, c);
    sum_g += g;
    sum_gn = fmaf(g, (Conv<float, T>::widen(p.x[offset + c]) - mean) * rstd, sum_gn);
  }
  int turn = 0;
  float sums[2] = {sum_g, sum_gn};
  row_sums<kElementThreads>(sums, &scratch, turn, 1);
  const float mean_g = sums[0] * scale, mean_gn = sums[1] * scale;
#pragma unroll 4
  for (int c = threadIdx.x; c < p.hidden; c += kElementThreads) {
    const float g = Conv<float, T>::widen(p.grad_out[offset + c]) * weight_at(p, c);
    const float n = (Conv<float, T>::widen(p.x[offset + c]) - mean) * rstd;
    const float inner = rstd * fmaf(-n, mean_gn, g - mean_g);
    p.grad_x[offset + c] = Conv<float, T>::narrow(p.grad_resid ? inner + Conv<float, T>::widen(p.grad_resid[offset + c]) : inner);
  }
}

// The column sums that go with it: thread per column, CTA per slab of rows.
template <typename T>
__global__ void __launch_bounds__(kElementThreads)
norm_backward_columns(const __grid_constant__ Backward<T> p, size_t slab_rows) {
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
  float* share = p.partial + (size_t)blockIdx.y * 2 * p.hidden;
  share[c] = grad_weight;
  share[p.hidden + c] = grad_bias;
}

// grad_weight and grad_bias from the shares: 32 columns to a CTA, 32 warps over the shares, so a thread has its handful of
// loads in flight at once.
template <typename W>
__global__ void __launch_bounds__(1024)
join_columns(const float* __restrict__ partial, int shares, int hidden, W* __restrict__ grad_weight, W* __restrict__ grad_bias) {
  __shared__ float2 parts[32][33];
  dependent_launch_prologue();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float2 sum = make_float2(0.0f, 0.0f);
  if (c < hidden) {
#pragma unroll 8
    for (int s = warp; s < shares; s += 32) {
      sum.x += partial[(size_t)s * 2 * hidden + c];
      sum.y += partial[(size_t)s * 2 * hidden + hidden + c];
    }
  }
  parts[warp][lane] = sum;
  __syncthreads();
  sum = parts[lane][warp];  // warp w joins column w
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) {
    sum.x += __shfl_xor_sync(0xffffffffu, sum.x, offset);
    sum.y += __shfl_xor_sync(0xffffffffu, sum.y, offset);
  }
  const int mine = blockIdx.x * 32 + warp;
  if (lane == 0 && mine < hidden) {
    grad_weight[mine] = Conv<float, W>::narrow(sum.x);
    if (grad_bias) grad_bias[mine] = Conv<float, W>::narrow(sum.y);
  }
}

template <typename T> int join(const Backward<T>& p, int shares, cudaStream_t stream) {
  const dim3 grid((p.hidden + 31) / 32), block(1024);
  const float* partial = p.partial;
  if (p.wide) launch_dependent(join_columns<float>, grid, block, 0, stream, partial, shares, p.hidden, static_cast<float*>(p.grad_weight), static_cast<float*>(p.grad_bias));
  else launch_dependent(join_columns<T>, grid, block, 0, stream, partial, shares, p.hidden, static_cast<T*>(p.grad_weight), static_cast<T*>(p.grad_bias));
  return check_launch("layernorm_backward join launch");
}

// Where two turns of 16 CTAs take all the rows, the grid is one cluster that joins the column sums by itself: no second
// launch, no workspace (64 x 1024 f32: 6.5 us a call, 9.4 us with them).
constexpr unsigned kMostCtas = 16;

template <typename T, typename Rows, bool RESIDUAL> int launch_cluster(const Backward<T>& p, size_t wanted, cudaStream_t stream) {
  constexpr auto kernel = norm_backward_rows<T, Rows, RESIDUAL, true>;
  if (int status = allow_shared_memory<kernel>(Rows::kBytes, "cudaFuncSetAttribute(layernorm_backward)")) return status;
  unsigned ctas = 1;
  while (ctas < kMostCtas && ctas < wanted) ctas *= 2;
  launch_dependent_cluster(kernel, dim3(ctas), dim3(kRowThreads), ctas, (size_t)Rows::kBytes, stream, p);
  return check_launch("layernorm_backward kernel launch");
}

template <typename T, typename Rows, bool RESIDUAL, bool MAY_CLUSTER> int launch_rows(Backward<T> p, cudaStream_t stream) {
  const size_t wanted = (p.rows + Rows::GROUPS - 1) / Rows::GROUPS, most = (size_t)multiprocessor_count();
  if constexpr (MAY_CLUSTER) {
    if (wanted <= 8 || (wanted <= 2 * kMostCtas && sixteen_fit<norm_backward_rows<T, Rows, RESIDUAL, true>>(kRowThreads, Rows::kBytes)))
      return launch_cluster<T, Rows, RESIDUAL>(p, wanted, stream);
  }
  constexpr auto kernel = norm_backward_rows<T, Rows, RESIDUAL, false>;
  if (int status = allow_shared_memory<kernel>(Rows::kBytes, "cudaFuncSetAttribute(layernorm_backward)")) return status;
  const int blocks = (int)(wanted < most ? wanted : most);
  Workspace workspace(stream);
  if (int status = workspace.take((size_t)blocks * 2 * p.hidden * sizeof(float), "layernorm_backward workspace")) return status;
  p.partial = reinterpret_cast<float*>(workspace.data());
  launch_dependent(kernel, dim3(blocks), dim3(kRowThreads), (size_t)Rows::kBytes, stream, p);
  if (int status = check_launch("layernorm_backward kernel launch")) return status;
  if (int status = join(p, blocks, stream)) return status;
  return workspace.release("cudaFreeAsync(layernorm_backward workspace)");
}

// Rows that fill all vectors of a group have nothing past their end to ask about, which is worth kernels of their own for the
// wide ones (65536 x 4096 bf16 261 and 267 us, 65536 x 8192 with residual equal; up to 1024 columns no difference either).
template <typename T, int LANES, int VPT, bool RESIDUAL> int launch_vectors(const Backward<T>& p, cudaStream_t stream) {
  constexpr int TENSORS = RESIDUAL ? 3 : 2;
  if constexpr (LANES >= 128) {
    if (p.hidden == LANES * VPT * 16 / (int)sizeof(T))
      return launch_rows<T, VectorRows<T, kRowThreads, LANES, VPT, TENSORS, kMostSmem, true>, RESIDUAL, true>(p, stream);
  }
  return launch_rows<T, VectorRows<T, kRowThreads, LANES, VPT, TENSORS, kMostSmem>, RESIDUAL, true>(p, stream);
}

template <typename T> int backward(Backward<T> p, bool aligned, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  const int nvec = p.hidden / VEC;
  if (aligned && p.hidden % VEC == 0) {
    // two vectors a thread (16 columns, 8 for f32): weight, both column sums and the row's two products fit the registers
#define BB200_VECTOR_ROWS(LANES, VPT) \
  if (nvec <= (LANES) * (VPT)) return p.grad_resid ? launch_vectors<T, LANES, VPT, true>(p, stream) : launch_vectors<T, LANES, VPT, false>(p, stream)
    BB200_VECTOR_ROWS(4, 2);
    BB200_VECTOR_ROWS(8, 2);
    BB200_VECTOR_ROWS(16, 2);
    BB200_VECTOR_ROWS(32, 2);
    BB200_VECTOR_ROWS(64, 2);
    BB200_VECTOR_ROWS(128, 2);
    BB200_VECTOR_ROWS(256, 2);
    BB200_VECTOR_ROWS(512, 2);
    if constexpr (VEC == 4) BB200_VECTOR_ROWS(512, 4);
#undef BB200_VECTOR_ROWS
  } else if (aligned) {
#define BB200_SHIFTED_ROWS(LANES, COLUMNS, SURE)                                                                           \
  if (p.hidden <= (LANES) * (COLUMNS))                                                                                 \
    return p.grad_resid ? launch_rows<T, ShiftedRows<T, kRowThreads, LANES, COLUMNS, SURE, 3, kMostSmem>, true, false>(p, stream)   \
                        : launch_rows<T, ShiftedRows<T, kRowThreads, LANES, COLUMNS, SURE, 2, kMostSmem>, false, false>(p, stream)
    constexpr int kColumns = 2 * VEC;  // 16, or 8 of f32, so that three stages fit
    BB200_SHIFTED_ROWS(32, 4, 0);
    BB200_SHIFTED_ROWS(32, 8, 4);
    if constexpr (VEC == 8) BB200_SHIFTED_ROWS(32, 16, 8);
    BB200_SHIFTED_ROWS(64, kColumns, kColumns / 2);
    BB200_SHIFTED_ROWS(128, kColumns, kColumns / 2);
    BB200_SHIFTED_ROWS(256, kColumns, kColumns / 2);
    BB200_SHIFTED_ROWS(512, kColumns, kColumns / 2);
#undef BB200_SHIFTED_ROWS
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
  launch_dependent(norm_backward_by_element<T>, dim3((unsigned)p.rows), dim3(kElementThreads), 0, stream, p);
  if (int status = check_launch("layernorm_backward kernel launch")) return status;
  launch_dependent(norm_backward_columns<T>, dim3((unsigned)blocks, (unsigned)slabs), dim3(kElementThreads), 0, stream, p, slab_rows);
  if (int status = check_launch("layernorm_backward columns launch")) return status;
  if (int status = join(p, (int)slabs, stream)) return status;
  return workspace.release("cudaFreeAsync(layernorm_backward workspace)");
}

}  // namespace
}  // namespace bb200

using namespace bb200;

extern "C" int bb200_layernorm_backward(bb200_dtype dtype, bb200_dtype weight_dtype, const void* grad_out, const void* x, const float* mean,
                                        const float* rstd, const void* weight, const void* grad_resid, void* grad_x, void* grad_weight,
                                        void* grad_bias, size_t rows, size_t hidden, void* stream) {
  if (!grad_out || !x || !mean || !rstd || !weight || !grad_x || !grad_weight)
    return fail(BB200_E_INVALID_ARGUMENT, "layernorm_backward: null tensor pointer");
  if (int status = check_norm("layernorm_backward", dtype, weight_dtype, rows, hidden)) return status;
  const size_t size = dtype_bytes(dtype), weight_size = dtype_bytes(weight_dtype), row_bytes = rows * hidden * size;
  bool aligned = true;
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
#define BB200_BACKWARD(T)                                                                                                       \
  backward<T>({static_cast<const T*>(grad_out), static_cast<const T*>(x), mean, rstd, weight, static_cast<const T*>(grad_resid),  \
               static_cast<T*>(grad_x), nullptr, grad_weight, grad_bias, rows, (int)hidden, weight_dtype != dtype},                                 \
              aligned, static_cast<cudaStream_t>(stream))
  switch (dtype) {
    case BB200_BF16: return BB200_BACKWARD(__nv_bfloat16);
    case BB200_F16: return BB200_BACKWARD(__half);
    default: return BB200_BACKWARD(float);
  }
#undef BB200_BACKWARD
}
