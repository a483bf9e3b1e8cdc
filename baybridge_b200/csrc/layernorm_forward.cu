// layernorm_forward.cu — LayerNorm for training, forward pass that keeps its statistics, sm_100a:
//
//   s = x (+ residual, stored);  out = (s - mean) * rstd * weight + bias;  mean, rstd = 1 / sqrt(variance + eps) per row, stored
//
// Bound by HBM bytes: x (and residual) are read once, out (and out_resid) written once.  fp32 throughout, one rounding per
// output; the variance is the mean of squared differences from the mean, taken from registers, so a large mean costs no
// precision.  Two forms: many brief CTAs that read the weights again for every row, and persistent CTAs that keep them in
// registers while rows are copied ahead into shared memory (bb200_rows.cuh); forward() says which is taken when.
#include "bb200_rows.cuh"
#include "layernorm_train.h"

namespace bb200 {
namespace {

template <typename T> struct Forward {
  const T* x;
  const T* residual;  // null: none, and out_resid is null too
  const void* weight;
  const void* bias;  // null: none
  T* out;
  T* out_resid;
  float* mean;
  float* rstd;
  size_t rows;
  int hidden;
  float epsilon;
  bool wide;  // weight and bias are f32 beside 16-bit rows
};

constexpr int kRowThreads = 512, kMostSmem = 204800;

template <typename T, typename Rows, bool RESIDUAL>
__global__ void __launch_bounds__(kRowThreads, 1)
norm_rows(const __grid_constant__ Forward<T> p) {
  constexpr int PAIRS = Rows::PAIRS, LANES = Rows::LANES, GROUPS = Rows::GROUPS;
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ RowSums<LANES, 1> scratch[GROUPS];
  dependent_launch_prologue();
  const int group = threadIdx.x / LANES, lane = threadIdx.x % LANES, barrier = group + 1;
  const T* sources[RESIDUAL ? 2 : 1];
  sources[0] = p.x;
  if constexpr (RESIDUAL) sources[1] = p.residual;
  Rows rows(shared, sources, p.rows, p.hidden, lane, group);
  const size_t stride = (size_t)gridDim.x * GROUPS;
  size_t row = (size_t)blockIdx.x * GROUPS + group;
  rows.start(row, stride, barrier);
  F2 weight[PAIRS], bias[PAIRS];
  column_pairs<T>(rows, p.weight, p.wide, weight);
  column_pairs<T>(rows, p.bias, p.wide, bias);
  const float scale = 1.0f / (float)p.hidden;
  int turn = 0;
  // all groups of the CTA take the same number of turns, so every thread of a warp is there for the exchanges
  for (size_t first = (size_t)blockIdx.x * GROUPS; first < p.rows; first += stride, row += stride, rows.next()) {
    const bool active = row < p.rows;
    rows.arrive(row, stride);
    F2 s[PAIRS];
    F2 sum2 = both(0.0f);
    const size_t offset = row * (size_t)p.hidden;
    if (active) {
      rows.get(0, s);
      if constexpr (RESIDUAL) {
        F2 r[PAIRS];
        rows.get(1, r);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) s[i] = s[i] + r[i];
        rows.put(p.out_resid + offset, s);
      }
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) sum2 = sum2 + s[i];
    }
    float sum[1] = {total(sum2)};
    rows.before_sums();
    row_sums<LANES>(sum, &scratch[group], turn, barrier);
    rows.after_sums(row, stride);
    const float mean = sum[0] * scale;
    F2 centred = both(0.0f);
    if (active) {
      const F2 minus_mean = both(-mean);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        s[i] = s[i] + minus_mean;
        const F2 kept = rows.inside(i, s[i]);
        centred = fma2(kept, kept, centred);
      }
    }
    sum[0] = total(centred);
    row_sums<LANES>(sum, &scratch[group], turn, barrier);
    const float rstd = 1.0f / sqrtf(sum[0] * scale + p.epsilon);
    if (active) {
      if (lane == 0) {
        p.mean[row] = mean;
        p.rstd[row] = rstd;
      }
      const F2 r = both(rstd);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) s[i] = fma2(s[i] * r, weight[i], bias[i]);
      rows.put(p.out + offset, s);
    }
  }
  copy_async_wait<0>();
}

// Rows of whole vectors with weights of their own type, 16-byte aligned: LANES threads a row, ROWS rows a CTA, no CTA stays.
// Many small CTAs hide the two sums of a row behind each other's loads.
template <typename T, int LANES, int ROWS, int VPT, bool RESIDUAL>
__global__ void __launch_bounds__(LANES * ROWS)
norm_brief_rows(const __grid_constant__ Forward<T> p) {
  constexpr int VEC = 16 / sizeof(T), PAIRS = VEC / 2;
  __shared__ RowSums<LANES, 1> scratch[ROWS];
  dependent_launch_prologue();
  const int group = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const size_t row = (size_t)blockIdx.x * ROWS + group;
  if (LANES >= 32 && row >= p.rows) return;
  const bool active = row < p.rows;
  const size_t offset = row * (size_t)p.hidden;
  const float scale = 1.0f / (float)p.hidden;
  F2 s[VPT][PAIRS];
  F2 sum2 = both(0.0f);
  {
    Pack<T, VEC> a[VPT], b[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (lane + j * LANES) * VEC;
      if (c < p.hidden && active) {
        a[j] = load_stream<T, VEC>(p.x + offset + c);
        if constexpr (RESIDUAL) b[j] = load_stream<T, VEC>(p.residual + offset + c);
      } else {
        *reinterpret_cast<uint4*>(&a[j]) = make_uint4(0, 0, 0, 0);
        if constexpr (RESIDUAL) *reinterpret_cast<uint4*>(&b[j]) = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        s[j][i] = Pairs<T>::get(a[j], i);
        if constexpr (RESIDUAL) {
          s[j][i] = s[j][i] + Pairs<T>::get(b[j], i);
          Pairs<T>::set(a[j], i, s[j][i]);
        }
        sum2 = sum2 + s[j][i];
      }
      if constexpr (RESIDUAL) {
        const int c = (lane + j * LANES) * VEC;
        if (c < p.hidden && active) store_stream<T, VEC>(p.out_resid + offset + c, a[j]);
      }
    }
  }
  int turn = 0;
  float sum[1] = {total(sum2)};
  row_sums<LANES>(sum, &scratch[group], turn, group);
  const float mean = sum[0] * scale;
  const F2 minus_mean = both(-mean);
  F2 centred = both(0.0f);
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    F2 part = both(0.0f);
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      s[j][i] = s[j][i] + minus_mean;
      part = fma2(s[j][i], s[j][i], part);
    }
    if ((lane + j * LANES) * VEC < p.hidden) centred = centred + part;
  }
  sum[0] = total(centred);
  row_sums<LANES>(sum, &scratch[group], turn, group);
  const float rstd = 1.0f / sqrtf(sum[0] * scale + p.epsilon);
  if (!active) return;
  if (lane == 0) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
  const F2 r = both(rstd);
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = (lane + j * LANES) * VEC;
    if (c < p.hidden) {
      Pack<T, VEC> o;
      const Pack<T, VEC> w = load_shared_operand<T, VEC>(static_cast<const T*>(p.weight) + c);
      Pack<T, VEC> b;
      *reinterpret_cast<uint4*>(&b) = make_uint4(0, 0, 0, 0);
      if (p.bias) b = load_shared_operand<T, VEC>(static_cast<const T*>(p.bias) + c);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) Pairs<T>::set(o, i, fma2(s[j][i] * r, Pairs<T>::get(w, i), Pairs<T>::get(b, i)));
      store_stream<T, VEC>(p.out + offset + c, o);
    }
  }
}

template <typename T, int LANES, int ROWS, int VPT> int launch_brief(const Forward<T>& p, cudaStream_t stream) {
  const dim3 grid((unsigned)((p.rows + ROWS - 1) / ROWS)), block(LANES * ROWS);
  if (p.residual) launch_dependent(norm_brief_rows<T, LANES, ROWS, VPT, true>, grid, block, 0, stream, p);
  else launch_dependent(norm_brief_rows<T, LANES, ROWS, VPT, false>, grid, block, 0, stream, p);
  return check_launch("layernorm_forward kernel launch");
}

// One row to a CTA, all of it in registers: rows of more than 8192 columns, which the persistent kernel does not take.  Weights are read
// element by element for every row, which is what bounds it (16384 x 12288 bf16 487 us, 16384 x 8192 in brief CTAs 97 us).
template <typename T, int THREADS, int VPT>
__global__ void __launch_bounds__(THREADS)
norm_long_rows(const __grid_constant__ Forward<T> p) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ RowSums<THREADS, 1> scratch;
  dependent_launch_prologue();
  const size_t row = blockIdx.x, offset = row * (size_t)p.hidden;
  const float scale = 1.0f / (float)p.hidden;
  float s[VPT][VEC];
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = (threadIdx.x + j * THREADS) * VEC;
    if (c < p.hidden) {
      const Pack<T, VEC> a = load_stream<T, VEC>(p.x + offset + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[j][e] = Conv<float, T>::widen(a.v[e]);
      if (p.residual) {
        const Pack<T, VEC> b = load_stream<T, VEC>(p.residual + offset + c);
        Pack<T, VEC> r;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          s[j][e] += Conv<float, T>::widen(b.v[e]);
          r.v[e] = Conv<float, T>::narrow(s[j][e]);
        }
        store_stream<T, VEC>(p.out_resid + offset + c, r);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum += s[j][e];
    }
  }
  int turn = 0;
  float sums[1] = {sum};
  row_sums<THREADS>(sums, &scratch, turn, 1);
  const float mean = sums[0] * scale;
  float centred = 0.0f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    if ((threadIdx.x + j * THREADS) * VEC < p.hidden) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        s[j][e] -= mean;
        centred = fmaf(s[j][e], s[j][e], centred);
      }
    }
  }
  sums[0] = centred;
  row_sums<THREADS>(sums, &scratch, turn, 1);
  const float rstd = 1.0f / sqrtf(sums[0] * scale + p.epsilon);
  if (threadIdx.x == 0) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = (threadIdx.x + j * THREADS) * VEC;
    if (c < p.hidden) {
      Pack<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float w = p.wide ? static_cast<const float*>(p.weight)[c + e] : Conv<float, T>::widen(static_cast<const T*>(p.weight)[c + e]);
        const float b = !p.bias ? 0.0f : p.wide ? static_cast<const float*>(p.bias)[c + e] : Conv<float, T>::widen(static_cast<const T*>(p.bias)[c + e]);
        o.v[e] = Conv<float, T>::narrow(fmaf(s[j][e] * rstd, w, b));
      }
      store_stream<T, VEC>(p.out + offset + c, o);
    }
  }
}

// Rows of any width and alignment, a brief CTA for ROWS of them: thread `lane` of LANES owns the columns lane, lane + LANES,
// ..., and keeps them in registers; SURE of its COLUMNS lie inside every row this form is used for and are not asked about.
template <typename T, int LANES, int ROWS, int COLUMNS, int SURE, bool RESIDUAL>
__global__ void __launch_bounds__(LANES * ROWS)
norm_rows_by_element(const __grid_constant__ Forward<T> p) {
  __shared__ RowSums<LANES, 1> scratch[ROWS];
  dependent_launch_prologue();
  const int group = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const size_t row = (size_t)blockIdx.x * ROWS + group;
  if (row >= p.rows) return;
  const size_t offset = row * (size_t)p.hidden + lane;
  const float scale = 1.0f / (float)p.hidden;
  const auto has = [&](int k) { return k < SURE || lane + k * LANES < p.hidden; };
  float s[COLUMNS];
  T a[COLUMNS], b[COLUMNS];
#pragma unroll
  for (int k = 0; k < COLUMNS; ++k) {
    if (has(k)) {
      a[k] = p.x[offset + k * LANES];
      if constexpr (RESIDUAL) b[k] = p.residual[offset + k * LANES];
    }
  }
  float sum[1] = {0.0f};
#pragma unroll
  for (int k = 0; k < COLUMNS; ++k) {
    s[k] = has(k) ? Conv<float, T>::widen(a[k]) : 0.0f;
    if constexpr (RESIDUAL) {
      if (has(k)) {
        s[k] += Conv<float, T>::widen(b[k]);
        p.out_resid[offset + k * LANES] = Conv<float, T>::narrow(s[k]);
      }
    }
    sum[0] += s[k];
  }
  int turn = 0;
  row_sums<LANES>(sum, &scratch[group], turn, group);
  const float mean = sum[0] * scale;
  sum[0] = 0.0f;
#pragma unroll
  for (int k = 0; k < COLUMNS; ++k) {
    s[k] -= mean;
    if (has(k)) sum[0] = fmaf(s[k], s[k], sum[0]);
  }
  row_sums<LANES>(sum, &scratch[group], turn, group);
  const float rstd = 1.0f / sqrtf(sum[0] * scale + p.epsilon);
  if (lane == 0) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
#pragma unroll
  for (int k = 0; k < COLUMNS; ++k) {
    if (has(k)) {
      const int c = lane + k * LANES;
      const float w = p.wide ? static_cast<const float*>(p.weight)[c] : Conv<float, T>::widen(static_cast<const T*>(p.weight)[c]);
      const float v = !p.bias ? 0.0f : p.wide ? static_cast<const float*>(p.bias)[c] : Conv<float, T>::widen(static_cast<const T*>(p.bias)[c]);
      p.out[offset + k * LANES] = Conv<float, T>::narrow(fmaf(s[k] * rstd, w, v));
    }
  }
}

template <typename T, int LANES, int ROWS, int COLUMNS, int SURE> int launch_by_element(const Forward<T>& p, cudaStream_t stream) {
  const dim3 grid((unsigned)((p.rows + ROWS - 1) / ROWS)), block(LANES * ROWS);
  if (p.residual) launch_dependent(norm_rows_by_element<T, LANES, ROWS, COLUMNS, SURE, true>, grid, block, 0, stream, p);
  else launch_dependent(norm_rows_by_element<T, LANES, ROWS, COLUMNS, SURE, false>, grid, block, 0, stream, p);
  return check_launch("layernorm_forward kernel launch");
}

template <typename T, typename Rows, bool RESIDUAL> int launch_rows(const Forward<T>& p, cudaStream_t stream) {
  constexpr auto kernel = norm_rows<T, Rows, RESIDUAL>;
  if (int status = allow_shared_memory<kernel>(Rows::kBytes, "cudaFuncSetAttribute(layernorm_forward)"))
    return status;
  const size_t wanted = (p.rows + Rows::GROUPS - 1) / Rows::GROUPS, most = (size_t)multiprocessor_count();
  launch_dependent(kernel, dim3((unsigned)(wanted < most ? wanted : most)), dim3(kRowThreads), (size_t)Rows::kBytes, stream, p);
  return check_launch("layernorm_forward kernel launch");
}

template <typename T> int forward(const Forward<T>& p, bool aligned, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  const int nvec = p.hidden / VEC;
  if (aligned && p.hidden % VEC == 0) {
    // Weights of the rows' own type are read again for every row (from L1 and L2, 16 bytes a load); f32 weights beside 16-bit
    // rows would be twice the rows' own bytes, so they stay in a persistent kernel's registers.  65536 rows, bf16: brief
    // kernel and persistent one with bf16 weights 84 and 97 us (1024 wide, residual), 315 and 352 us (4096, residual), 392 and
    // 395 us (8192); with f32 weights 176 and 95 us (2048), 833 and 660 us (8192, residual).
    if (!p.wide && nvec <= 512 && aligned16(p.weight) && aligned16(p.bias)) {
      if (nvec <= 8) return launch_brief<T, 8, 32, 1>(p, stream);
      if (nvec <= 16) return launch_brief<T, 16, 16, 1>(p, stream);
      if (nvec <= 32) return launch_brief<T, 32, 8, 1>(p, stream);
      if (nvec <= 64) return launch_brief<T, 32, 8, 2>(p, stream);
      if (nvec <= 128) return launch_brief<T, 32, 8, 4>(p, stream);
      if (nvec <= 256) return launch_brief<T, 128, 2, 2>(p, stream);
      return launch_brief<T, 256, 1, 2>(p, stream);
    }
    // Up to 32 columns a thread, whose weight and bias fit the registers beside the row; two groups of 256 threads hide each
    // other's sums (8192 wide, bf16: 395 us against 523 us for one group of 512).
#define BB200_VECTOR_ROWS(LANES, VPT)                                                              \
  if (nvec <= (LANES) * (VPT))                                                                     \
    return p.residual ? launch_rows<T, VectorRows<T, kRowThreads, LANES, VPT, 2, kMostSmem>, true>(p, stream) : launch_rows<T, VectorRows<T, kRowThreads, LANES, VPT, 1, kMostSmem>, false>(p, stream)
    BB200_VECTOR_ROWS(4, 2);
    BB200_VECTOR_ROWS(8, 2);
    BB200_VECTOR_ROWS(16, 2);
    BB200_VECTOR_ROWS(32, 2);
    BB200_VECTOR_ROWS(32, 4);
    BB200_VECTOR_ROWS(64, 4);
    // Around 4096 columns of 16 bits: four groups of 128 threads, which hide each other's sums (65536 x 4096 bf16: 177 us, with
    // two of 256 259 us), but with a residual there is as much in flight either way, and the longer rows a group has in hand
    // cost more than that (373 and 349 us); a few rows take the groups that finish one sooner (200 rows: 8.0 and 6.4 us).
    if (!p.residual && p.rows > 2 * (size_t)multiprocessor_count()) {
      if (nvec <= 512) return launch_rows<T, VectorRows<T, kRowThreads, 128, 4, 1, kMostSmem>, false>(p, stream);
    }
    BB200_VECTOR_ROWS(256, 2);
    BB200_VECTOR_ROWS(256, 4);
    if constexpr (VEC == 4) BB200_VECTOR_ROWS(512, 4);
#undef BB200_VECTOR_ROWS
    const dim3 grid((unsigned)p.rows), block(1024);
    if (VEC == 8 && nvec <= 2048) {
      if constexpr (VEC == 8) launch_dependent(norm_long_rows<T, 1024, 2>, grid, block, 0, stream, p);
    } else {
      launch_dependent(norm_long_rows<T, 1024, 4>, grid, block, 0, stream, p);
    }
    return check_launch("layernorm_forward kernel launch");
  }
  // Other rows: a brief CTA for a few of them takes the fewest microseconds, the persistent form moves more bytes a second
  // once there are many (4099 x 1535 f16: 10 us brief, 13 us persistent; 65536 x 1001 bf16 with residual: 141 and 112 us; 65536 x
  // 65: 15 and 24 us).
  if (aligned && p.hidden > 256 && p.rows * (size_t)p.hidden > ((size_t)1 << 24)) {
#define BB200_SHIFTED_ROWS(LANES, COLUMNS, SURE)                                                    \
  if (p.hidden <= (LANES) * (COLUMNS))                                                             \
    return p.residual ? launch_rows<T, ShiftedRows<T, kRowThreads, LANES, COLUMNS, SURE, 2, kMostSmem>, true>(p, stream) : launch_rows<T, ShiftedRows<T, kRowThreads, LANES, COLUMNS, SURE, 1, kMostSmem>, false>(p, stream)
    constexpr int kColumns = 2 * VEC;
    if constexpr (VEC == 8) BB200_SHIFTED_ROWS(32, kColumns, kColumns / 2);
    BB200_SHIFTED_ROWS(64, kColumns, kColumns / 2);
    BB200_SHIFTED_ROWS(128, kColumns, kColumns / 2);
    BB200_SHIFTED_ROWS(256, kColumns, kColumns / 2);
    BB200_SHIFTED_ROWS(512, kColumns, kColumns / 2);
#undef BB200_SHIFTED_ROWS
  }
  if (p.hidden <= 128) return launch_by_element<T, 32, 8, 4, 0>(p, stream);
  if (p.hidden <= 256) return launch_by_element<T, 32, 8, 8, 4>(p, stream);
  if (p.hidden <= 512) return launch_by_element<T, 64, 4, 8, 4>(p, stream);
  if (p.hidden <= 1024) return launch_by_element<T, 128, 2, 8, 4>(p, stream);
  if (p.hidden <= 2048) return launch_by_element<T, 256, 1, 8, 4>(p, stream);
  if (p.hidden <= 4096) return launch_by_element<T, 512, 1, 8, 4>(p, stream);
  if (p.hidden <= 8192) return launch_by_element<T, 1024, 1, 8, 4>(p, stream);
  if constexpr (VEC == 8) {  // rows of f32 end at 16384
    if (p.hidden > 16384) return launch_by_element<T, 1024, 1, 32, 16>(p, stream);
  }
  return launch_by_element<T, 1024, 1, 16, 8>(p, stream);
}

}  // namespace
}  // namespace bb200

using namespace bb200;

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
  for (const void* p : {weight, bias})
    if (misaligned(p, weight_size)) return fail(BB200_E_MISALIGNED, "layernorm_forward: a tensor is not aligned to its element size");
  if (misaligned(mean, 4) || misaligned(rstd, 4)) return fail(BB200_E_MISALIGNED, "layernorm_forward: a tensor is not aligned to its element size");
  // out_resid may be x or residual itself: every element is read by the thread that writes it
  const Range written[] = {{out, row_bytes}, {mean, rows * 4}, {rstd, rows * 4}, {out_resid, row_bytes}};
  const Range read[] = {{x == out_resid ? nullptr : x, row_bytes}, {residual == out_resid ? nullptr : residual, row_bytes},
                        {weight, hidden * weight_size}, {bias, hidden * weight_size}};
  if (clash(written, read) || overlap(out, row_bytes, x, row_bytes) || overlap(out, row_bytes, residual, row_bytes))
    return fail(BB200_E_INVALID_ARGUMENT, "layernorm_forward: an output shares memory with another tensor");
#define BB200_FORWARD(T)                                                                                                          \
  forward<T>({static_cast<const T*>(x), static_cast<const T*>(residual), weight, bias, static_cast<T*>(out), static_cast<T*>(out_resid), \
              mean, rstd, rows, (int)hidden, epsilon, weight_dtype != dtype},                                                 \
             aligned, static_cast<cudaStream_t>(stream))
  switch (dtype) {
    case BB200_BF16: return BB200_FORWARD(__nv_bfloat16);
    case BB200_F16: return BB200_FORWARD(__half);
    default: return BB200_FORWARD(float);
  }
#undef BB200_FORWARD
}
