// adamw.cu — one AdamW step over many tensors for sm_100a, 32-bit moments, optional 32-bit master copies.
//
//   g = grad * factor;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
//   p = p (1 - rate decay) - rate (m / (1 - beta1^step)) / (sqrt(v / (1 - beta2^step)) + eps)
//
// Bound by HBM bytes: 22 per element with 16-bit parameters and gradients, 28 with masters and all-f32 tensors; every
// element is read once and written once.  One launch covers several hundred tensors: their addresses travel in the
// kernel's parameters (so nothing is copied to the device before, and a recorded launch owns its table), and a CTA
// finds its tensor by a binary search over the tensors' first tiles.  rate, step and factor are read from device
// memory.  All arithmetic is fp32; 1 - beta^step is -expm1(step log beta), which keeps its digits for beta near 1.
#include <math.h>

#include "bb200_elementwise.cuh"
#include "bb200_internal.h"

namespace bb200 {
namespace {

constexpr int kThreads = 256, kVec = 8, kTileElements = kThreads * kVec;

struct Entry {
  void* param;
  const void* grad;
  float* exp_avg;
  float* exp_avg_sq;
  float* master;
  unsigned long long numel;
  float decay;
  int vector_ok;  // every tensor 16-byte aligned
};

// Kernel parameters hold at most 32764 bytes; the small table keeps the parameter block of ordinary calls short.
template <int CAPACITY> struct Table {
  const float* schedule;
  float beta1, beta2, one_minus_beta1, one_minus_beta2, log_beta1, log_beta2, epsilon;
  int count;
  Entry entry[CAPACITY];
  unsigned first_tile[CAPACITY + 1];
};
constexpr int kSmallTable = 32, kLargeTable = 512;
static_assert(sizeof(Table<kLargeTable>) <= 32764, "the table has to fit the kernel parameters");

struct Step {
  float rate, factor, beta1, beta2, one_minus_beta1, one_minus_beta2, inverse1, inverse2, epsilon;
  __device__ __forceinline__ void update(float grad, float decay_factor, float& value, float& m, float& v) const {
    const float g = grad * factor;
    m = fmaf(beta1, m, one_minus_beta1 * g);
    v = fmaf(beta2, v, one_minus_beta2 * g * g);
    value = fmaf(-rate, (m * inverse1) / (sqrtf(v * inverse2) + epsilon), value * decay_factor);
  }
};

template <typename P, typename G, bool MASTERS, int CAPACITY>
__global__ void __launch_bounds__(kThreads)
adamw_step(const __grid_constant__ Table<CAPACITY> table) {
  __shared__ float corrections[2];
  dependent_launch_prologue();
  int low = 0, high = table.count - 1;  // the last tensor whose first tile is not behind this one
  while (low < high) {
    const int middle = (low + high + 1) >> 1;
    if (table.first_tile[middle] <= blockIdx.x) low = middle;
    else high = middle - 1;
  }
  const Entry& entry = table.entry[low];
  const unsigned long long base = (unsigned long long)(blockIdx.x - table.first_tile[low]) * kTileElements;
  const unsigned long long at = base + threadIdx.x * kVec;
  P* param = static_cast<P*>(entry.param);
  const G* grad = static_cast<const G*>(entry.grad);
  const bool whole = entry.vector_ok && at + kVec <= entry.numel;
  // the tile's loads are issued before anything waits for the schedule
  Pack<P, kVec> p;
  Pack<G, kVec> g;
  Pack<float, kVec> m, v, master;
  if (whole) {
    g = load_stream<G, kVec>(grad + at);
    m = load_stream<float, kVec>(entry.exp_avg + at);
    v = load_stream<float, kVec>(entry.exp_avg_sq + at);
    if constexpr (MASTERS) master = load_stream<float, kVec>(entry.master + at);
    else p = load_stream<P, kVec>(param + at);
  }
  const float rate = table.schedule[0], count = table.schedule[1], factor = table.schedule[2];
  if (threadIdx.x == 0) corrections[0] = -1.0f / expm1f(count * table.log_beta1);
  if (threadIdx.x == 32) corrections[1] = -1.0f / expm1f(count * table.log_beta2);
  __syncthreads();
  const Step step = {rate, factor, table.beta1, table.beta2, table.one_minus_beta1, table.one_minus_beta2, corrections[0], corrections[1],
                     table.epsilon};
  const float decay_factor = 1.0f - rate * entry.decay;
  if (whole) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      float value = MASTERS ? master.v[e] : Conv<float, P>::widen(p.v[e]);
      step.update(Conv<float, G>::widen(g.v[e]), decay_factor, value, m.v[e], v.v[e]);
      if constexpr (MASTERS) master.v[e] = value;
      p.v[e] = Conv<float, P>::narrow(value);
    }
    store_stream<float, kVec>(entry.exp_avg + at, m);
    store_stream<float, kVec>(entry.exp_avg_sq + at, v);
    if constexpr (MASTERS) store_stream<float, kVec>(entry.master + at, master);
    store_stream<P, kVec>(param + at, p);
  }
  // the ragged end of a tensor, or tensors that are not 16-byte aligned: neighbouring threads take neighbouring elements
  const unsigned long long tile_end = base + kTileElements < entry.numel ? base + kTileElements : entry.numel;
  const unsigned long long first = entry.vector_ok ? tile_end - tile_end % kVec : base;
  for (unsigned long long i = first + threadIdx.x; i < tile_end; i += kThreads) {
    float value = MASTERS ? entry.master[i] : Conv<float, P>::widen(param[i]);
    float one_m = entry.exp_avg[i], one_v = entry.exp_avg_sq[i];
    step.update(Conv<float, G>::widen(grad[i]), decay_factor, value, one_m, one_v);
    entry.exp_avg[i] = one_m;
    entry.exp_avg_sq[i] = one_v;
    if constexpr (MASTERS) entry.master[i] = value;
    param[i] = Conv<float, P>::narrow(value);
  }
}

struct Call {
  int count;
  const size_t* numels;
  const int* param_dtypes;
  const int* grad_dtypes;
  const float* decays;
  void* const* params;
  const void* const* grads;
  void* const* exp_avgs;
  void* const* exp_avg_sqs;
  void* const* masters;
  const float* schedule;
  double beta1, beta2;
  float epsilon;
};

template <typename P, typename G, bool MASTERS, int CAPACITY> int launch_table(const Table<CAPACITY>& table, unsigned tiles, cudaStream_t stream) {
  launch_dependent(adamw_step<P, G, MASTERS, CAPACITY>, dim3(tiles), dim3(kThreads), 0, stream, table);
  return check_launch("adamw kernel launch");
}

// Launches the tensors of one pair of dtypes, as many to a launch as the table holds.
template <typename P, typename G, bool MASTERS, int CAPACITY>
int launch_pair(const Call& call, int param_code, int grad_code, cudaStream_t stream) {
  Table<CAPACITY> table;
  table.schedule = call.schedule;
  table.beta1 = (float)call.beta1;
  table.beta2 = (float)call.beta2;
  table.one_minus_beta1 = (float)(1.0 - call.beta1);
  table.one_minus_beta2 = (float)(1.0 - call.beta2);
  table.log_beta1 = (float)log(call.beta1);
  table.log_beta2 = (float)log(call.beta2);
  table.epsilon = call.epsilon;
  table.count = 0;
  unsigned long long tiles = 0;
  for (int i = 0; i <= call.count; ++i) {
    const bool mine = i < call.count && call.param_dtypes[i] == param_code && call.grad_dtypes[i] == grad_code;
    const unsigned long long more = mine ? ((unsigned long long)call.numels[i] + kTileElements - 1) / kTileElements : 0;
    if (table.count && (i == call.count || (mine && (table.count == CAPACITY || tiles + more > 0x7fffffffull)))) {
      table.first_tile[table.count] = (unsigned)tiles;
      if (int status = launch_table<P, G, MASTERS, CAPACITY>(table, (unsigned)tiles, stream)) return status;
      table.count = 0;
      tiles = 0;
    }
    if (!mine) continue;
    Entry& entry = table.entry[table.count];
    entry.param = call.params[i];
    entry.grad = call.grads[i];
    entry.exp_avg = static_cast<float*>(call.exp_avgs[i]);
    entry.exp_avg_sq = static_cast<float*>(call.exp_avg_sqs[i]);
    entry.master = MASTERS ? static_cast<float*>(call.masters[i]) : nullptr;
    entry.numel = call.numels[i];
    entry.decay = call.decays[i];
    entry.vector_ok = aligned16(entry.param) && aligned16(entry.grad) && aligned16(entry.exp_avg) && aligned16(entry.exp_avg_sq) &&
                      (!MASTERS || aligned16(entry.master));
    table.first_tile[table.count++] = (unsigned)tiles;
    tiles += more;
  }
  return BB200_OK;
}

template <typename P, typename G> int launch_kind(const Call& call, int param_code, int grad_code, cudaStream_t stream) {
  int count = 0;
  for (int i = 0; i < call.count; ++i) count += call.param_dtypes[i] == param_code && call.grad_dtypes[i] == grad_code;
  if (!count) return BB200_OK;
  if (call.masters)
    return count <= kSmallTable ? launch_pair<P, G, true, kSmallTable>(call, param_code, grad_code, stream)
                                : launch_pair<P, G, true, kLargeTable>(call, param_code, grad_code, stream);
  return count <= kSmallTable ? launch_pair<P, G, false, kSmallTable>(call, param_code, grad_code, stream)
                              : launch_pair<P, G, false, kLargeTable>(call, param_code, grad_code, stream);
}

}  // namespace
}  // namespace bb200

using namespace bb200;

extern "C" int bb200_adamw(int count, const size_t* numels, const int* param_dtypes, const int* grad_dtypes, const float* weight_decays,
                           void* const* params, const void* const* grads, void* const* exp_avgs, void* const* exp_avg_sqs,
                           void* const* masters, const float* schedule, double beta1, double beta2, float epsilon, void* stream) {
  if (count < 1) return fail(BB200_E_INVALID_ARGUMENT, "adamw: at least one tensor is needed (got %d)", count);
  if (!numels || !param_dtypes || !grad_dtypes || !weight_decays || !params || !grads || !exp_avgs || !exp_avg_sqs || !schedule)
    return fail(BB200_E_INVALID_ARGUMENT, "adamw: null array");
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0) || !(epsilon >= 0.0f))
    return fail(BB200_E_INVALID_ARGUMENT, "adamw: betas must lie in [0, 1) and epsilon must not be negative");
  for (int i = 0; i < count; ++i) {
    const int p = param_dtypes[i], g = grad_dtypes[i];
    if ((p != BB200_F32 && p != BB200_BF16 && p != BB200_F16) || (g != p && g != BB200_F32))
      return fail(BB200_E_INVALID_ARGUMENT, "adamw: tensor %d has dtypes %d and %d; parameters are bf16/f16/f32, gradients alike or f32", i, p, g);
    if (numels[i] == 0) return fail(BB200_E_INVALID_ARGUMENT, "adamw: tensor %d is empty", i);
    if (numels[i] > (size_t)kTileElements * 0x7fffffffu) return fail(BB200_E_UNSUPPORTED_SHAPE, "adamw: tensor %d is too large", i);
    const size_t param_bytes = numels[i] * dtype_bytes((bb200_dtype)p), grad_bytes = numels[i] * dtype_bytes((bb200_dtype)g), wide = numels[i] * 4;
    const struct { const void* p; size_t bytes, size; } tensors[5] = {
        {params[i], param_bytes, dtype_bytes((bb200_dtype)p)}, {exp_avgs[i], wide, 4}, {exp_avg_sqs[i], wide, 4},
        {masters ? masters[i] : nullptr, wide, 4}, {grads[i], grad_bytes, dtype_bytes((bb200_dtype)g)}};
    for (int a = 0; a < 5; ++a) {
      if (!tensors[a].p && !(a == 3 && !masters)) return fail(BB200_E_INVALID_ARGUMENT, "adamw: tensor %d has a null pointer", i);
      if (reinterpret_cast<uintptr_t>(tensors[a].p) % tensors[a].size)
        return fail(BB200_E_MISALIGNED, "adamw: tensor %d is not aligned to its element size", i);
      for (int b = 0; b < a; ++b)
        if (overlap(tensors[a].p, tensors[a].bytes, tensors[b].p, tensors[b].bytes))
          return fail(BB200_E_INVALID_ARGUMENT, "adamw: two of the tensors number %d share memory", i);
    }
  }
  const Call call = {count, numels, param_dtypes, grad_dtypes, weight_decays, params, grads, exp_avgs, exp_avg_sqs, masters, schedule,
                     beta1, beta2, epsilon};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int status = launch_kind<float, float>(call, BB200_F32, BB200_F32, s)) return status;
  if (int status = launch_kind<__nv_bfloat16, __nv_bfloat16>(call, BB200_BF16, BB200_BF16, s)) return status;
  if (int status = launch_kind<__nv_bfloat16, float>(call, BB200_BF16, BB200_F32, s)) return status;
  if (int status = launch_kind<__half, __half>(call, BB200_F16, BB200_F16, s)) return status;
  return launch_kind<__half, float>(call, BB200_F16, BB200_F32, s);
}
