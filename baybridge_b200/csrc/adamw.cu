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
#include <stdlib.h>

#include <algorithm>

#include "bb200_internal.h"
#include "bb200_rows.cuh"

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
  int access;  // 2: tensors aligned to a thread's eight elements (16 or 32 bytes); 1: to 16 bytes; 0: less
};

// Kernel parameters hold at most 32764 bytes; smaller tables keep the parameter block of ordinary calls short, because every launch
// copies it whole.  Host time of a step with tables of 32, 160 and 512: 8 tensors 8.4, 9.0 and 10.9 us; 32 tensors 9.0, 9.6 and 11.6; 100
// tensors, too many for the first, 11.3 and 13.2; 160 tensors 12.2 and 14.2.
template <int CAPACITY> struct Table {
  const float* schedule;
  float beta1, beta2, one_minus_beta1, one_minus_beta2, log_beta1, log_beta2, epsilon;
  int count;
  Entry entry[CAPACITY];
  unsigned first_tile[CAPACITY + 1];
};
constexpr int kSmallTable = 32, kMiddleTable = 160, kLargeTable = 512;
static_assert(sizeof(Table<kLargeTable>) <= 32764, "the table has to fit the kernel parameters");

struct Step {
  float rate, factor, beta1, beta2, one_minus_beta1, one_minus_beta2, inverse1, inverse2, epsilon;
  // two elements
  __device__ __forceinline__ void update(F2 grad, F2 decay_factor, F2& value, F2& m, F2& v) const {
    const F2 g = grad * both(factor);
    m = fma2(both(beta1), m, both(one_minus_beta1) * g);
    v = fma2(both(beta2), v, both(one_minus_beta2) * g * g);
    float m_low, m_high, v_low, v_high;
    split(m * both(inverse1), m_low, m_high);
    split(v * both(inverse2), v_low, v_high);
    value = fma2(both(-rate), make_f2(m_low / (sqrtf(v_low) + epsilon), m_high / (sqrtf(v_high) + epsilon)), value * decay_factor);
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
  const bool whole = entry.access && at + kVec <= entry.numel, wide = entry.access == 2;
  // the tile's loads are issued before anything waits for the schedule
  Pack<P, kVec> p;
  Pack<G, kVec> g;
  Pack<float, kVec> m, v, master;
  if (whole) {
    g = load_stream_32<G, kVec>(grad + at, wide);
    m = load_stream_32<float, kVec>(entry.exp_avg + at, wide);
    v = load_stream_32<float, kVec>(entry.exp_avg_sq + at, wide);
    if constexpr (MASTERS) master = load_stream_32<float, kVec>(entry.master + at, wide);
    else p = load_stream_32<P, kVec>(param + at, wide);
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
    for (int i = 0; i < kVec / 2; ++i) {
      F2 value = MASTERS ? Pairs<float>::get(master, i) : Pairs<P>::get(p, i);
      F2 m_pair = Pairs<float>::get(m, i), v_pair = Pairs<float>::get(v, i);
      step.update(Pairs<G>::get(g, i), both(decay_factor), value, m_pair, v_pair);
      Pairs<float>::set(m, i, m_pair);
      Pairs<float>::set(v, i, v_pair);
      if constexpr (MASTERS) Pairs<float>::set(master, i, value);
      Pairs<P>::set(p, i, value);
    }
    store_stream_32<float, kVec>(entry.exp_avg + at, m, wide);
    store_stream_32<float, kVec>(entry.exp_avg_sq + at, v, wide);
    if constexpr (MASTERS) store_stream_32<float, kVec>(entry.master + at, master, wide);
    store_stream_32<P, kVec>(param + at, p, wide);
  }
  // the ragged end of a tensor, or tensors that are not 16-byte aligned: neighbouring threads take neighbouring elements
  const unsigned long long tile_end = base + kTileElements < entry.numel ? base + kTileElements : entry.numel;
  const unsigned long long first = entry.access ? tile_end - tile_end % kVec : base;
  for (unsigned long long i = first + threadIdx.x; i < tile_end; i += kThreads) {
    F2 value = both(MASTERS ? entry.master[i] : Conv<float, P>::widen(param[i]));
    F2 one_m = both(entry.exp_avg[i]), one_v = both(entry.exp_avg_sq[i]);
    step.update(both(Conv<float, G>::widen(grad[i])), both(decay_factor), value, one_m, one_v);
    float low, unused;
    split(one_m, low, unused);
    entry.exp_avg[i] = low;
    split(one_v, low, unused);
    entry.exp_avg_sq[i] = low;
    split(value, low, unused);
    if constexpr (MASTERS) entry.master[i] = low;
    param[i] = Conv<float, P>::narrow(low);
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
  DependentLaunch launch(dim3(tiles), dim3(kThreads), 1, 0, stream);
  void* parameters[] = {const_cast<Table<CAPACITY>*>(&table)};  // by address: no copies of the table on the way
  cudaLaunchKernelExC(&launch.config, reinterpret_cast<const void*>(adamw_step<P, G, MASTERS, CAPACITY>), parameters);
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
    const auto vector = [](const void* p, size_t size) { return size == 4 ? aligned32(p) : aligned16(p); };
    const bool sixteen = aligned16(entry.param) && aligned16(entry.grad) && aligned16(entry.exp_avg) && aligned16(entry.exp_avg_sq) &&
                         (!MASTERS || aligned16(entry.master));
    const bool whole = vector(entry.param, sizeof(P)) && vector(entry.grad, sizeof(G)) && aligned32(entry.exp_avg) &&
                       aligned32(entry.exp_avg_sq) && (!MASTERS || aligned32(entry.master));
    entry.access = whole ? 2 : sixteen ? 1 : 0;
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
    return count <= kSmallTable    ? launch_pair<P, G, true, kSmallTable>(call, param_code, grad_code, stream)
           : count <= kMiddleTable ? launch_pair<P, G, true, kMiddleTable>(call, param_code, grad_code, stream)
                                   : launch_pair<P, G, true, kLargeTable>(call, param_code, grad_code, stream);
  return count <= kSmallTable    ? launch_pair<P, G, false, kSmallTable>(call, param_code, grad_code, stream)
         : count <= kMiddleTable ? launch_pair<P, G, false, kMiddleTable>(call, param_code, grad_code, stream)
                                 : launch_pair<P, G, false, kLargeTable>(call, param_code, grad_code, stream);
}

struct Span {
  uintptr_t begin, end;
};

// Refuses tensors that share memory, whichever lists they come from: two CTAs would step the same elements.  The lists are
// sorted by address one by one (mostly they are already: allocated one after the other) and merged where they interleave,
// so a call costs a few passes over them.
int check_disjoint(const Call& call) {
  const void* const* const lists[] = {call.params, call.grads, const_cast<const void* const*>(call.exp_avgs),
                                      const_cast<const void* const*>(call.exp_avg_sqs), const_cast<const void* const*>(call.masters)};
  const size_t used = call.masters ? 5 : 4, count = (size_t)call.count, all = used * count + 1;
  Span* const buffer = static_cast<Span*>(malloc(2 * all * sizeof(Span)));
  if (!buffer) return fail(BB200_E_INVALID_ARGUMENT, "adamw: no host memory for a table of %zu tensors", all);
  Span *spans = buffer, *other = buffer + all;
  const auto before = [](const Span& a, const Span& b) { return a.begin < b.begin; };
  const auto append = [&](size_t have, size_t more, bool rising) {
    Span* added = spans + have;
    if (!rising) std::sort(added, added + more, before);
    if (have && added[0].begin < added[-1].begin) {
      std::merge(spans, added, added, added + more, other, before);
      std::swap(spans, other);
    }
  };
  size_t order[] = {0, 1, 2, 3, 4};  // by the first addresses: lists that lie apart need no merging then
  std::sort(order, order + used, [&](size_t a, size_t b) { return reinterpret_cast<uintptr_t>(lists[a][0]) < reinterpret_cast<uintptr_t>(lists[b][0]); });
  for (size_t k = 0; k < used; ++k) {
    const size_t list = order[k];
    const int* dtypes = list == 0 ? call.param_dtypes : list == 1 ? call.grad_dtypes : nullptr;
    Span* added = spans + k * count;
    bool rising = true;
    uintptr_t last = 0;
    for (size_t i = 0; i < count; ++i) {
      const uintptr_t begin = reinterpret_cast<uintptr_t>(lists[list][i]);
      added[i] = {begin, begin + (dtypes && dtypes[i] != BB200_F32 ? 2 : 4) * call.numels[i]};
      rising &= begin >= last;
      last = begin;
    }
    append(k * count, count, rising);
  }
  const uintptr_t schedule = reinterpret_cast<uintptr_t>(call.schedule);
  spans[all - 1] = {schedule, schedule + 3 * sizeof(float)};
  append(all - 1, 1, true);
  size_t k = 1;
  while (k < all && spans[k - 1].end <= spans[k].begin) ++k;
  const uintptr_t first = spans[k - 1].begin, second = k < all ? spans[k].begin : 0;
  free(buffer);
  if (k == all) return BB200_OK;
  return fail(BB200_E_INVALID_ARGUMENT, "adamw: two of the tensors (the schedule among them) share memory: at %#zx and %#zx", (size_t)first, (size_t)second);
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
    const struct { const void* p; size_t size; } tensors[5] = {{params[i], dtype_bytes((bb200_dtype)p)}, {grads[i], dtype_bytes((bb200_dtype)g)},
                                                               {exp_avgs[i], 4}, {exp_avg_sqs[i], 4}, {masters ? masters[i] : nullptr, 4}};
    for (int a = 0; a < (masters ? 5 : 4); ++a) {
      if (!tensors[a].p) return fail(BB200_E_INVALID_ARGUMENT, "adamw: tensor %d has a null pointer", i);
      if (reinterpret_cast<uintptr_t>(tensors[a].p) % tensors[a].size)
        return fail(BB200_E_MISALIGNED, "adamw: tensor %d is not aligned to its element size", i);
    }
  }
  if (reinterpret_cast<uintptr_t>(schedule) % sizeof(float)) return fail(BB200_E_MISALIGNED, "adamw: the schedule is not aligned to its element size");
  const Call call = {count, numels, param_dtypes, grad_dtypes, weight_decays, params, grads, exp_avgs, exp_avg_sqs, masters, schedule,
                     beta1, beta2, epsilon};
  if (int status = check_disjoint(call)) return status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int status = launch_kind<float, float>(call, BB200_F32, BB200_F32, s)) return status;
  if (int status = launch_kind<__nv_bfloat16, __nv_bfloat16>(call, BB200_BF16, BB200_BF16, s)) return status;
  if (int status = launch_kind<__nv_bfloat16, float>(call, BB200_BF16, BB200_F32, s)) return status;
  if (int status = launch_kind<__half, __half>(call, BB200_F16, BB200_F16, s)) return status;
  return launch_kind<__half, float>(call, BB200_F16, BB200_F32, s);
}
