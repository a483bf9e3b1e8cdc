// layernorm_train.h — what the training LayerNorm's forward and backward entry points share (host side).
#pragma once
#include "bb200_internal.h"

namespace bb200 {

inline int check_norm(const char* what, bb200_dtype dtype, bb200_dtype weight_dtype, size_t rows, size_t hidden) {
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

inline bool misaligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

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

}  // namespace bb200
