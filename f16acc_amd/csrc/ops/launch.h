// What the C entry points share: limits, alignment, the choice of a kernel by type.
#pragma once

#include "common.h"

namespace f16ops {

// Bytes from an element of a row to the last one's end stay below the copies'
// 31-bit offsets.
constexpr int64_t kMaxRow = 1 << 22;  // bytes between rows of a staged operand: 256 rows stay below 2^31
constexpr int64_t kMaxExtent = (int64_t)1 << 40;

inline bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
inline int64_t up128(int64_t v) { return cdiv(v, kBlock) * kBlock; }
inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

inline bool wide_loads(const void* x, int type, int64_t sr, int64_t sc) {
  return sc == 1 && aligned16(x) && sr * type_size(type) % 16 == 0;
}

template <class F>
int by_type(int type, F f) {
  switch (type) {
    case F16ACC_TYPE_F16: return f((f16*)nullptr);
    case F16ACC_TYPE_BF16: return f((bf16*)nullptr);
    case F16ACC_TYPE_F32: return f((float*)nullptr);
  }
  return F16ACC_OPS_E_ARG;
}

inline int quant_check(const void* x, int type, int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0 || type < 0 || type > F16ACC_TYPE_F32) return F16ACC_OPS_E_ARG;
  if (rows > kMaxExtent || cols > kMaxExtent) return F16ACC_OPS_E_UNSUPPORTED;
  if (rows && cols && !x) return F16ACC_OPS_E_ARG;
  return 0;
}

}  // namespace f16ops
