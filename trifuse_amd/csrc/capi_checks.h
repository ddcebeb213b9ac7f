// Argument checks that the entry points around the block share.
#pragma once

#include <initializer_list>

#include "tfm_internal.h"

namespace tfm {

inline void need_rows(int64_t rows) { need(rows >= 0 && rows <= kMaxRows, "rows out of range"); }

inline void need_storage(int32_t dtype) {
  need(dtype == TFM_DTYPE_BF16 || dtype == TFM_DTYPE_F16, "unknown dtype");
}

// The bytes of one buffer; null or empty ones share memory with nothing.
struct Span {
  const void* at;
  size_t bytes;
};
inline bool meet(const Span& a, const Span& b) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a.at), q = reinterpret_cast<uintptr_t>(b.at);
  return p && q && (p > q ? p - q < b.bytes : q - p < a.bytes) && a.bytes && b.bytes;
}

// No output shares memory with an input or another output.
inline void need_apart(std::initializer_list<Span> outs, std::initializer_list<Span> ins, const char* message) {
  for (const Span* o = outs.begin(); o != outs.end(); ++o) {
    for (const Span& in : ins) need(!meet(*o, in), message);
    for (const Span* other = outs.begin(); other != o; ++other) need(!meet(*o, *other), message);
  }
}

inline size_t size_of(int32_t dtype) { return dtype == TFM_DTYPE_F32 ? 4 : 2; }

}  // namespace tfm
