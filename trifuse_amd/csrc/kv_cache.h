// What the kernels of the 8-bit cache share: which rows a sequence of a batch
// brings, where its tokens lie, and codes in registers.
#pragma once

#include "tfm_device.h"
#include "tfm_internal.h"

namespace tfm {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// A sequence of the batch, by its own table row, length and rows, each held to
// what the arrays have: whatever the device arrays say, no access leaves them.
struct KvSeq {
  int start;  // its first row
  int n;      // its rows
  int first;  // position of its first row (negative: rows before the first token)
  int len;    // its tokens, those rows' own included, that the table has room for: rows from there on have no place
};

__device__ __forceinline__ KvSeq kv_seq(const KvBatchArgs& a, int b) {
  KvSeq s;
  int from, to;
  if (a.starts) {
    from = a.starts[b];
    to = a.starts[b + 1];
  } else {
    from = b * a.max_rows;
    to = from + a.max_rows;
  }
  from = min(max(from, 0), a.rows);
  to = min(max(to, from), a.rows);
  s.start = from;
  s.n = min(to - from, a.max_rows);
  const int tokens = max(a.lengths[b], 0);
  s.first = tokens - s.n;
  s.len = min(tokens, a.table_width << a.page_shift);
  return s;
}

// The page of a sequence's token, or -1: past the table, or an id that no page has.
__device__ __forceinline__ int kv_page(const KvBatchArgs& a, int b, int token) {
  const int at = token >> a.page_shift;
  if (token < 0 || at >= a.table_width) return -1;
  const int page = a.table[(int64_t)b * a.table_width + at];
  return (uint32_t)page < (uint32_t)a.pages ? page : -1;
}

// Codes as halves, in words already XORed with 0x80 a byte, where a code c reads c + 128.
// For keys a byte becomes the subnormal half (c + 128) 2^-24 by itself: one permute for two;
// what 128 adds to a score follows from the sum of q alone.
constexpr float kKeyUnit = 0x1p24f;
__device__ __forceinline__ f16x2_t key_codes_lo(uint32_t w) { return __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0, w, 0x0c010c00u)); }
__device__ __forceinline__ f16x2_t key_codes_hi(uint32_t w) { return __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0, w, 0x0c030c02u)); }
// For values byte N of two words (two tokens' codes of one channel), made c 2^-9 exactly by a
// fused multiply-add; the 128 left in would cost the sums over many tokens their last bits.
constexpr float kValueUnit = 0x1p9f;
template <int N>
__device__ __forceinline__ f16x2_t value_codes(uint32_t a, uint32_t b) {
  const f16x2_t x = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(b, a, 0x0c000c00u | N | (uint32_t)(4 + N) << 16));
  const f16x2_t up = {(_Float16)0x1p15f, (_Float16)0x1p15f}, down = {(_Float16)-0.25f, (_Float16)-0.25f};
  return __builtin_elementwise_fma(x, up, down);
}

}  // namespace tfm
