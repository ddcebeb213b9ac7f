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
  int len;    // its tokens, those rows' own included
  __device__ int first() const { return len - n; }  // position of its first row (negative: rows before the first token)
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
  s.len = min(max(a.lengths[b], 0), a.table_width << a.page_shift);
  return s;
}

// The page of a sequence's token, or -1: past the table, or an id that no page has.
__device__ __forceinline__ int kv_page(const KvBatchArgs& a, int b, int token) {
  const int at = token >> a.page_shift;
  if (token < 0 || at >= a.table_width) return -1;
  const int page = a.table[(int64_t)b * a.table_width + at];
  return (uint32_t)page < (uint32_t)a.pages ? page : -1;
}

// Codes to half, exactly: with c ^ 0x80 = c + 128 as the low byte of 0x6400 a half
// reads 1024 + (c + 128), and 1152 less is c. `w` holds four codes already XORed
// with 0x80; two halves a call, from bytes 0 and 1 or 2 and 3.
__device__ __forceinline__ f16x2_t minus1152(uint32_t w) {
  return __builtin_bit_cast(f16x2_t, w) - f16x2_t{(_Float16)1152.0f, (_Float16)1152.0f};
}
__device__ __forceinline__ f16x2_t codes_lo(uint32_t w) { return minus1152(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)); }
__device__ __forceinline__ f16x2_t codes_hi(uint32_t w) { return minus1152(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)); }
// Byte n of two words (two keys' codes of one channel).
template <int N>
__device__ __forceinline__ f16x2_t codes_of(uint32_t a, uint32_t b) {
  return minus1152(__builtin_amdgcn_perm(b, a, 0x0c000c00u | N | (uint32_t)(4 + N) << 16) | 0x64006400u);
}

}  // namespace tfm
