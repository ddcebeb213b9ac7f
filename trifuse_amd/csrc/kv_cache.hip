// Writing tokens into the paged cache of 8-bit codes, and reading them back.
//
// A page and head has one scale. Tokens that come to it take it along or raise it:
//   s' = max(s, max|x| / 127), old codes c' = round(c * s / s'), new codes round(x / s')
// (s = 0 where the page starts with them). One workgroup owns a page of a head, for keys
// or for values: it holds the new tokens in registers between the maximum and the codes,
// so k and v are read once; old codes are touched only where the scale grows. Keys are
// turned to their positions on the way.
//
// Bound: memory (2 bytes in and 1 out an element), and at a token a sequence the launch.
#include "kv_cache.h"
#include "rotary.h"
#include "rows.h"

namespace tfm {

namespace {

__device__ __forceinline__ uint2 pack_codes(const float* x, float inverse, bool good) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int c = good ? (int)__builtin_rintf(x[j] * inverse) : 0;
    w[j / 4] |= (uint32_t)(c & 0xff) << (8 * (j & 3));
  }
  return make_uint2(w[0], w[1]);
}

// An item is 16 channels of a token: two vectors of eight, which are the halves of
// eight pairs where those are turned. NI items a thread cover a whole page. One wave a page
// (NT = 64): four pages a workgroup. A workgroup passes over HEADS heads of its pages, whose
// angles are the same.
template <bool F16, int D, int NT, int NI, int HEADS>
__global__ __launch_bounds__(NT == 64 ? 256 : NT) void cache_append_kernel(KvAppendArgs a, int slots) {
  __shared__ uint32_t most[2][(NT + 63) / 64];
  constexpr int PAGES = NT == 64 ? 4 : 1;
  const KvBatchArgs& g = a.b;
  const int thread = threadIdx.x % NT, unit = blockIdx.x * PAGES + threadIdx.x / NT;
  const int b = unit / slots;
  if (b >= g.sequences) return;
  const bool values = blockIdx.z != 0;
  const KvSeq s = kv_seq(g, b);
  if (s.first >= s.len) return;  // no row has a place
  const int page_tokens = 1 << g.page_shift;
  const int at = (max(s.first, 0) >> g.page_shift) + unit % slots;  // table entry
  const int base = at << g.page_shift;
  const int begin = max(max(s.first, 0), base), end = min(s.len, base + page_tokens);
  if (begin >= end) return;
  const int held = begin - base;  // tokens of the page that stay

  const uint16_t* x = values ? a.v : a.k;
  const int64_t row_stride = values ? a.v_row : a.k_row, head_stride = values ? a.v_head : a.k_head;
  const bool rotate = !values && a.frequencies;
  const int per = D / 16, turned = rotate ? a.pairs / 8 : 0;  // items a token, and those with pairs
  const int items = (end - begin) * per;
  const bool halves = !a.interleaved;
  auto channels = [&](int c, int& d0, int& d1) {
    if (c < turned && halves) {
      d0 = 8 * c;
      d1 = d0 + a.pairs;
    } else {
      d0 = 16 * c;  // behind `turned` items of halves lie 16 channels each, too
      d1 = d0 + 8;
    }
  };
  Vec8 raw[NI][2];
  auto fetch = [&](int head) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int item = thread + i * NT;
      if (item < items) {
        const uint16_t* row = x + (int64_t)(s.start + begin + item / per - s.first) * row_stride + head * head_stride;
        int d0, d1;
        channels(item % per, d0, d1);
        raw[i][0] = load8<true>(row + d0, 8);
        raw[i][1] = load8<true>(row + d1, 8);
      }
    }
  };
  // The tokens are on their way while the page is looked up and the angles are made.
  const int head0 = blockIdx.y * HEADS;
  fetch(head0);
  const int page = kv_page(g, b, begin);
  if (page < 0) return;
  float2 turn[NI][8];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int item = thread + i * NT, token = begin + item / per, c = item % per;
    if (item < items && c < turned) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        turn[i][j] = turn_cos_sin((double)token * (a.frequencies[8 * c + j] * kTurnsPerRadian), a.scale);
    }
  }
#pragma unroll 1
  for (int h = 0; h < HEADS && head0 + h < g.kv_heads; ++h) {
    const int64_t place = (int64_t)page * g.kv_heads + head0 + h;
    int8_t* codes = (values ? g.v : g.k) + (place << g.page_shift) * D;
    float* scale = (values ? g.v_scales : g.k_scales) + place;
    const float before = held > 0 ? *scale : 0.0f;
    float v[NI][16];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int item = thread + i * NT;
      if (item < items) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[i][j] = elem<F16>(raw[i][0], j);
          v[i][8 + j] = elem<F16>(raw[i][1], j);
        }
        if (item % per < turned) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 t = turn[i][j];
            float& x1 = v[i][halves ? j : 2 * j];
            float& x2 = v[i][halves ? 8 + j : 2 * j + 1];
            const float y1 = __builtin_fmaf(x1, t.x, -(x2 * t.y)), y2 = __builtin_fmaf(x2, t.x, x1 * t.y);
            x1 = y1;
            x2 = y2;
          }
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(v[i][j]) & 0x7fffffffu);
      }
    }
    if (h + 1 < HEADS && head0 + h + 1 < g.kv_heads) fetch(head0 + h + 1);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, kWave));
    if (NT > 64) {
      if ((thread & 63) == 0) most[h & 1][thread >> 6] = top;
      __syncthreads();  // behind every thread's read of the old scale, too
#pragma unroll
      for (int w = 0; w < (NT + 63) / 64; ++w) top = max(top, most[h & 1][w]);
    }
    const bool good = top < 0x7f800000u && before == before;
    const float now = good ? fmaxf(before, fmaxf(__uint_as_float(top), 0x1p-40f) / 127.0f) : __builtin_nanf("");
    const float inverse = 1.0f / now;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int item = thread + i * NT;
      if (item < items) {
        const int token = begin + item / per, c = item % per;
        int8_t* to = codes + (token - base) * D;
        int d0, d1;
        channels(c, d0, d1);
        *reinterpret_cast<uint2*>(to + d0) = pack_codes(v[i], inverse, good);
        *reinterpret_cast<uint2*>(to + d1) = pack_codes(v[i] + 8, inverse, good);
      }
    }
    if (held > 0 && now > before) {
      const float ratio = before / now;
      for (int i = thread; i < held * (D / 16); i += NT) {
        uint4* at16 = reinterpret_cast<uint4*>(codes) + i;
        const uint4 old = *at16;
        uint32_t w[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t r = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int c = (int8_t)(w[j] >> (8 * k));
            r |= (uint32_t)((int)__builtin_rintf((float)c * ratio) & 0xff) << (8 * k);
          }
          w[j] = r;
        }
        *at16 = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    if (thread == 0) *scale = now;
  }
}

template <typename T>
__device__ __forceinline__ void put4(T* p, const float* v);
template <>
__device__ __forceinline__ void put4<float>(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <>
__device__ __forceinline__ void put4<__bf16>(__bf16* p, const float* v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}
template <>
__device__ __forceinline__ void put4<_Float16>(_Float16* p, const float* v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]));
}

// A thread reads 16 codes of a token and head.
template <typename T, int D>
__global__ __launch_bounds__(256) void cache_read_kernel(KvBatchArgs g, T* k, T* v) {
  constexpr int per = D / 16;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / (per * g.kv_heads);
  if (row >= (int64_t)g.rows) return;
  const int b = row / g.max_rows, c = i % per, head = i / per % g.kv_heads;
  const KvSeq s = kv_seq(g, b);
  const int token = s.first + (int)(row - s.start);
  const int page = kv_page(g, b, token);
  const bool values = blockIdx.y != 0;
  T* to = (values ? v : k) + i * 16;
  float scale = 0.0f;
  uint32_t w[4] = {0, 0, 0, 0};
  if (page >= 0) {
    const int64_t place = (int64_t)page * g.kv_heads + head;
    scale = (values ? g.v_scales : g.k_scales)[place];
    const int64_t at = ((place << g.page_shift) + (token & ((1 << g.page_shift) - 1))) * D + 16 * c;
    const uint4 u = *reinterpret_cast<const uint4*>((values ? g.v : g.k) + at);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float x[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) x[n] = (float)(int8_t)(w[j] >> (8 * n)) * scale;
    put4(to + 4 * j, x);
  }
}

template <typename T>
void read_as(int head_dim, const KvBatchArgs& b, void* k, void* v, hipStream_t s) {
  const int64_t items = (int64_t)b.rows * b.kv_heads * (head_dim / 16);
  const dim3 grid((uint32_t)((items + 255) / 256), 2);
  auto* kernel = head_dim == 64 ? cache_read_kernel<T, 64> : cache_read_kernel<T, 128>;
  tfm_launch(kernel, grid, dim3(256), 0, s, b, static_cast<T*>(k), static_cast<T*>(v));
}

// Threads by the items of a page, so that NI <= 2 (32 registers of values).
template <bool F16, int D, int HEADS>
void append(const KvAppendArgs& a, uint32_t units, int slots, hipStream_t s) {
  auto go = [&](auto* kernel, int threads, int pages = 1) {
    tfm_launch(kernel, dim3((units + pages - 1) / pages, (a.b.kv_heads + HEADS - 1) / HEADS, 2), dim3(threads), 0, s, a, slots);
  };
  switch ((D / 16) << a.b.page_shift) {
    case 64: go(cache_append_kernel<F16, D, 64, 1, HEADS>, 256, 4); break;
    case 128: go(cache_append_kernel<F16, D, 128, 1, HEADS>, 128); break;
    case 256: go(cache_append_kernel<F16, D, 256, 1, HEADS>, 256); break;
    case 512: go(cache_append_kernel<F16, D, 256, 2, HEADS>, 256); break;
    case 1024: go(cache_append_kernel<F16, D, 512, 2, HEADS>, 512); break;
    default: go(cache_append_kernel<F16, D, 1024, 2, HEADS>, 1024);
  }
}
template <bool F16, int D>
void append(const KvAppendArgs& a, hipStream_t s) {
  const int page = 1 << a.b.page_shift;
  const int slots = (a.b.max_rows + page - 2) / page + 1;  // pages that max_rows tokens can meet
  const uint32_t units = (uint32_t)a.b.sequences * slots;
  // Enough waves: two or four heads share their angles. Tokens of 16 heads of 128, written, us with 1, 2 and 4: 4000
  // in pages of 16 (16000 waves) 17.5, 16.9, 15.2; in pages of 256, two items a thread (8700) 20.9, 18.6, 24.3, of 64
  // (8200) 17.5, 18.4, 17.2; 1200 in pages of 16 (8200) 10.2, 9.8, 12.1, of 64 (6100) 11.2, 11.9, 15.4.
  const int items = page * D / 16, threads = items <= 256 ? items : items / 2;
  const int64_t waves = (int64_t)units * a.b.kv_heads * 2 * (threads / 64);
  if (waves >= 12288)
    append<F16, D, 4>(a, units, slots, s);
  else if (waves > (items <= 256 ? 7168 : 8192))
    append<F16, D, 2>(a, units, slots, s);
  else
    append<F16, D, 1>(a, units, slots, s);
}

}  // namespace

void launch_cache_append(bool f16, int head_dim, const KvAppendArgs& a, hipStream_t s) {
  if (head_dim == 64)
    f16 ? append<true, 64>(a, s) : append<false, 64>(a, s);
  else
    f16 ? append<true, 128>(a, s) : append<false, 128>(a, s);
  check_hip(hipGetLastError(), "cache_append launch");
}

void launch_cache_read(int dtype, int head_dim, const KvBatchArgs& b, void* k, void* v, hipStream_t s) {
  if (dtype == TFM_DTYPE_F32)
    read_as<float>(head_dim, b, k, v, s);
  else if (dtype == TFM_DTYPE_F16)
    read_as<_Float16>(head_dim, b, k, v, s);
  else
    read_as<__bf16>(head_dim, b, k, v, s);
  check_hip(hipGetLastError(), "cache_read launch");
}

}  // namespace tfm
