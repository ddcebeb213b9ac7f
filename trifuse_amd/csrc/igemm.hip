// Product in 8-bit integers with a scale for each token and each channel:
//   out[t, n] = st(float(sum_k x[t, k] w[n, k]) * x_scales[t] * w_scales[n] + bias[n])
// The sum is an exact int32 (K <= 131056 bounds it), so every split of it gives
// the same bits. Both operands are rows of K int8.
//
// igemm_tile_kernel: BM tokens x BN channels a workgroup, 32x32x32 MFMAs. Both
// operands go from memory straight into LDS (16 bytes a lane), 128 bytes of K a
// stage, S stages; a row's eight 16-byte pieces are stored in the order
// piece ^ (row / 2 % 8), so that the 16 rows that are read at a time (256 bytes a
// clock) lie in different banks (row % 8 instead: half of the LDS cycles are
// conflicts, 319 k against 170 k cycles a CU at 8192 x 4096 x 12288; the reads hide
// behind the MFMAs either way, 364 us). Bound: MFMAs, busy 62 % of a CU's cycles at the
// clock that their power leaves, about 1.8 GHz; 2.26 POP/s there, 2.43 at 8192^3 and 16384^3.
#include <type_traits>

#include "tfm_device.h"
#include "tfm_internal.h"
#include "rows.h"

namespace tfm {

namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));

constexpr int kBK = 128;  // bytes of K a stage

__device__ __forceinline__ __amdgpu_buffer_rsrc_t ig_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}

// 16 bytes per lane from a buffer into LDS: lane l writes dst + 16 * l (dst is
// wave-uniform). Out-of-range offsets deliver zeros.
__device__ __forceinline__ void ig_dma16(__amdgpu_buffer_rsrc_t r, int8_t* dst, uint32_t voff, uint32_t soff) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, voff, soff, 0, 0);
#else
  (void)r; (void)dst; (void)voff; (void)soff;
#endif
}

__device__ __forceinline__ i32x16_t mfma_i8(i32x4_t a, i32x4_t b, i32x16_t c) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
#else
  (void)a; (void)b;
  return c;
#endif
}

__device__ __forceinline__ i32x4_t mfma_i8_16(i32x4_t a, i32x4_t b, i32x4_t c) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
#else
  (void)a; (void)b;
  return c;
#endif
}

// All but the last OUT vector memory operations of this wave are done, and its
// LDS reads; then a barrier.
template <int OUT>
__device__ __forceinline__ void stage_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(OUT) : "memory");
}

// One output in the storage type OUT (TFM_DTYPE_*).
template <int OUT>
struct Out {
  using type = std::conditional_t<OUT == TFM_DTYPE_F32, float, uint16_t>;
  __device__ static __forceinline__ void pair(type* to, float a, float b) {
    if constexpr (OUT == TFM_DTYPE_F32) {
      to[0] = a;
      to[1] = b;
    } else {
      const uint32_t p = pack_st2<OUT == TFM_DTYPE_F16>(a, b);
      __builtin_memcpy(to, &p, 4);
    }
  }
  __device__ static __forceinline__ float wide(type v) {
    if constexpr (OUT == TFM_DTYPE_F32) return v;
    else return st2f<OUT == TFM_DTYPE_F16>(v);
  }
};

struct IgArgs {
  const int8_t* x;
  const int8_t* w;
  const float* xs;
  const float* ws;
  const void* bias;
  void* out;
  int T, N, K;
  int mt, nt;     // tiles of the grid
  bool vec_out;   // rows of out start at 16-byte lines
};

// Tile of workgroup `id` of a grid of mt x nt tiles: workgroups go round robin
// to the 8 XCDs, each of which takes a contiguous run of tiles, in bands of
// kBand token tiles walked channel tile by channel tile, so that the tiles an
// XCD works on at a time share rows of both operands in its L2.
constexpr int kXcds = 8, kBand = 8;
__device__ __forceinline__ int2 ig_tile(int id, int mt, int nt) {
  const int tiles = mt * nt, q = tiles / kXcds, r = tiles % kXcds;
  const int xcd = id % kXcds, at = xcd * q + (xcd < r ? xcd : r) + id / kXcds;
  const int band = at / (kBand * nt), left = mt - band * kBand, h = left < kBand ? left : kBand;
  const int in = at - band * kBand * nt;
  return make_int2(band * kBand + in % h, in / h);
}

// PIECE outputs (16 bytes) at column c of a row, those below N.
template <typename T, int PIECE>
__device__ __forceinline__ void store_piece(T* row, int c, int N, bool vec, const T* v) {
  if (vec && c + PIECE <= N) {
    *reinterpret_cast<uint4*>(row + c) = *reinterpret_cast<const uint4*>(v);
  } else {
#pragma unroll
    for (int j = 0; j < PIECE; ++j)
      if (c + j < N) row[c + j] = v[j];
  }
}

// BM x BN tile, waves of WM x WN, S stages, MINW waves a SIMD at least.
template <int BM, int BN, int WM, int WN, int S, int MINW, int OUT>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64, MINW) void igemm_tile_kernel(IgArgs a) {
  constexpr int WAVES_M = BM / WM, WAVES_N = BN / WN, WAVES = WAVES_M * WAVES_N;
  constexpr int MB = WM / 32, NB = WN / 32;
  constexpr int LX = BM / 8 / WAVES, LW = BN / 8 / WAVES;  // 8-row copies a wave makes per stage
  static_assert(WAVES == 4 || WAVES == 8, "a stage array serves one or two waves in the epilogue");
  static_assert(LX * 8 * WAVES == BM && LW * 8 * WAVES == BN, "copies tile the rows");
  // One array a stage and operand, so that reads of one stage do not wait for copies into the other.
  static_assert(S == 2 || S == 4, "stages");
  constexpr int MX = S == 4 ? BM * kBK : 16, MW = S == 4 ? BN * kBK : 16;
  __shared__ __attribute__((aligned(128))) int8_t sx0[BM * kBK], sx1[BM * kBK], sx2[MX], sx3[MX];
  __shared__ __attribute__((aligned(128))) int8_t sw0[BN * kBK], sw1[BN * kBK], sw2[MW], sw3[MW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int2 tile = ig_tile(blockIdx.x, a.mt, a.nt);
  const int m0 = tile.x * BM, n0 = tile.y * BN;
  const int K = a.K, KT = (K + kBK - 1) / kBK;
  const int mrows = a.T - m0 < BM ? a.T - m0 : BM, nrows = a.N - n0 < BN ? a.N - n0 : BN;
  const auto rx = ig_rsrc(a.x + (int64_t)m0 * K, (uint32_t)mrows * (uint32_t)K);
  const auto rw = ig_rsrc(a.w + (int64_t)n0 * K, (uint32_t)nrows * (uint32_t)K);
  // This lane's piece of an 8-row copy. Rows past the matrix are out of the
  // buffer's range and pieces past K are sent there: both read as zeros.
  const int crow = lane >> 3, piece = (lane & 7) ^ ((4 * wave + (crow >> 1)) & 7);  // rows 8 apart by wave, then by 8 * WAVES
  const uint32_t v0 = (uint32_t)((wave * 8 + crow) * K + piece * 16);
  const uint32_t hop = (uint32_t)(WAVES * 8 * K);  // between this wave's copies
  auto load = [&](int8_t* dx, int8_t* dw, int kt) {
    const uint32_t soff = (uint32_t)(kt * kBK), v = (int)soff + piece * 16 >= K ? 0x80000000u : v0;
#pragma unroll
    for (int i = 0; i < LX; ++i) ig_dma16(rx, dx + (i * WAVES + wave) * 8 * kBK, v + i * hop, soff);
#pragma unroll
    for (int i = 0; i < LW; ++i) ig_dma16(rw, dw + (i * WAVES + wave) * 8 * kBK, v + i * hop, soff);
  };
  const int wm = wave % WAVES_M * WM, wn = wave / WAVES_M * WN;
  const int fr = lane & 31, fk = lane >> 5;  // fragment row, its 16-byte half of 32
  i32x4_t fx[2][MB], fw[2][NB];
  auto read = [&](auto buf, const int8_t* sx, const int8_t* sw, int ks) {
    constexpr int B = decltype(buf)::value;
    const int at = fr * kBK + (((2 * ks + fk) ^ ((fr >> 1) & 7)) << 4);
#pragma unroll
    for (int m = 0; m < MB; ++m) fx[B][m] = *reinterpret_cast<const i32x4_t*>(sx + (wm + 32 * m) * kBK + at);
#pragma unroll
    for (int n = 0; n < NB; ++n) fw[B][n] = *reinterpret_cast<const i32x4_t*>(sw + (wn + 32 * n) * kBK + at);
  };
  i32x16_t acc[NB][MB];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[n][m][i] = 0;
  auto mma = [&](auto buf, int from, int to) {
    constexpr int B = decltype(buf)::value;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int m = 0; m < MB; ++m)
        if (n * MB + m >= from && n * MB + m < to) acc[n][m] = mfma_i8(fw[B][n], fx[B][m], acc[n][m]);
  };
  using B0 = std::integral_constant<int, 0>;
  using B1 = std::integral_constant<int, 1>;
  // A step's fragment reads spread over its products.
  auto spread = [&] {
#pragma unroll
    for (int i = 0; i < MB + NB; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, (MB * NB + MB + NB - 1) / (MB + NB), 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // One stage: four steps of 32 bytes of K, each step's fragments read during
  // the one before. The stage's last fragments are in registers before its last
  // step's products: there all waves meet, the next stage is complete, its first
  // fragments are read and this stage's arrays take the stage S later.
  auto stage = [&](int8_t* cx, int8_t* cw, int8_t* nx, int8_t* nw, int kt) {
    constexpr int ALL = MB * NB, FIRST = ALL > MB ? MB : 0;
    read(B1{}, cx, cw, 1);
    mma(B0{}, 0, ALL);
    spread();
    read(B0{}, cx, cw, 2);
    mma(B1{}, 0, ALL);
    spread();
    read(B1{}, cx, cw, 3);
    mma(B0{}, 0, ALL);
    spread();
    mma(B1{}, 0, FIRST);
    // This wave's copies of the next stage are done (later stages' may be
    // outstanding) and so are its reads of this one; then every wave's.
    stage_wait<(S - 2) * (LX + LW)>();
    __builtin_amdgcn_sched_barrier(0);
    read(B0{}, nx, nw, 0);
    load(cx, cw, kt + S);
    mma(B1{}, FIRST, ALL);
#pragma unroll
    for (int i = 0; i < ALL - FIRST; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, (MB + NB + ALL - FIRST - 1) / (ALL - FIRST), 0);
      __builtin_amdgcn_sched_group_barrier(0x020, (LX + LW + ALL - FIRST - 1) / (ALL - FIRST), 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  load(sx0, sw0, 0);
  load(sx1, sw1, 1);
  if constexpr (S == 4) {
    load(sx2, sw2, 2);
    load(sx3, sw3, 3);
  }
  stage_wait<(S - 1) * (LX + LW)>();
  read(B0{}, sx0, sw0, 0);
  // Stages past the last are zeros: the loop ends on a multiple of S.
  for (int kt = 0; kt < KT; kt += S) {
    stage(sx0, sw0, sx1, sw1, kt);
    if constexpr (S == 2) {
      stage(sx1, sw1, sx0, sw0, kt + 1);
    } else {
      stage(sx1, sw1, sx2, sw2, kt + 1);
      stage(sx2, sw2, sx3, sw3, kt + 2);
      stage(sx3, sw3, sx0, sw0, kt + 3);
    }
  }
  stage_wait<0>();  // the copies past the end: the epilogue writes where they land
  // Epilogue. Lane l holds token l % 32 and channels 8 (i / 4) + 4 (l / 32) + i % 4
  // of each 32 x 32 block: scaled and rounded, 32 tokens at a time go through the
  // wave's own part of LDS (every wave is past its last read of it) and leave as
  // 16-byte pieces of rows.
  using O = Out<OUT>;
  using T = typename O::type;
  constexpr int PIECE = 16 / (int)sizeof(T), ROW = WN + PIECE;  // staging row, padded
  constexpr int STAGING = (32 * ROW * (int)sizeof(T) + 8 * WN + 15) / 16 * 16;
  static_assert(STAGING * (WAVES / 4) <= (BM < BN ? BM : BN) * kBK, "the staging fits the arrays");
  int8_t* mine = (wave % 4 == 0 ? sx0 : wave % 4 == 1 ? sx1 : wave % 4 == 2 ? sw0 : sw1) + wave / 4 * STAGING;
  T* st = reinterpret_cast<T*>(mine);
  float* cs = reinterpret_cast<float*>(mine + 32 * ROW * sizeof(T));  // channel scales, then biases
  const T* bias = static_cast<const T*>(a.bias);
  for (int i = lane; i < WN; i += 64) {
    const int c = n0 + wn + i < a.N ? n0 + wn + i : a.N - 1;
    cs[i] = a.ws[c];
    cs[WN + i] = bias ? O::wide(bias[c]) : 0.0f;
  }
  const bool vec = a.vec_out;
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int t0 = m0 + wm + 32 * m, t = t0 + fr;
    const float xs = a.xs[t < a.T ? t : a.T - 1];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        T v[4];
        const int c = 32 * n + 8 * g + 4 * fk;
        const f32x4_t ws = *reinterpret_cast<const f32x4_t*>(cs + c);
        f32x4_t bs = {0.0f, 0.0f, 0.0f, 0.0f};
        if (bias) bs = *reinterpret_cast<const f32x4_t*>(cs + WN + c);
#pragma unroll
        for (int i = 0; i < 4; i += 2)
          O::pair(v + i, (float)acc[n][m][4 * g + i] * xs * ws[i] + bs[i],
                  (float)acc[n][m][4 * g + i + 1] * xs * ws[i + 1] + bs[i + 1]);
        __builtin_memcpy(st + fr * ROW + c, v, sizeof v);
      }
    constexpr int PIECES = WN / PIECE;  // of a row
#pragma unroll
    for (int i = 0; i < 32 * PIECES / 64; ++i) {
      const int at = i * 64 + lane, r = at / PIECES, c = at % PIECES * PIECE;
      T v[PIECE];
      *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(st + r * ROW + c);
      if (t0 + r < a.T)
        store_piece<T, PIECE>(static_cast<T*>(a.out) + (int64_t)(t0 + r) * a.N, n0 + wn + c, a.N, vec, v);
    }
  }
}

// Up to 16 tokens: each wave multiplies 16 channels, whose weights go from memory
// to registers as MFMA operands (16x16x64: lane l holds channel l % 16, bytes
// 16 (l / 16) .. of each 64), with all tokens, whose codes stand in LDS. KS waves
// share 16 channels, every KS-th 64 bytes of K each, and join their sums in LDS.
// With FUSED the codes are made here from x itself, in every workgroup; the first
// weights are on their way meanwhile. Bound: the weights' stream where they are many
// (8 x 2048 x 50304 22.9 us, 4.5 TB/s), else latency (1 x 2048 x 2048 4.9 us).
constexpr int kFewRows = 16;
constexpr int kFewLds = 64 << 10;
constexpr int kFewStep = 64;   // bytes of K an MFMA
constexpr int kFewAhead = 8;   // MFMAs a wave has weights in flight for

__host__ __device__ inline int few_row_bytes(int K) { return (K + kFewStep - 1) / kFewStep * kFewStep + 16; }
inline bool few_fits(int64_t rows, int K) {
  return rows <= kFewRows && rows * (int64_t)few_row_bytes(K) + 8192 + 64 <= kFewLds;
}

template <bool FUSED, bool F16X, int WV, int KS, int OUT>
__global__ __launch_bounds__(64 * WV) void igemm_few_kernel(IgArgs a, const uint16_t* xh) {
  extern __shared__ __attribute__((aligned(16))) int8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int K = a.K, T = a.T, N = a.N;
  const int RB = few_row_bytes(K);  // rows 16 bytes off a multiple of 64: 8 rows of one piece hit different banks
  int8_t* const sx = lds;
  float* const sscale = reinterpret_cast<float*>(lds + T * RB);
  i32x4_t* const spart = reinterpret_cast<i32x4_t*>(lds + (T * RB + 64 + 15) / 16 * 16);
  const int n0 = (blockIdx.x * (WV / KS) + wave / KS) * 16, part = wave % KS;
  const int S = (K + kFewStep - 1) / kFewStep;
  const int row = n0 + (lane & 15) < N ? n0 + (lane & 15) : N - 1;
  const int kc = (lane >> 4) * 16;
  const int8_t* const wp = a.w + (int64_t)row * K + kc;

  i32x4_t w[2][kFewAhead];
  auto load = [&](auto buf, int s0) {
    constexpr int B = decltype(buf)::value;
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int k = (s0 + i * KS) * kFewStep;
      w[B][i] = i32x4_t{0, 0, 0, 0};
      if (k + kc < K) w[B][i] = *reinterpret_cast<const i32x4_t*>(wp + k);
    }
  };
  using B0 = std::integral_constant<int, 0>;
  using B1 = std::integral_constant<int, 1>;
  constexpr int HOP = kFewAhead * KS;
  load(B0{}, part);
  load(B1{}, part + HOP);

  if constexpr (FUSED) {
    for (int t = wave; t < T; t += WV) {
      const RowScale rs = quantize_row_wave<F16X>(xh + (int64_t)t * K, K, sx + t * RB, lane);
      if (lane == 0) sscale[t] = rs.scale;
    }
  } else {
    const int pieces = K / 16;
    for (int i = threadIdx.x; i < T * pieces; i += 64 * WV) {
      const int t = i / pieces, p = i % pieces;
      *reinterpret_cast<uint4*>(sx + t * RB + 16 * p) = *reinterpret_cast<const uint4*>(a.x + (int64_t)t * K + 16 * p);
    }
    if (threadIdx.x < T) sscale[threadIdx.x] = a.xs[threadIdx.x];
  }
  __syncthreads();

  // Columns past the last token repeat it; pieces past K meet zero weights.
  const int col = lane & 15, t = col < T ? col : T - 1;
  const int8_t* const xp = sx + t * RB + kc;
  i32x4_t acc = {0, 0, 0, 0};
  auto mma = [&](auto buf, int s0) {
    constexpr int B = decltype(buf)::value;
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int s = s0 + i * KS;
      if (s < S) acc = mfma_i8_16(w[B][i], *reinterpret_cast<const i32x4_t*>(xp + s * kFewStep), acc);
    }
  };
  for (int s = part; s < S; s += 2 * HOP) {
    mma(B0{}, s);
    load(B0{}, s + 2 * HOP);
    mma(B1{}, s + HOP);
    load(B1{}, s + 3 * HOP);
  }
  if constexpr (KS > 1) {
    if (part) spart[wave * 64 + lane] = acc;
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int p = 1; p < KS; ++p) acc += spart[(wave + p) * 64 + lane];
  }
  if (col >= T) return;
  using O = Out<OUT>;
  typename O::type* out = static_cast<typename O::type*>(a.out) + (int64_t)col * N;
  const typename O::type* bias = static_cast<const typename O::type*>(a.bias);
  const float xs = sscale[col];
  const int c = n0 + 4 * (lane >> 4);
  typename O::type v[4];
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    float f[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = c + i + j < N ? c + i + j : N - 1;
      f[j] = (float)acc[i + j] * xs * a.ws[n] + (bias ? O::wide(bias[n]) : 0.0f);
    }
    O::pair(v + i, f[0], f[1]);
  }
  if (a.vec_out && c + 4 <= N) {
    __builtin_memcpy(__builtin_assume_aligned(out + c, sizeof v), v, sizeof v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < N) out[c + i] = v[i];
  }
}

template <int WV, int KS, typename Kernel>
void launch_few(Kernel kernel, const IgArgs& a, const uint16_t* xh, hipStream_t s) {
  const unsigned groups = (unsigned)((a.N + 15) / 16), blocks = (groups + WV / KS - 1) / (WV / KS);
  const size_t lds = ((size_t)a.T * few_row_bytes(a.K) + 64 + 15) / 16 * 16 + (KS > 1 ? WV * 1024 : 0);
  kernel<<<blocks, 64 * WV, lds, s>>>(a, xh);
}

// Codes made in the kernel.
template <int WV, int KS>
void launch_few_x(int dtype, const IgArgs& a, const uint16_t* xh, hipStream_t s) {
  if (dtype == TFM_DTYPE_F16)
    launch_few<WV, KS>(igemm_few_kernel<true, true, WV, KS, TFM_DTYPE_F16>, a, xh, s);
  else
    launch_few<WV, KS>(igemm_few_kernel<true, false, WV, KS, TFM_DTYPE_BF16>, a, xh, s);
}

// Codes given.
template <int WV, int KS>
void launch_few_codes(int dtype, const IgArgs& a, hipStream_t s) {
  if (dtype == TFM_DTYPE_F32)
    launch_few<WV, KS>(igemm_few_kernel<false, false, WV, KS, TFM_DTYPE_F32>, a, nullptr, s);
  else if (dtype == TFM_DTYPE_F16)
    launch_few<WV, KS>(igemm_few_kernel<false, true, WV, KS, TFM_DTYPE_F16>, a, nullptr, s);
  else
    launch_few<WV, KS>(igemm_few_kernel<false, false, WV, KS, TFM_DTYPE_BF16>, a, nullptr, s);
}

template <int BM, int BN, int WM, int WN, int S, int MINW>
void launch_tile(int dtype, IgArgs a, hipStream_t s) {
  const int64_t mt = ((int64_t)a.T + BM - 1) / BM, nt = ((int64_t)a.N + BN - 1) / BN;
  if (mt * nt > (1 << 22)) fail(TFM_E_UNSUPPORTED, "int8 product: too many output tiles in one call");
  a.mt = (int)mt;
  a.nt = (int)nt;
  const dim3 grid((unsigned)(mt * nt)), block(BM / WM * (BN / WN) * 64);
  if constexpr (BM == BN) {  // the 256 x 192 tile has no room to stage fp32 rows and is not picked for them
    if (dtype == TFM_DTYPE_F32) {
      igemm_tile_kernel<BM, BN, WM, WN, S, MINW, TFM_DTYPE_F32><<<grid, block, 0, s>>>(a);
      return;
    }
  }
  if (dtype == TFM_DTYPE_F16)
    igemm_tile_kernel<BM, BN, WM, WN, S, MINW, TFM_DTYPE_F16><<<grid, block, 0, s>>>(a);
  else
    igemm_tile_kernel<BM, BN, WM, WN, S, MINW, TFM_DTYPE_BF16><<<grid, block, 0, s>>>(a);
}

IgArgs ig_args(int dtype, const int8_t* x, const float* x_scales, int64_t rows, const int8_t* w,
               const float* w_scales, const void* bias, int N, int K, void* out) {
  const size_t size = dtype == TFM_DTYPE_F32 ? 4 : 2;
  const bool vec = (size_t)N * size % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  return IgArgs{x, w, x_scales, w_scales, bias, out, (int)rows, N, K, 0, 0, vec};
}

// Waves that share 16 channels: one where the channels alone fill the chip, else
// four. us with one / four, codes given, four waves a workgroup: 1 x 2048 x 2048
// 7.2 / 4.2, 8 x 4096 x 12288 15.7 / 13.8, 8 x 2048 x 50304 22.6 / 24.8, 16 x 2048 x 50304
// 24.2 / 31.1.
// Waves of a workgroup: sixteen of one each, so that few workgroups make the same
// codes (codes made, 4 / 8 / 16 waves: 8 x 2048 x 50304 25.7 / 24.8 / 23.0, 1 row 22.7 / 21.9 /
// 21.9; right at the border of 32768 channels half of the CUs have no workgroup, codes
// given, 4 x 2048 x 32768: 14.3 / 14.1 / 17.7); of four each four, but eight where four rows or
// more are made into codes for many channels (5 x 4096 x 8192 13.7 / 11.7, 8 x 4096 x 12288
// 18.6 / 16.8, 1 x 4096 x 12288 13.9 / 14.5).
bool few_alone(int N) { return N >= 512 * 64; }

void run_few_x(int dtype, const IgArgs& a, const uint16_t* xh, hipStream_t s) {
  if (few_alone(a.N))
    launch_few_x<16, 1>(dtype, a, xh, s);
  else if (a.T >= 4 && a.N >= 8192)
    launch_few_x<8, 4>(dtype, a, xh, s);
  else
    launch_few_x<4, 4>(dtype, a, xh, s);
}

void run_few_codes(int dtype, const IgArgs& a, hipStream_t s) {
  if (few_alone(a.N))
    launch_few_codes<16, 1>(dtype, a, s);
  else
    launch_few_codes<4, 4>(dtype, a, s);
}

}  // namespace

// The tile whose rounds of the chip take least time by the measured time of a
// round for each 128 bytes of K: 256 x 256 and 256 x 192 (one workgroup a CU)
// 2.0 and 1.62 us, 128 x 128 (two a CU) 1.17, or 0.75 where each CU has one, 64 x 64
// (two a CU) 0.42, or 0.36 and 0.25 in a single round of two and one. us at
// T x K x N, in that order (* the one taken):
//   8192 x 4096 x 12288   364* / 402 / 451 / 654
//   4096 x 2048 x 6144    61.2 / 55.3* / 60.1 / 95
//   8192 x 2048 x 2048    36.0* / 48.9 / 41.3 / 66
//   4096 x 2048 x 2048    30.2 / 27.1 / 22.5* / 34.6
//   2048 x 1536 x 2560    23.6 / 19.8 / 14.9* / 20.1
//   1024 x 2048 x 2048    25.8 / 23.3 / 14.6 / 10.5*
//   64 x 4096 x 12288     39.0 / 34.6 / 22.9 / 11.2*
// The 64 x 64 tile keeps four stages of K in LDS (with two: 18.2 at the last line,
// 11.6 above it): a CU's few workgroups there do not hide each other's loads.
enum Tile { kTile256, kTile192, kTile128, kTile64 };
static Tile pick_tile(int64_t T, int64_t N, bool half_out) {
  auto tiles = [&](int bm, int bn) { return ((T + bm - 1) / bm) * ((N + bn - 1) / bn); };
  auto rounds = [](int64_t n, int slots) { return (double)((n + slots - 1) / slots); };
  const int64_t n128 = tiles(128, 128), n64 = tiles(64, 64);
  const double cost[] = {2.0 * rounds(tiles(256, 256), 256),
                         half_out ? 1.62 * rounds(tiles(256, 192), 256) : 1e30,  // fp32 rows do not fit its staging
                         n128 <= 256 ? 0.75 : 1.17 * rounds(n128, 512),
                         n64 <= 256 ? 0.25 : n64 <= 512 ? 0.36 : 0.42 * rounds(n64, 512)};
  int best = 0;
  for (int i = 1; i < 4; ++i)
    if (cost[i] < cost[best]) best = i;
  return (Tile)best;
}

void launch_int8_qmm(int dtype, const int8_t* x, const float* x_scales, int64_t rows, const int8_t* w,
                     const float* w_scales, const void* bias, int N, int K, void* out, hipStream_t s) {
  if (rows <= 0) return;
  const IgArgs a = ig_args(dtype, x, x_scales, rows, w, w_scales, bias, N, K, out);
  if (few_fits(rows, K)) {
    run_few_codes(dtype, a, s);
  } else {
    switch (pick_tile(rows, N, dtype != TFM_DTYPE_F32)) {
      case kTile256: launch_tile<256, 256, 128, 64, 2, 2>(dtype, a, s); break;
      case kTile192: launch_tile<256, 192, 64, 96, 2, 2>(dtype, a, s); break;
      case kTile128: launch_tile<128, 128, 64, 32, 2, 2>(dtype, a, s); break;
      case kTile64: launch_tile<64, 64, 32, 32, 4, 2>(dtype, a, s); break;
    }
  }
  check_hip(hipGetLastError(), "int8_qmm launch");
}

// Codes made in every workgroup against a launch of their own and the product, us:
//   1 x 2048 x 2048 4.9 / 6.5     8 x 2048 x 2048 6.2 / 7.5     8 x 2048 x 50304 23.8 / 25.4
//   8 x 4096 x 4096 11.1 / 11.1   8 x 7104 x 4096 16.9 / 14.7
// Past 8 rows neither side wins throughout: up to 1.4 less at 16 x 512 and 9 x 2048, as much
// more at 9 x 1536 x 8191 (9.9 / 8.9) and 16 x 1536 x 2560 (8.7 / 8.0), far more for long rows
// (12 x 3520 x 2560 11.7 / 10.5, 9 x 6000 x 2560 20.1 / 13.0).
bool int8_linear_few(int64_t rows, int K) { return rows <= 8 && few_fits(rows, K); }

void launch_int8_linear_few(bool f16, const uint16_t* x, int64_t rows, const int8_t* w, const float* w_scales,
                            const void* bias, int N, int K, void* out, hipStream_t s) {
  if (rows <= 0) return;
  const int dtype = f16 ? TFM_DTYPE_F16 : TFM_DTYPE_BF16;
  run_few_x(dtype, ig_args(dtype, nullptr, nullptr, rows, w, w_scales, bias, N, K, out), x, s);
  check_hip(hipGetLastError(), "int8_linear launch");
}

}  // namespace tfm
