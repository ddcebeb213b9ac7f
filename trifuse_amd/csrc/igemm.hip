// Product in 8-bit integers with a scale for each token and each channel:
//   out[t, n] = st(float(sum_k x[t, k] w[n, k]) * x_scales[t] * w_scales[n] + bias[n])
// The sum is an exact int32 (K <= 131056 bounds it), so every split of it gives
// the same bits. Both operands are rows of K int8.
//
// igemm_tile_kernel: BM tokens x BN channels a workgroup, 32x32x32 MFMAs. Both
// operands go from memory straight into LDS (16 bytes a lane), 128 bytes of K a
// stage, two stages; a row's eight 16-byte pieces are stored in the order
// piece ^ (row % 8), so that the 8 rows a quarter-wave reads lie in different banks.
#include <type_traits>

#include "tfm_device.h"
#include "tfm_internal.h"

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

// One output in the storage type OUT (TFM_DTYPE_*).
template <int OUT>
struct Out {
  using type = std::conditional_t<OUT == TFM_DTYPE_F32, float, uint16_t>;
  __device__ static __forceinline__ type make(float v) {
    if constexpr (OUT == TFM_DTYPE_F32) return v;
    else return f2st<OUT == TFM_DTYPE_F16>(v);
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
};

template <int BM, int BN, int WM, int WN, int OUT>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64) void igemm_tile_kernel(IgArgs a) {
  constexpr int WAVES_M = BM / WM, WAVES_N = BN / WN, WAVES = WAVES_M * WAVES_N;
  constexpr int MB = WM / 32, NB = WN / 32;
  constexpr int LX = BM / 8 / WAVES, LW = BN / 8 / WAVES;  // 8-row copies a wave makes per stage
  static_assert(LX * 8 * WAVES == BM && LW * 8 * WAVES == BN, "copies tile the rows");
  __shared__ __attribute__((aligned(128))) int8_t sx0[BM * kBK], sx1[BM * kBK], sw0[BN * kBK], sw1[BN * kBK];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN;
  const int K = a.K, KT = (K + kBK - 1) / kBK;
  const int mrows = a.T - m0 < BM ? a.T - m0 : BM, nrows = a.N - n0 < BN ? a.N - n0 : BN;
  const auto rx = ig_rsrc(a.x + (int64_t)m0 * K, (uint32_t)mrows * (uint32_t)K);
  const auto rw = ig_rsrc(a.w + (int64_t)n0 * K, (uint32_t)nrows * (uint32_t)K);
  // This lane's piece of an 8-row copy; pieces past K read out of range (zeros).
  const int crow = lane >> 3, piece = (lane & 7) ^ crow;
  auto load = [&](int8_t* dx, int8_t* dw, int kt) {
    const bool past = kt * kBK + piece * 16 >= K;
#pragma unroll
    for (int i = 0; i < LX; ++i) {
      const int r = (i * WAVES + wave) * 8;
      ig_dma16(rx, dx + r * kBK, past ? 0x80000000u : (uint32_t)((r + crow) * K + piece * 16), (uint32_t)(kt * kBK));
    }
#pragma unroll
    for (int i = 0; i < LW; ++i) {
      const int r = (i * WAVES + wave) * 8;
      ig_dma16(rw, dw + r * kBK, past ? 0x80000000u : (uint32_t)((r + crow) * K + piece * 16), (uint32_t)(kt * kBK));
    }
  };
  const int wm = wave % WAVES_M * WM, wn = wave / WAVES_M * WN;
  const int fr = lane & 31, fk = lane >> 5;  // fragment row, its 16-byte half of 32
  auto frag = [&](const int8_t* s, int row, int ks) {
    return *reinterpret_cast<const i32x4_t*>(s + row * kBK + (((2 * ks + fk) ^ (row & 7)) << 4));
  };
  i32x16_t acc[NB][MB];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[n][m][i] = 0;
  auto compute = [&](const int8_t* sx, const int8_t* sw) {
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      i32x4_t fx[MB], fw[NB];
#pragma unroll
      for (int m = 0; m < MB; ++m) fx[m] = frag(sx, wm + 32 * m + fr, ks);
#pragma unroll
      for (int n = 0; n < NB; ++n) fw[n] = frag(sw, wn + 32 * n + fr, ks);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[n][m] = mfma_i8(fw[n], fx[m], acc[n][m]);
    }
  };
  load(sx0, sw0, 0);
  __syncthreads();
  for (int kt = 0; kt < KT; kt += 2) {
    if (kt + 1 < KT) load(sx1, sw1, kt + 1);
    compute(sx0, sw0);
    __syncthreads();
    if (kt + 1 >= KT) break;
    if (kt + 2 < KT) load(sx0, sw0, kt + 2);
    compute(sx1, sw1);
    __syncthreads();
  }
  // Lane l holds token l % 32 and channels 8 (i / 4) + 4 (l / 32) + i % 4 of each 32 x 32 block.
  using O = Out<OUT>;
  typename O::type* out = static_cast<typename O::type*>(a.out);
  const typename O::type* bias = static_cast<const typename O::type*>(a.bias);
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int t = m0 + wm + 32 * m + fr;
    if (t >= a.T) continue;
    const float xs = a.xs[t];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int c = n0 + wn + 32 * n + 8 * (i / 4) + 4 * fk + i % 4;
        if (c < a.N) {
          float v = (float)acc[n][m][i] * xs * a.ws[c];
          if (bias) v += O::wide(bias[c]);
          out[(int64_t)t * a.N + c] = O::make(v);
        }
      }
  }
}

template <int BM, int BN, int WM, int WN>
void launch_tile(int dtype, const IgArgs& a, hipStream_t s) {
  const int64_t mt = ((int64_t)a.T + BM - 1) / BM, nt = ((int64_t)a.N + BN - 1) / BN;
  if (mt > 65535 || nt > (1 << 22)) fail(TFM_E_UNSUPPORTED, "int8 product: too many output tiles in one call");
  const dim3 grid((unsigned)nt, (unsigned)mt), block(BM / WM * (BN / WN) * 64);
  if (dtype == TFM_DTYPE_F32)
    igemm_tile_kernel<BM, BN, WM, WN, TFM_DTYPE_F32><<<grid, block, 0, s>>>(a);
  else if (dtype == TFM_DTYPE_F16)
    igemm_tile_kernel<BM, BN, WM, WN, TFM_DTYPE_F16><<<grid, block, 0, s>>>(a);
  else
    igemm_tile_kernel<BM, BN, WM, WN, TFM_DTYPE_BF16><<<grid, block, 0, s>>>(a);
}

}  // namespace

void launch_int8_qmm(int dtype, const int8_t* x, const float* x_scales, int64_t rows, const int8_t* w,
                     const float* w_scales, const void* bias, int N, int K, void* out, hipStream_t s) {
  if (rows <= 0) return;
  const IgArgs a{x, w, x_scales, w_scales, bias, out, (int)rows, N, K};
  if (rows > 64)
    launch_tile<128, 128, 64, 64>(dtype, a, s);
  else
    launch_tile<64, 64, 32, 32>(dtype, a, s);
  check_hip(hipGetLastError(), "int8_qmm launch");
}

}  // namespace tfm
