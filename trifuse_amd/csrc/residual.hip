// The step between two blocks of a decoder layer, and rows to 8-bit codes.
//
// norm_residual: with y a block's output and r the residual stream,
//   b = y,  or  y * rsqrt(mean(y^2) + post_eps) * w_post     (post norm)
//   h = r + m * g * b                                         (gate g, residual multiplier m)
//   x = h * rsqrt(mean(h^2) + pre_eps) * w_pre                (the next block's pre norm)
// x is taken from h before h is rounded, and each output is rounded once, to
// the storage dtype (h, x) or to codes (below). Everything between is fp32.
//
// Codes of a row x: a = max(max|x|, 2^-100), scale = a / 127,
//   code = round_half_even(x * (127 / a)), in [-127, 127];
// a row that holds an infinity or a NaN gets codes 0 and scale NaN, so that
// its products are NaN. The floor on a keeps 127 / a finite; a zero row has
// codes 0.
//
// Bound: memory (y, r in, h, x out: 8 bytes an element). A team of lanes owns
// a row and keeps it in registers from the loads to the stores, so every
// byte moves once; both norms' sums are a lane's own sequential sum, then
// the pairwise tree over the wave, then the waves in order. The team follows
// from the width alone, so that a row has the same bits in every batch (four waves
// a row of 2048: 16 rows 3.2 against 4.0 us, 300 rows 3.7 against 4.3, 4096 rows 14.7
// against 14.2). 16384 x 2048 with a gate for each element 60 us, 5.6 TB/s; without
// one, to codes, 40 us; quantize_rows of the same 16.5 us, 6.1 TB/s.
#include <type_traits>

#include "tfm_device.h"
#include "tfm_internal.h"
#include "rows.h"

namespace tfm {

namespace {

struct NormArgs {
  tfm_norm_step s;
  int rows, width;
};

// TEAM lanes a row, NV vectors of eight elements a lane (vector i of lane l
// holds elements 8 * (l + TEAM * i) ..). Teams of 64 share a workgroup of four.
template <int TEAM, int NV, bool F16, bool UNALIGNED>
__global__ __launch_bounds__(TEAM < 256 ? 256 : TEAM) void norm_residual_kernel(NormArgs a) {
  __shared__ float part0[16], part1[16];
  __shared__ uint32_t part2[16];
  constexpr int TEAMS = TEAM < 256 ? 256 / TEAM : 1;
  const int lane = threadIdx.x % TEAM;
  const int t = blockIdx.x * TEAMS + threadIdx.x / TEAM;
  if (t >= a.rows) return;  // whole waves, and no barrier with several teams
  const int H = a.width;
  const int64_t base = (int64_t)t * H;
  const uint16_t* y = static_cast<const uint16_t*>(a.s.y) + base;
  const uint16_t* r = a.s.residual ? static_cast<const uint16_t*>(a.s.residual) + base : nullptr;
  const uint16_t* wpost = static_cast<const uint16_t*>(a.s.post_weight);
  const uint16_t* wpre = static_cast<const uint16_t*>(a.s.pre_weight);
  const int gk = a.s.gate_kind;
  const uint16_t* gate = gk == TFM_GATE_FULL      ? static_cast<const uint16_t*>(a.s.gate) + base
                         : gk == TFM_GATE_CHANNEL ? static_cast<const uint16_t*>(a.s.gate)
                                                  : nullptr;
  // Every operand is on its way before the first is used, but the weights of the
  // widest rows, whose registers are full without them.
  constexpr bool EARLY = TEAM < 1024;
  Vec8 yv[NV], rv[NV], gv[NV], av[NV], bv[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (lane + TEAM * i);
    yv[i] = load8<UNALIGNED>(y + c, H - c);
  }
  if (r) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (lane + TEAM * i);
      rv[i] = load8<UNALIGNED>(r + c, H - c);
    }
  }
  if (gate) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (lane + TEAM * i);
      gv[i] = load8<UNALIGNED>(gate + c, H - c);
    }
  }
  if (EARLY && wpost) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (lane + TEAM * i);
      av[i] = load8<UNALIGNED>(wpost + c, H - c);
    }
  }
  if (EARLY && wpre) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (lane + TEAM * i);
      bv[i] = load8<UNALIGNED>(wpre + c, H - c);
    }
  }
  auto weight = [&](const Vec8* early, const uint16_t* w, int i) {
    const int c = 8 * (lane + TEAM * i);
    return EARLY ? early[i] : load8<UNALIGNED>(w + c, H - c);
  };
  const float m = gk == TFM_GATE_TOKEN ? a.s.residual_multiplier * static_cast<const float*>(a.s.gate)[t]
                                       : a.s.residual_multiplier;

  float h[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) h[i][j] = elem<F16>(yv[i], j);
  if (wpost) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s = __builtin_fmaf(h[i][j], h[i][j], s);
    const float inv = 1.0f / sqrtf(team_sum<TEAM>(s, part0) / (float)H + a.s.post_eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Vec8 w = weight(av, wpost, i);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] = h[i][j] * inv * elem<F16>(w, j);
    }
  }
  if (gate) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] *= elem<F16>(gv[i], j);
  }
  if (r) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] = __builtin_fmaf(m, h[i][j], elem<F16>(rv[i], j));
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] *= m;
  }
  // h may be written over y or r: this lane's elements of both are in registers.
  if (a.s.h) {
    uint16_t* out = static_cast<uint16_t*>(a.s.h) + base;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (lane + TEAM * i);
      Vec8 o;
#pragma unroll
      for (int k = 0; k < 4; ++k) o.w[k] = pack_st2<F16>(h[i][2 * k], h[i][2 * k + 1]);
      store8<UNALIGNED>(out + c, o, H - c);
    }
  }
  if (!wpre) return;

  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __builtin_fmaf(h[i][j], h[i][j], s);
  const float inv = 1.0f / sqrtf(team_sum<TEAM>(s, part1) / (float)H + a.s.pre_eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Vec8 w = weight(bv, wpre, i);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[i][j] = h[i][j] * inv * elem<F16>(w, j);
  }
  if (a.s.x) {
    uint16_t* out = static_cast<uint16_t*>(a.s.x) + base;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (lane + TEAM * i);
      Vec8 o;
#pragma unroll
      for (int k = 0; k < 4; ++k) o.w[k] = pack_st2<F16>(h[i][2 * k], h[i][2 * k + 1]);
      store8<UNALIGNED>(out + c, o, H - c);
    }
  }
  if (a.s.codes) {
    // Elements past the row are exact zeros unless inv or m is not finite;
    // they take no part in the row's largest magnitude.
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t u = __float_as_uint(h[i][j]) & 0x7fffffffu;
        if (u > big && 8 * (lane + TEAM * i) + j < H) big = u;
      }
    const RowScale rs = row_scale(team_umax<TEAM>(big, part2));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (lane + TEAM * i);
      store_codes8<UNALIGNED>(a.s.codes + base + c, codes8(h[i], rs), H - c);
    }
    if (lane == 0) a.s.scales[t] = rs.scale;
  }
}

template <int TEAM, int NV, bool F16, bool UNALIGNED>
__global__ __launch_bounds__(TEAM < 256 ? 256 : TEAM) void quantize_kernel(const uint16_t* __restrict__ x, int rows,
                                                                           int H, int8_t* __restrict__ codes,
                                                                           float* __restrict__ scales) {
  __shared__ uint32_t part[16];
  constexpr int TEAMS = TEAM < 256 ? 256 / TEAM : 1;
  const int lane = threadIdx.x % TEAM;
  const int t = blockIdx.x * TEAMS + threadIdx.x / TEAM;
  if (t >= rows) return;  // whole waves, and no barrier with several teams
  const int64_t base = (int64_t)t * H;
  // The widest rows do not fit their registers: read again (from the cache).
  constexpr bool HOLD = TEAM < 1024;
  Vec8 v[NV];
  u16x2_t big = {0, 0};
#pragma unroll HOLD ? NV : 4
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (lane + TEAM * i);
    const Vec8 u = load8<UNALIGNED>(x + base + c, H - c);
    if constexpr (HOLD) v[i] = u;
    big = abs_max(big, u);
  }
  const RowScale rs = row_scale(team_umax<TEAM>(abs_bits<F16>(big), part));
#pragma unroll HOLD ? NV : 4
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (lane + TEAM * i);
    Vec8 u;
    if constexpr (HOLD)
      u = v[i];
    else
      u = load8<UNALIGNED>(x + base + c, H - c);
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = elem<F16>(u, j);
    store_codes8<UNALIGNED>(codes + base + c, codes8(f, rs), H - c);
  }
  if (lane == 0) scales[t] = rs.scale;
}

bool aligned(const void* p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Calls f(TEAM, NV) as compile-time constants: one wave a row up to 2048
// elements, four up to 8192, sixteen beyond.
template <int MAXNV, typename F>
void by_width(int H, F&& f) {
  const int v = (H + 7) / 8;
  using std::integral_constant;
  if (v <= 64)
    f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (v <= 128)
    f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (v <= 192)
    f(integral_constant<int, 64>{}, integral_constant<int, 3>{});
  else if (v <= 256)
    f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  else if (v <= 512)
    f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (v <= 1024)
    f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  else
    f(integral_constant<int, 1024>{}, integral_constant<int, MAXNV>{});
}

}  // namespace

void launch_norm_residual(bool f16, const tfm_norm_step& st, int rows, int width, hipStream_t s) {
  if (rows <= 0) return;
  const bool full_gate = st.gate_kind == TFM_GATE_FULL || st.gate_kind == TFM_GATE_CHANNEL;
  const bool plain = width % 8 == 0 && aligned(st.y, 16) && aligned(st.residual, 16) && aligned(st.post_weight, 16) &&
                     (!full_gate || aligned(st.gate, 16)) && aligned(st.pre_weight, 16) && aligned(st.h, 16) &&
                     aligned(st.x, 16) && aligned(st.codes, 8);
  const NormArgs a{st, rows, width};
  by_width<4>(width, [&](auto team, auto nv) {
    constexpr int TEAM = decltype(team)::value, NV = decltype(nv)::value;
    constexpr int threads = TEAM < 256 ? 256 : TEAM, teams = threads / TEAM;
    const unsigned blocks = (unsigned)((rows + teams - 1) / teams);
    if (f16 && plain)
      norm_residual_kernel<TEAM, NV, true, false><<<blocks, threads, 0, s>>>(a);
    else if (f16)
      norm_residual_kernel<TEAM, NV, true, true><<<blocks, threads, 0, s>>>(a);
    else if (plain)
      norm_residual_kernel<TEAM, NV, false, false><<<blocks, threads, 0, s>>>(a);
    else
      norm_residual_kernel<TEAM, NV, false, true><<<blocks, threads, 0, s>>>(a);
  });
  check_hip(hipGetLastError(), "norm_residual launch");
}

void launch_quantize_rows(bool f16, const uint16_t* x, int rows, int width, int8_t* codes, float* scales,
                          hipStream_t s) {
  if (rows <= 0) return;
  const bool plain = width % 8 == 0 && aligned(x, 16) && aligned(codes, 8);
  by_width<16>(width, [&](auto team, auto nv) {
    constexpr int TEAM = decltype(team)::value, NV = decltype(nv)::value;
    constexpr int threads = TEAM < 256 ? 256 : TEAM, teams = threads / TEAM;
    const unsigned blocks = (unsigned)((rows + teams - 1) / teams);
    if (f16 && plain)
      quantize_kernel<TEAM, NV, true, false><<<blocks, threads, 0, s>>>(x, rows, width, codes, scales);
    else if (f16)
      quantize_kernel<TEAM, NV, true, true><<<blocks, threads, 0, s>>>(x, rows, width, codes, scales);
    else if (plain)
      quantize_kernel<TEAM, NV, false, false><<<blocks, threads, 0, s>>>(x, rows, width, codes, scales);
    else
      quantize_kernel<TEAM, NV, false, true><<<blocks, threads, 0, s>>>(x, rows, width, codes, scales);
  });
  check_hip(hipGetLastError(), "quantize_rows launch");
}

}  // namespace tfm
