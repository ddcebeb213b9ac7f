// Rotary positions: pairs of a head's channels turned by position * frequency.
//   (x1, x2) -> (x1 c - x2 s, x2 c + x1 s)
// An angle serves every head of its token, so a workgroup makes the cosines and
// sines of a few tokens once, in LDS, and then passes over up to kHeadBlock heads
// of them with 16-byte loads and stores.
//
// Bound: memory (4 bytes an element), and at few tokens the launch.
#include "rotary.h"
#include "rows.h"
#include "tfm_internal.h"

namespace tfm {

namespace {

constexpr int kThreads = 256;
constexpr int kAngles = kRotaryMaxDim / 2;  // of one workgroup: at least one token's
constexpr int kHeadBlock = 16;

// VEC pairs an item: 8, or 1 where the pairs or the rest are no multiple of 8.
template <bool F16, int VEC>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a, int tokens) {
  __shared__ float2 turn[kAngles];
  const int t0 = blockIdx.x * tokens, nt = min(tokens, a.rows - t0);
  const int h0 = blockIdx.y * kHeadBlock, nh = min(kHeadBlock, a.heads - h0);
  for (int i = threadIdx.x; i < nt * a.pairs; i += kThreads) {
    const int t = t0 + i / a.pairs;
    const double at = a.positions64 ? (double)static_cast<const int64_t*>(a.positions)[t]
                                    : (double)static_cast<const int32_t*>(a.positions)[t];
    turn[i] = turn_cos_sin(at * (a.frequencies[i % a.pairs] * kTurnsPerRadian), a.scale);
  }
  __syncthreads();
  const uint32_t turned = a.pairs / VEC, each = turned + a.rest / VEC;  // items of a head
  for (uint32_t i = threadIdx.x; i < each * nh * nt; i += kThreads) {
    const int c = i % each, h = h0 + i / each % nh, t = i / each / nh;
    const uint16_t* x = a.x + (t0 + t) * a.x_row + h * a.x_head;
    uint16_t* out = a.out + (t0 + t) * a.out_row + h * a.out_head;
    const float2* cs = turn + t * a.pairs + c * VEC;
    if (c >= (int)turned) {  // behind the pairs
      const int d = 2 * a.pairs + (c - turned) * VEC;
      if constexpr (VEC == 8)
        store8<true>(out + d, load8<true>(x + d, 8), 8);
      else
        out[d] = x[d];
    } else if constexpr (VEC == 1) {
      const int d0 = a.interleaved ? 2 * c : c, d1 = a.interleaved ? d0 + 1 : c + a.pairs;
      const float x1 = st2f<F16>(x[d0]), x2 = st2f<F16>(x[d1]);
      out[d0] = f2st<F16>(__builtin_fmaf(x1, cs->x, -(x2 * cs->y)));
      out[d1] = f2st<F16>(__builtin_fmaf(x2, cs->x, x1 * cs->y));
    } else {
      const int d0 = a.interleaved ? 16 * c : 8 * c, d1 = a.interleaved ? d0 + 8 : d0 + a.pairs;
      const Vec8 u = load8<true>(x + d0, 8), v = load8<true>(x + d1, 8);
      Vec8 p, q;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (a.interleaved) {  // words hold a pair each
          const float2 m = cs[j], n = cs[4 + j];
          const float u1 = lo_st<F16>(u.w[j]), u2 = hi_st<F16>(u.w[j]), v1 = lo_st<F16>(v.w[j]), v2 = hi_st<F16>(v.w[j]);
          p.w[j] = pack_st2<F16>(__builtin_fmaf(u1, m.x, -(u2 * m.y)), __builtin_fmaf(u2, m.x, u1 * m.y));
          q.w[j] = pack_st2<F16>(__builtin_fmaf(v1, n.x, -(v2 * n.y)), __builtin_fmaf(v2, n.x, v1 * n.y));
        } else {
          const float2 m = cs[2 * j], n = cs[2 * j + 1];
          const float u1 = lo_st<F16>(u.w[j]), u2 = hi_st<F16>(u.w[j]), v1 = lo_st<F16>(v.w[j]), v2 = hi_st<F16>(v.w[j]);
          p.w[j] = pack_st2<F16>(__builtin_fmaf(u1, m.x, -(v1 * m.y)), __builtin_fmaf(u2, n.x, -(v2 * n.y)));
          q.w[j] = pack_st2<F16>(__builtin_fmaf(v1, m.x, u1 * m.y), __builtin_fmaf(v2, n.x, u2 * n.y));
        }
      }
      store8<true>(out + d0, p, 8);
      store8<true>(out + d1, q, 8);
    }
  }
}

}  // namespace

void launch_rotary(bool f16, const RotaryArgs& a, hipStream_t s) {
  const int tokens = std::max(1, std::min(kThreads, kAngles) / std::max(a.pairs, 1));
  const dim3 grid((a.rows + tokens - 1) / tokens, (a.heads + kHeadBlock - 1) / kHeadBlock);
  const bool vec = a.pairs % 8 == 0 && a.rest % 8 == 0;
  auto* kernel = f16 ? (vec ? rotary_kernel<true, 8> : rotary_kernel<true, 1>)
                     : (vec ? rotary_kernel<false, 8> : rotary_kernel<false, 1>);
  tfm_launch(kernel, grid, dim3(kThreads), 0, s, a, tokens);
  check_hip(hipGetLastError(), "rotary launch");
}

}  // namespace tfm
