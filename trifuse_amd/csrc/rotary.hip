// Rotary positions: pairs of a head's channels turned by position * frequency.
//   (x1, x2) -> (x1 c - x2 s, x2 c + x1 s)
// An angle serves every head of its token, so a workgroup makes the cosines and sines of a
// few tokens once, in LDS, while its first elements are on their way, and then passes over
// up to kHeadBlock heads of them, eight pairs or eight copied channels an item. A pair is one
// thread's, which has read it before it writes: out may be x.
//
// Bound: memory (4 bytes an element), and at few tokens the launch: 16384 tokens of 16 heads of
// 128 take 25 us (5.4 TB/s), one token 4.5 on the host.
#include "rotary.h"
#include "rows.h"
#include "tfm_internal.h"

namespace tfm {

namespace {

constexpr int kThreads = 256;
constexpr int kAngles = kRotaryMaxDim / 2;  // of one workgroup: at least one token's
constexpr int kHeadBlock = 16;

template <bool F16>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a, int tokens) {
  __shared__ float2 turn[kAngles + 8];  // an item with fewer than eight pairs reads on
  const int t0 = blockIdx.x * tokens, nt = min(tokens, a.rows - t0);
  const int h0 = blockIdx.y * kHeadBlock, nh = min(kHeadBlock, a.heads - h0);
  const uint32_t turned = (a.pairs + 7) / 8, each = turned + (a.rest + 7) / 8;  // items of a head
  const uint32_t total = each * nh * nt;
  // An item's two vectors: halves (or neighbours) of eight pairs, or one of copied channels.
  struct Place {
    const uint16_t* x;
    uint16_t* out;
    const float2* cs;
    int d0, d1, n0, n1;  // channels, and how many there are
    bool pairs;
  };
  auto place = [&](uint32_t i) {
    const int c = i % each, h = h0 + i / each % nh, t = i / each / nh;
    Place p;
    p.x = a.x + (t0 + t) * a.x_row + h * a.x_head;
    p.out = a.out + (t0 + t) * a.out_row + h * a.out_head;
    p.cs = turn + t * a.pairs + 8 * c;
    p.pairs = c < (int)turned;
    const int left = a.pairs - 8 * c;
    if (!p.pairs) {
      p.d0 = 2 * a.pairs + 8 * (c - turned);
      p.d1 = p.d0;
      p.n0 = 2 * a.pairs + a.rest - p.d0;
      p.n1 = 0;
    } else if (a.interleaved) {
      p.d0 = 16 * c;
      p.d1 = p.d0 + 8;
      p.n0 = 2 * left;
      p.n1 = 2 * left - 8;
    } else {
      p.d0 = 8 * c;
      p.d1 = p.d0 + a.pairs;
      p.n0 = p.n1 = left;
    }
    return p;
  };
  Vec8 u{}, v{};
  auto fetch = [&](const Place& p) {
    u = load8<true>(p.x + p.d0, p.n0);
    v = load8<true>(p.x + p.d1, p.n1);
  };
  uint32_t i = threadIdx.x;
  Place p{};
  if (i < total) {
    p = place(i);
    fetch(p);
  }
  for (int k = threadIdx.x; k < nt * a.pairs; k += kThreads) {
    const int t = t0 + k / a.pairs;
    const double at = a.positions64 ? (double)static_cast<const int64_t*>(a.positions)[t]
                                    : (double)static_cast<const int32_t*>(a.positions)[t];
    turn[k] = turn_cos_sin(at * (a.frequencies[k % a.pairs] * kTurnsPerRadian), a.scale);
  }
  __syncthreads();
  while (i < total) {
    if (p.pairs) {
      Vec8 x, y;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float u1 = lo_st<F16>(u.w[j]), u2 = hi_st<F16>(u.w[j]), v1 = lo_st<F16>(v.w[j]), v2 = hi_st<F16>(v.w[j]);
        if (a.interleaved) {  // words hold a pair each
          const float2 m = p.cs[j], n = p.cs[4 + j];
          x.w[j] = pack_st2<F16>(__builtin_fmaf(u1, m.x, -(u2 * m.y)), __builtin_fmaf(u2, m.x, u1 * m.y));
          y.w[j] = pack_st2<F16>(__builtin_fmaf(v1, n.x, -(v2 * n.y)), __builtin_fmaf(v2, n.x, v1 * n.y));
        } else {
          const float2 m = p.cs[2 * j], n = p.cs[2 * j + 1];
          x.w[j] = pack_st2<F16>(__builtin_fmaf(u1, m.x, -(v1 * m.y)), __builtin_fmaf(u2, n.x, -(v2 * n.y)));
          y.w[j] = pack_st2<F16>(__builtin_fmaf(v1, m.x, u1 * m.y), __builtin_fmaf(v2, n.x, u2 * n.y));
        }
      }
      u = x;
      v = y;
    }
    store8<true>(p.out + p.d0, u, p.n0);
    store8<true>(p.out + p.d1, v, p.n1);
    i += kThreads;
    if (i < total) {
      p = place(i);
      fetch(p);
    }
  }
}

}  // namespace

void launch_rotary(bool f16, const RotaryArgs& a, hipStream_t s) {
  // Tokens of a workgroup: enough for an item a thread, no more than about 1000 workgroups need, and
  // an angle a thread (901 tokens of 24 heads of 64, 32 channels turned: 4.9 us, one token a workgroup 6.9).
  const int blocks = (a.heads + kHeadBlock - 1) / kHeadBlock;
  const int items = std::min(a.heads, kHeadBlock) * ((a.pairs + 7) / 8 + (a.rest + 7) / 8);
  const int least = (kThreads + items - 1) / items, most = std::max(1, kThreads / a.pairs);
  const int tokens = std::max(1, std::min(std::max(least, (int)((int64_t)a.rows * blocks / 1024)), most));
  const dim3 grid((a.rows + tokens - 1) / tokens, blocks);
  tfm_launch(f16 ? rotary_kernel<true> : rotary_kernel<false>, grid, dim3(kThreads), 0, s, a, tokens);
  check_hip(hipGetLastError(), "rotary launch");
}

}  // namespace tfm
