// Log probabilities of given tokens, entropy and the most likely alternatives
// of softmax(scale * logits), one workgroup a row, one pass over the logits.
//
// With M the row's largest logit, y = scale (l - M) / ln 2, S = sum 2^y and D = sum y 2^y:
//   log p(l) = scale (l - M) - ln S,   entropy = ln S - ln 2 D / S.
// Both terms of the entropy are non-negative: nothing cancels. Each thread keeps
// M, S and D of what it has read and rescales S and D when M grows; differences
// of logits are taken before the scale, so they are exact for 16-bit logits
// near the maximum, the ones that count. A term of D counts while 2^y does not
// vanish, so D stays as small as S whatever the scale. Where one token is nearly sure, S is
// 1 + R with R far below 1: one thread alone adds the 1, its other terms are
// summed again without it, and ln S = log1p(R) keeps its precision.
//
// Alternatives: logits order by a key, their value's bits made monotonic
// (NaN below -inf) and below it the complement of their place, so that ties go
// to the lower place and no two keys are equal. A row's items are its whole
// vectors and then the logits left over, one by one; each thread knows the
// largest key among the items it has read (their maxima, the item's place).
// 64 buckets, lane l of every wave, give 64 maxima; the top-th largest of them
// is a threshold that at least `top` logits reach. Only threads whose own
// maximum reaches it can hold such logits. They read the item of their maximum
// again; those whose second largest item may reach it too go over all of theirs
// (no line of theirs is in the cache any more, and 25 threads' items are half the
// row's lines: 4096 x 50304 97 us with that for every such thread). The logits that
// reach the threshold go to a list in LDS, and each one's rank in the list is its
// place among the alternatives.
// A row made so that the list overflows takes one scan per alternative.
//
// Bound: arithmetic beside the stream, 13 vector instructions a logit, the
// exponential among them. 4096 x 50304 bf16: 80 us without alternatives (5.2 TB/s),
// 86 to 88 with 20; one row 8.5 us, one workgroup's arithmetic.
#include "tfm_device.h"
#include "tfm_internal.h"

namespace tfm {

namespace {

constexpr int kAhead = 4;        // items a thread has in flight
constexpr int kCap = 1024;       // keys the candidate list holds
constexpr float kLow = -3.402823466e38f;
constexpr float kSure = 1.0f;  // R below which the roundings of 1 + R (a few 2^-24) count beside ln S

// Logits of one 16-byte vector.
template <int DT>
struct Logits {
  static constexpr int N = DT == TFM_DTYPE_F32 ? 4 : 8;
  static constexpr int SIZE = DT == TFM_DTYPE_F32 ? 4 : 2;
  __device__ static __forceinline__ float one(const char* row, int64_t i) {
    if constexpr (DT == TFM_DTYPE_F32) return *reinterpret_cast<const float*>(row + 4 * i);
    return st2f<DT == TFM_DTYPE_F16>(*reinterpret_cast<const uint16_t*>(row + 2 * i));
  }
  // Rows start at any element: the vector may straddle 16-byte lines.
  __device__ static __forceinline__ uint4 load(const char* row, int64_t v) {
    uint4 u;
    __builtin_memcpy(&u, row + 16 * v, 16);
    return u;
  }
  __device__ static __forceinline__ float get(const uint4& u, int j) {
    if constexpr (DT == TFM_DTYPE_F32) return __uint_as_float(word_of(u, j));
    const uint32_t w = word_of(u, j / 2);
    return j & 1 ? hi_st<DT == TFM_DTYPE_F16>(w) : lo_st<DT == TFM_DTYPE_F16>(w);
  }
};

// Monotonic in the value: NaN 1, then -inf .. +inf, the two zeros equal. 0 is
// left for "nothing".
__device__ __forceinline__ uint32_t order_of(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);  // -0 + 0 = +0
  if ((u & 0x7fffffffu) > 0x7f800000u) return 1u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  if (o == 1u) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t key_of(uint32_t order, uint32_t place) { return (uint64_t)order << 32 | ~place; }

// Sums of the logits read so far at their maximum m (kLow before any).
struct Stats {
  float m, s, d;
};

// The same sums at a maximum m' >= m. The exponent is kept finite, far below where
// 2^y vanishes, so that nothing becomes 0 * inf.
__device__ __forceinline__ Stats rescaled(const Stats& a, float m, float c) {
  const float y = fmaxf((a.m - m) * c, -1e30f);
  const float e = __builtin_amdgcn_exp2f(y);
  return Stats{m, a.s * e, e * __builtin_fmaf(y, a.s, a.d)};
}

template <int CTRL, int ROW_MASK>
__device__ __forceinline__ float dpp_fmax(float v) {
  const int b = __float_as_int(v);
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(b, b, CTRL, ROW_MASK, 0xf, false)));
}
__device__ __forceinline__ float wave_fmax(float v) {
  v = dpp_fmax<0xb1, 0xf>(v);
  v = dpp_fmax<0x4e, 0xf>(v);
  v = dpp_fmax<0x141, 0xf>(v);
  v = dpp_fmax<0x140, 0xf>(v);
  v = dpp_fmax<0x142, 0xa>(v);
  v = dpp_fmax<0x143, 0xc>(v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

template <int DT, int THREADS>
__global__ __launch_bounds__(THREADS) void token_logprobs_kernel(LogprobsArgs a) {
  using L = Logits<DT>;
  constexpr int N = L::N, WAVES = THREADS / 64;
  __shared__ float sm[WAVES], ss[WAVES], sh[WAVES], sd[WAVES];
  __shared__ int sn[WAVES];
  __shared__ uint64_t keys[THREADS];
  __shared__ uint64_t cand[kCap];
  __shared__ uint8_t rank[WAVES][64];
  __shared__ int chosen[THREADS];
  __shared__ int n_chosen, n_cand, holder;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int t = blockIdx.x;
  const int V = a.vocab;
  const char* row = static_cast<const char*>(a.logits) + (int64_t)t * a.row_stride * L::SIZE;
  // Thread i reads items i, i + THREADS, ...
  const int full = V / N, items = full + V % N;
  const float c = a.scale * 1.44269504f;

  // The given token's logit, read early.
  int64_t token = -1;
  float tl = 0.0f;
  if (tid == 0) {
    n_chosen = n_cand = 0;
    if (a.logprobs) {
      token = a.tokens64 ? static_cast<const int64_t*>(a.tokens)[t] : static_cast<const int32_t*>(a.tokens)[t];
      if (token >= 0 && token < V) tl = L::one(row, token);
    }
  }

  auto term = [&](float f, float m, float& s, float& d) {
    const float y = (f - m) * c;
    const float e = __builtin_amdgcn_exp2f(y);
    s += e;
    d = __builtin_fmaf(fmaxf(y, kLow), e, d);  // a masked logit: e = 0, not -inf * 0
  };
  auto max_of = [&](const float* f) {
    float m = f[0];
#pragma unroll
    for (int j = 1; j < N; ++j) m = fmaxf(m, f[j]);
    return m;
  };
  Stats st{kLow, 0.0f, 0.0f};
  int best_item = -1;  // the first item that holds st.m
  float second = -__builtin_inff();  // no other item's maximum is larger
  // kAhead vectors a thread are on their way at a time; past the last one a
  // thread reads that one again and leaves it out.
  for (int v = tid; v < (full + THREADS - 1) / THREADS * THREADS; v += kAhead * THREADS) {
    uint4 u[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = v + i * THREADS;
      u[i] = L::load(row, at < full ? at : full - 1);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (v + i * THREADS >= full) break;
      float f[N];
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = L::get(u[i], j);
      const float m = max_of(f);
      second = __builtin_amdgcn_fmed3f(second, st.m, m);
      if (m > st.m) {
        st = rescaled(st, m, c);
        best_item = v + i * THREADS;
      }
#pragma unroll
      for (int j = 0; j < N; ++j) term(f[j], st.m, st.s, st.d);
    }
  }
  // The logits left over: item full + j to the thread whose turn it is.
  const int turn = (tid - full % THREADS + THREADS) % THREADS;
  if (turn < items - full) {
    const float f = L::one(row, (int64_t)full * N + turn);
    second = __builtin_amdgcn_fmed3f(second, st.m, f);
    if (f > st.m) {
      st = rescaled(st, f, c);
      best_item = full + turn;
    }
    term(f, st.m, st.s, st.d);
  }

  // An item again: its logits and how many they are.
  auto fetch = [&](int v, float* f) {
    if (v < full) {
      const uint4 u = L::load(row, v);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = L::get(u, j);
      return N;
    }
    f[0] = L::one(row, (int64_t)full * N + (v - full));
#pragma unroll
    for (int j = 1; j < N; ++j) f[j] = 0.0f;
    return 1;
  };
  uint64_t best = 0;
  if (a.top > 0) {
    if (best_item >= 0) {
      best = key_of(order_of(st.m), (uint32_t)best_item);
    } else {  // nothing above the lowest number: masked logits, or none
      for (int v = tid; v < items; v += THREADS) {
        float f[N];
        const int n = fetch(v, f);
        const uint64_t k = key_of(order_of(n == N ? max_of(f) : f[0]), (uint32_t)v);
        best = k > best ? k : best;
      }
    }
    keys[tid] = best;
  }

  // The row's maximum, then its sums at that maximum; a thread that holds it
  // adds the maximum's own 1 apart (one of them: the row's holder).
  const float wm = wave_fmax(st.m);
  if (lane == 0) sm[wave] = wm;
  __syncthreads();
  float m = sm[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) m = fmaxf(m, sm[w]);
  const bool holds = best_item >= 0 && st.m == m;
  if (holds) holder = tid;
  st = rescaled(st, m, c);
  const float ws = wave_tree_sum64(holds ? 0.0f : st.s), wh = wave_tree_sum64(holds ? st.s - 1.0f : 0.0f);
  const float wd = wave_tree_sum64(st.d);
  const int wn = __popcll(__ballot(holds));
  if (lane == 63) {
    ss[wave] = ws;
    sh[wave] = wh;
    sd[wave] = wd;
    sn[wave] = wn;
  }
  // Bucket `lane`'s largest key (an empty one has a key of its own below all
  // others); wave w counts how many of its share of the buckets exceed it.
  uint64_t bucket = 63 - lane;
  if (a.top > 0) {
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const uint64_t o = keys[64 * w + lane];
      bucket = o > bucket ? o : bucket;
    }
    constexpr int SHARE = 64 / WAVES;
    int above = 0;
#pragma unroll
    for (int i = 0; i < SHARE; ++i) {
      const int l = wave * SHARE + i;
      const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(bucket >> 32), l) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)bucket, l);
      above += o > bucket;
    }
    rank[wave][lane] = (uint8_t)above;
  }
  __syncthreads();
  float r = ss[0], rh = sh[0], d = sd[0];
  int ones = sn[0];  // threads that hold the maximum
#pragma unroll
  for (int w = 1; w < WAVES; ++w) {
    r += ss[w];
    rh += sh[w];
    d += sd[w];
    ones += sn[w];
  }
  if (ones == 1 && r + rh < kSure) {
    // The holder's other terms, 64 of its items at a time (every wave the same sum).
    const int h = holder;
    float part = 0.0f;
    int before = 0;  // maxima in items ahead of this lane's
    for (int v0 = h; v0 < items; v0 += 64 * THREADS) {
      const int v = v0 + lane * THREADS;
      float f[N], unused = 0.0f;
      const int n = v < items ? fetch(v, f) : 0;
      bool first = false;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (j >= n) continue;
        if (f[j] == m && !first) {
          first = true;  // the item's first maximum: one of the row's stays out
          continue;
        }
        term(f[j], m, part, unused);
      }
      before += __popcll(__ballot(first));
    }
    part = wave_tree_sum64(part);
    rh = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(part), 63)) + (float)(before - 1);
  }
  r += rh;
  // +inf among the logits: NaN, as inf - inf makes their terms.
  const float s = m == __builtin_inff() ? __uint_as_float(0x7fc00000u) : r + (float)ones;
  const float ln_s = ones > 0 ? log1pf(s - 1.0f < 1.0f ? r + (float)(ones - 1) : s - 1.0f) : logf(s);
  const bool empty = s == 0.0f;  // every logit is -inf
  // Halves: l - m may pass the largest number where scale * (l - m) does not.
  auto logp = [&](float l) {
    return empty ? -__builtin_inff() : __builtin_fmaf(2.0f * a.scale, 0.5f * l - 0.5f * m, -ln_s);
  };
  if (tid == 0) {
    if (a.logprobs) a.logprobs[t] = token >= 0 && token < V ? logp(tl) : __uint_as_float(0x7fc00000u);
    if (a.entropy) a.entropy[t] = empty ? 0.0f : ln_s - 0.693147181f * d / s;
  }
  if (a.top <= 0) return;

  // The bucket that top - 1 others exceed is the threshold: each wave finds it.
  int above = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) above += rank[w][lane];
  const int at = __builtin_ctzll(__ballot(above == a.top - 1));
  const uint64_t thr = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(bucket >> 32), at) << 32 |
                       (uint32_t)__builtin_amdgcn_readlane((int)bucket, at);
  const float low = value_of((uint32_t)(thr >> 32));  // NaN: no logit is below
  auto scan = [&](int v) {
    float f[N];
    const int n = fetch(v, f);
    const uint32_t first = v < full ? (uint32_t)v * N : (uint32_t)(full * N + (v - full));
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j >= n || f[j] < low) continue;
      const uint32_t o = order_of(f[j]);
      if (key_of(o, (uint32_t)v) < thr) continue;
      const int p = atomicAdd(&n_cand, 1);
      if (p < kCap) cand[p] = key_of(o, first + j);
    }
  };
  if (best != 0 && best >= thr) {
    if (best_item >= 0 && second < low)
      scan(best_item);
    else
      chosen[atomicAdd(&n_chosen, 1)] = tid;
  }
  __syncthreads();
  const int nc = n_chosen, per = (items + THREADS - 1) / THREADS;
  const int bits = per > 1 ? 32 - __builtin_clz(per - 1) : 0;  // items of a thread, to a power of two
  for (int i = tid; i < nc << bits; i += THREADS) {
    const int v = chosen[i >> bits] + (i & ((1 << bits) - 1)) * THREADS;
    if (v < items) scan(v);
  }
  __syncthreads();
  int32_t* ids = a.top_ids + (int64_t)t * a.top;
  float* lps = a.top_logprobs + (int64_t)t * a.top;
  const int n = n_cand;
  if (n <= kCap) {
    for (int i = tid; i < n; i += THREADS) {
      const uint64_t k = cand[i];
      int place = 0;
      for (int j = 0; j < n; ++j) place += cand[j] > k;
      if (place < a.top) {
        ids[place] = (int32_t)~(uint32_t)k;
        lps[place] = logp(value_of((uint32_t)(k >> 32)));
      }
    }
    return;
  }
  // The list overflowed: the largest key below the last one, `top` times.
  uint64_t last = ~0ull;
  for (int r = 0; r < a.top; ++r) {
    uint64_t k = 0;
    for (int i = tid; i < V; i += THREADS) {
      const uint64_t o = key_of(order_of(L::one(row, i)), (uint32_t)i);
      if (o < last && o > k) k = o;
    }
    keys[tid] = k;
    __syncthreads();
    for (int w = THREADS / 2; w > 0; w >>= 1) {
      if (tid < w && keys[tid + w] > keys[tid]) keys[tid] = keys[tid + w];
      __syncthreads();
    }
    last = keys[0];
    __syncthreads();
    if (tid == 0) {
      ids[r] = (int32_t)~(uint32_t)last;
      lps[r] = logp(value_of((uint32_t)(last >> 32)));
    }
  }
}

template <int DT>
void launch_dt(const LogprobsArgs& a, hipStream_t s) {
  // Few rows leave CUs to spare: wider workgroups read a long row faster, narrower
  // ones have less to join. us of 256 / 512 threads, rows x vocabulary:
  //   1 x 4000 5.2 / 5.2     1 x 10007 5.7 / 5.4     1 x 50304 10.0 / 8.5
  //   256 x 10007 7.0 / 6.9  333 x 10007 8.0 / 8.3   256 x 50304 13.0 / 10.8
  //   333 x 50304 15.6 / 14.6   768 x 50304 19.8 / 20.3   1024 x 50304 25.0 / 25.3
  // (1024 threads: 9.0, 16.3 and 29.6 at 1, 333 and 1024 x 50304).
  if ((a.rows <= 256 && a.vocab >= 8192) || (a.rows <= 768 && a.vocab >= 32768))
    token_logprobs_kernel<DT, 512><<<a.rows, 512, 0, s>>>(a);
  else
    token_logprobs_kernel<DT, 256><<<a.rows, 256, 0, s>>>(a);
}

}  // namespace

void launch_token_logprobs(int dtype, const LogprobsArgs& a, hipStream_t s) {
  if (a.rows <= 0) return;
  if (dtype == TFM_DTYPE_F32)
    launch_dt<TFM_DTYPE_F32>(a, s);
  else if (dtype == TFM_DTYPE_F16)
    launch_dt<TFM_DTYPE_F16>(a, s);
  else
    launch_dt<TFM_DTYPE_BF16>(a, s);
  check_hip(hipGetLastError(), "token_logprobs launch");
}

}  // namespace tfm
