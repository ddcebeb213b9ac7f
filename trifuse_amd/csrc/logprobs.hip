// Log probabilities of given tokens, entropy and the most likely alternatives
// of softmax(scale * logits), one workgroup a row, one pass over the logits.
//
// With M the row's largest logit, S = sum e^(scale (l - M)) and
// D = sum (l - M) e^(scale (l - M)):
//   log p(l) = scale (l - M) - ln S,   entropy = ln S - scale D / S.
// Both terms of the entropy are non-negative: nothing cancels. Each thread keeps
// M, S and D of what it has read and rescales S and D when M grows; differences
// of logits are taken before the scale, so they are exact for 16-bit logits
// near the maximum, the ones that count. The maximum's own term, 1, is kept out
// of the running sum: ln S = log1p(R) holds its precision where one token is
// nearly sure and R, the others' sum, is far below 1.
//
// Alternatives: logits order by a key, their value's bits made monotonic
// (NaN below -inf) and below it the complement of their place, so that ties go
// to the lower place and no two keys are equal. Each thread also keeps the
// largest key among the vectors it has read (their maxima, the vector's place).
// 64 buckets, lane l of every wave, give 64 maxima; the top-th largest of them
// is a threshold that at least `top` logits reach. Only threads whose own
// maximum reaches it can hold such logits: their vectors are read again
// (a few in a thousand), the logits that reach the threshold go to a list in
// LDS, and each one's rank in the list is its place among the alternatives.
// A row made so that the list overflows takes one scan per alternative.
#include "tfm_device.h"
#include "tfm_internal.h"

namespace tfm {

namespace {

constexpr int kCap = 1024;       // keys the candidate list holds
constexpr float kLow = -3.402823466e38f;

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

// Sums of the logits read so far at their maximum m: s without the maximum's own
// term (one: 1 once there is a maximum), d the weighted differences.
struct Stats {
  float m, s, d, one;
};

// The same sums at a maximum m' >= m, the old maximum's term among them. The
// difference of maxima is kept finite: an empty part (s = d = one = 0) stays empty.
__device__ __forceinline__ Stats rescaled(Stats a, float m, float c) {
  const float dm = fmaxf(a.m - m, -1e30f);
  const float e = __builtin_amdgcn_exp2f(dm * c);
  const float all = a.s + a.one;
  return Stats{m, all * e, e * __builtin_fmaf(dm, all, a.d), 0.0f};
}

template <int DT, int THREADS>
__global__ __launch_bounds__(THREADS) void token_logprobs_kernel(LogprobsArgs a) {
  using L = Logits<DT>;
  constexpr int N = L::N, WAVES = THREADS / 64;
  __shared__ float sm[WAVES], ss[WAVES], sd[WAVES];
  __shared__ int sn[WAVES];
  __shared__ uint64_t keys[THREADS];
  __shared__ uint64_t cand[kCap];
  __shared__ uint64_t threshold;
  __shared__ int chosen[THREADS];
  __shared__ int n_chosen, n_cand;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int t = blockIdx.x;
  const int V = a.vocab;
  const char* row = static_cast<const char*>(a.logits) + (int64_t)t * a.row_stride * L::SIZE;
  const int nvec = (V + N - 1) / N;  // the last one may be partial
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

  Stats st{kLow, 0.0f, 0.0f, 0.0f};
  uint64_t best = 0;
  auto add = [&](float* f, int n, int v) {
    float m = f[0];
#pragma unroll
    for (int j = 1; j < N; ++j)
      if (j < n) m = fmaxf(m, f[j]);
    const uint64_t k = key_of(order_of(m), (uint32_t)v);
    if (k > best) best = k;
    if (m > st.m) {
      st = rescaled(st, m, c);
      st.one = 1.0f;
      bool found = false;  // the first of the vector's maxima leaves the sum
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const bool it = !found && j < n && f[j] == m;
        f[j] = it ? -__builtin_inff() : f[j];
        found = found || it;
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) {
        const float x = f[j] - st.m;
        const float e = __builtin_amdgcn_exp2f(x * c);
        st.s += e;
        st.d = __builtin_fmaf(fmaxf(x, kLow), e, st.d);  // a masked logit: e = 0, not -inf * 0
      }
  };
  const int full = V / N;
  for (int v = tid; v < full; v += THREADS) {
    const uint4 u = L::load(row, v);
    float f[N];
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = L::get(u, j);
    add(f, N, v);
  }
  if (nvec > full && tid == full % THREADS) {
    float f[N];
    const int n = V - full * N;
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = j < n ? L::one(row, (int64_t)full * N + j) : 0.0f;
    add(f, n, full);
  }

  // The row's maximum, then its sums at that maximum.
  float m = st.m;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, shfl_xor_f(m, x));
  if (lane == 0) sm[wave] = m;
  keys[tid] = best;
  __syncthreads();
  m = sm[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) m = fmaxf(m, sm[w]);
  const float one = st.m == m ? st.one : 0.0f;
  if (st.m != m) st = rescaled(st, m, c);
  const float ws = wave_tree_sum64(st.s), wd = wave_tree_sum64(st.d);
  const int wn = __popcll(__ballot(one != 0.0f));
  if (lane == 63) {
    ss[wave] = ws;
    sd[wave] = wd;
    sn[wave] = wn;
  }
  // Bucket `lane`'s largest key; the one that top - 1 others exceed.
  if (a.top > 0 && wave == 0) {
    uint64_t k = best;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      const uint64_t o = keys[64 * w + lane];
      k = o > k ? o : k;
    }
    int above = 0, equal_before = 0;  // empty buckets are equal
#pragma unroll 8
    for (int l = 0; l < 64; ++l) {
      const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), l) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)k, l);
      above += o > k;
      equal_before += o == k && l < lane;
    }
    if (above + equal_before == a.top - 1) threshold = k;
  }
  __syncthreads();
  float r = ss[0], d = sd[0];
  int ones = sn[0];  // threads that hold the maximum
#pragma unroll
  for (int w = 1; w < WAVES; ++w) {
    r += ss[w];
    d += sd[w];
    ones += sn[w];
  }
  // +inf among the logits: NaN, as inf - inf makes the other maxima.
  if (m == __builtin_inff()) r = __uint_as_float(0x7fc00000u);
  const float s = r + (float)ones;
  const float ln_s = ones > 0 ? log1pf(r + (float)(ones - 1)) : logf(s);
  const bool empty = s == 0.0f;  // every logit is -inf
  auto logp = [&](float l) { return empty ? -__builtin_inff() : __builtin_fmaf(a.scale, l - m, -ln_s); };
  if (tid == 0) {
    if (a.logprobs) a.logprobs[t] = token >= 0 && token < V ? logp(tl) : __uint_as_float(0x7fc00000u);
    if (a.entropy) a.entropy[t] = empty ? 0.0f : ln_s - a.scale * d / s;
  }
  if (a.top <= 0) return;

  const uint64_t thr = threshold;
  if (best != 0 && best >= thr) chosen[atomicAdd(&n_chosen, 1)] = tid;
  __syncthreads();
  const int nc = n_chosen, per = (nvec + THREADS - 1) / THREADS;
  for (int i = tid; i < nc * per; i += THREADS) {
    const int v = chosen[i % nc] + i / nc * THREADS;
    if (v >= nvec) continue;
    const int n = V - v * N < N ? V - v * N : N;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j >= n) break;
      const int64_t at = (int64_t)v * N + j;
      const uint32_t o = order_of(L::one(row, at));
      if (key_of(o, (uint32_t)v) < thr) continue;
      const int p = atomicAdd(&n_cand, 1);
      if (p < kCap) cand[p] = key_of(o, (uint32_t)at);
    }
  }
  __syncthreads();
  int32_t* ids = a.top_ids + (int64_t)t * a.top;
  float* lps = a.top_logprobs + (int64_t)t * a.top;
  const int n = n_cand;
  if (n <= kCap) {
    for (int i = tid; i < n; i += THREADS) {
      const uint64_t k = cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += cand[j] > k;
      if (rank < a.top) {
        ids[rank] = (int32_t)~(uint32_t)k;
        lps[rank] = logp(value_of((uint32_t)(k >> 32)));
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
  if (a.rows < 1024 && a.vocab >= 8192)
    token_logprobs_kernel<DT, 1024><<<a.rows, 1024, 0, s>>>(a);
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
