// Attention over the paged cache of 8-bit codes.
//
// For a row's query q in a head, over the tokens j that it sees, with codes c and the
// scales a (keys) and b (values) of token j's page:
//   s_j = scale * a_j * (q . ck_j),   out = sum_j e^(s_j) b_j cv_j / sum_j e^(s_j)
// One pass with a running maximum, over t_j = s_j log2(e) + log2(b_j):
//   w_j = 2^(t_j - m),   out = (sum_j w_j cv_j) / (sum_j w_j / b_j)
// so the page's value scale costs nothing an element (its logarithm rides in the
// exponent's fused multiply-add, its inverse on the sum of 8 or 16 weights). Codes enter the
// products as they are, as halves that hold them exactly (keys plus 128, which the sum of q
// takes out of a score again), q of bf16 exactly after a power of two for its row (28
// binades; what is smaller loses bits below 2^-25 of the largest), and w to 2^-11 of itself,
// the same in both sums, so that a row that looks at few tokens loses less. m is eight below a maximum
// that is taken again only when a weight has grown past a half's range (its relative precision is the
// same from 2^-14 to there), so most tiles look for none and rescale nothing: what is left a score is a
// multiply-add, an exponential, and half a conversion and half a sum of two. A weight below 2^-22 of
// the row's largest, 15 below its score, loses a bit a binade, and below 2^-33 it is nothing.
//
// "Columns" are the (row, head) pairs of one key head: they share its codes. Scores are
// taken transposed, keys along the rows of a product and columns along its lanes: a lane
// then owns one column's statistics, and the weights it computes are, without leaving
// their registers, the operand of the second product, since the order of keys inside a
// product is free as long as both operands keep it. A lane's keys of 32 are 16 (tile
// kernel) or 8 (few kernel) consecutive ones, which lie in one page.
//
// Kernels. Few columns (decoding, drafts; up to 32): memory decides. Each wave takes
// 32 tokens at a time straight from memory into registers: key codes as 16-byte pieces of
// a row, value codes as D/16 bytes a lane of eight rows, transposed by byte permutes into
// the product's operand. So it is for more columns while all their workgroups are there at
// once. Many: 256 a workgroup of eight waves, whose tiles of 128
// tokens are converted to halves once on their way into LDS; 128 of four waves and tiles of
// 64; or 64, where two waves share their columns and take a half of each tile.
//
// Work items are (sequence, tile of columns, part of its tokens). How many parts follows
// on the device from the lengths, so that ragged batches spread evenly and a captured
// call follows its lengths; parts are joined by a second kernel.
#include "kv_cache.h"

namespace tfm {

namespace {

constexpr float kLow = -3.402823466e38f;  // below every score; finite, so that differences are
// Weights enter the products times 2^8, so that those down to 2^-22 of a row's largest are normal
// halves: many such tokens may be all that a row brings, behind one whose value is zero. Sums of
// weights take it out again. Higher costs time, as the maximum is then taken again more often: of
// chunks of 7 prompts, whose heads are sharp, 46.8 us with 0, 49.5 with 8, 50.8 with 10; of 8192
// rows 291, 296 and 300.
constexpr float kLift = 8.0f, kLiftUnit = 0x1p8f;
constexpr float kMost = 0x1p100f;  // a lane's sum past this is infinite: a weight is past a half's range, and the maximum is taken again
// Where a maximum is taken again, weights follow from the same rounded scores as it does, t - m and not
// fma(.., shift - m): past 2^24 a score's step is binades of a weight, and what shift - m loses could
// put one past a half once more. m is eight below in two steps of four, since one step of eight rounds
// to 16 where fp32's step is that.
__device__ __forceinline__ float below(float top) { return top - kLift / 2 - kLift / 2; }
// Weights below 2^-22 are subnormal halves, each off by up to 2^-33. In the sum of w / b that is
// 2^-33 / b: pages whose 1 / b is over so many times the sum so far have theirs summed in fp32.
constexpr float kLeast = 16.0f;
constexpr float kOutUnit = kValueUnit / kLiftUnit;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Sum over the wave, and sums up to each lane, without leaving the registers.
__device__ __forceinline__ float wave_sum(float v) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wave_tree_sum64(v)), 63));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_upto(int v) {
  v = dpp_add<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);  // row_bcast:15, 31
  return dpp_add<0x143, 0xc>(v);
}

// What one work item is.
struct Item {
  int b;      // sequence, -1: none
  KvSeq s;
  int tile;   // of the sequence's columns
  int part;   // of `parts`
  int parts;
  int entry;  // index of part 0 of this tile
  int index;  // of the tile in the batch
};

// The first token that a row at `position` sees. Rows stand before the first token too, and windows
// are as long as an int: of a negative position nothing is taken off.
__device__ __forceinline__ int lowest(const AttentionArgs& a, int position) {
  return a.window ? max(0, max(position, 0) - a.window + 1) : 0;
}

// A sequence's tiles of columns, and tokens that some of its rows see.
__device__ __forceinline__ int tiles_of(const AttentionArgs& a, const KvSeq& s, int columns) {
  return (s.n * a.group + columns - 1) / columns;
}
__device__ __forceinline__ int tokens_of(const AttentionArgs& a, const KvSeq& s) {
  return max(s.len - lowest(a, s.first), 0);
}

// Item `index` of a batch of many sequences, none of them cut, without a look at all of them.
// With the same number of rows each it is a division. Else a sequence has its places from
// place(b) on: its columns before it over a tile's, and one for each sequence before it, for the
// rounding up; or one a column where that is fewer. They are at least its tiles, grow with b, and are
// found in log2 steps. A look at all costs each workgroup as many steps as there are 64 sequences: one
// token each of 32 heads over 8 of 128, 1000 sequences 97 us with it, 64 by search and 51 by division,
// 16384 13100, 1060 and 800; 150 sequences of 5 rows of 24 heads over 8 of 64 9.5, 11.2 and 8.2, 300
// of them 19.2, 18.4 and 13.1.
__device__ Item find_whole(const AttentionArgs& a, int columns, int index) {
  const KvBatchArgs& g = a.b;
  Item it{};
  it.b = -1;
  it.parts = 1;
  int b, before;
  if (g.starts) {
    const int all = g.rows * a.group;
    const bool by_column = all < all / columns + g.sequences;
    auto place = [&](int b) {
      const int at = min(max(g.starts[b], 0), g.rows) * a.group;
      return by_column ? at : at / columns + b;
    };
    b = 0;
    for (int end = g.sequences; end - b > 1;) {
      const int middle = b + (end - b) / 2;
      if (place(middle) <= index)
        b = middle;
      else
        end = middle;
    }
    before = place(b);
  } else {
    const int each = (g.max_rows * a.group + columns - 1) / columns;
    b = index / each;
    before = b * each;
    if (b >= g.sequences) return it;
  }
  const KvSeq s = kv_seq(g, b);
  if (index < before || index - before >= tiles_of(a, s, columns)) return it;
  it.b = b;
  it.s = s;
  it.tile = index - before;
  return it;
}

// Item `index` of the batch. Every wave finds it by itself, a sequence a lane. A part's
// tokens are all of them where the tiles fill the card by themselves, else such that there
// are at most a.target items: the batch's tokens (of every tile) over a.target where that
// comes out, else over a.target less one a tile, which always does (the sums' fp32 rounding is
// below the allowance of 2^-18; a chunk of 2^30 is all of any sequence). `tiles_cut` is the batch's number of tiles where they are
// cut, else 0.
__device__ Item find_item(const AttentionArgs& a, int columns, int index, int& tiles_cut) {
  tiles_cut = 0;
  if (!a.part_out && a.b.sequences > (a.b.starts ? 4 : 1) * kWave) return find_whole(a, columns, index);
  const int lane = threadIdx.x & 63;
  auto mine = [&](int b) {
    KvSeq s{0, 0, 0, 0};
    if (b < a.b.sequences) s = kv_seq(a.b, b);
    return s;
  };
  KvSeq s = mine(lane);
  int chunk = 1 << 30;
  if (a.part_out) {
    // Sum over the batch of what f says of a sequence's tiles and tokens.
    auto over_batch = [&](auto&& f) {
      float sum = 0.0f;
      for (int b0 = 0; b0 < a.b.sequences; b0 += kWave) {
        const KvSeq o = b0 ? mine(b0 + lane) : s;
        sum += wave_sum(f((float)tiles_of(a, o, columns), tokens_of(a, o)));
      }
      return sum;
    };
    const float tiles = over_batch([](float t, int) { return t; });
    if (tiles < (float)a.target) {
      const float tokens = over_batch([](float t, int n) { return t * (float)n; }) * (1.0f + 0x1p-18f);
      auto chunk_for = [&](float parts) { return max(a.min_chunk, 64 * ((int)fminf(tokens / (64.0f * parts), 0x1p24f - 1.0f) + 1)); };
      chunk = chunk_for((float)a.target);
      const float items = over_batch([&](float t, int n) { return t * (float)max(1, (n + chunk - 1) / chunk); });
      if (items > (float)a.target) chunk = chunk_for((float)a.target - tiles);
      tiles_cut = (int)tiles;
    }
  }
  int before = 0, tiles_before = 0;
  for (int b0 = 0; b0 < a.b.sequences; b0 += kWave) {
    if (b0) s = mine(b0 + lane);
    const int tiles = tiles_of(a, s, columns);
    const int parts = max(1, (tokens_of(a, s) + chunk - 1) / chunk);
    const int upto = wave_upto(tiles * parts), tiles_upto = wave_upto(tiles);
    const uint64_t hit = __ballot(index < before + upto);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      Item it;
      it.b = b0 + l;
      it.s = KvSeq{of(s.start), of(s.n), of(s.first), of(s.len)};
      it.parts = of(parts);
      const int first = before + of(upto) - of(tiles) * it.parts, local = index - first;
      it.tile = local / it.parts;
      it.part = local - it.tile * it.parts;
      it.entry = first + it.tile * it.parts;
      it.index = tiles_before + of(tiles_upto) - of(tiles) + it.tile;
      return it;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    tiles_before += __builtin_amdgcn_readlane(tiles_upto, 63);
  }
  Item none{};
  none.b = -1;
  return none;
}

// For the joining kernel: how many tiles are cut, and each one's first row, columns from
// there on, first item and parts. Part 0 of each writes its own.
__device__ __forceinline__ void tell_join(const AttentionArgs& a, const Item& it, int columns, int tiles_cut) {
  if (!a.part_out || threadIdx.x != 0) return;
  if (blockIdx.x == 0) a.cut[0] = make_int4(tiles_cut, 0, 0, 0);
  if (tiles_cut && it.b >= 0 && it.part == 0)
    a.cut[1 + it.index] = make_int4(it.s.start, it.tile * columns, it.s.n * a.group, it.parts);
  if (tiles_cut && it.b >= 0 && it.part == 0) a.cut_entry[it.index] = it.entry;
}

// A sequence's last rows see the most tokens.
__device__ __forceinline__ void longest_first(const AttentionArgs& a, int columns, Item& it) {
  if (!a.causal) return;
  const int tiles = tiles_of(a, it.s, columns);
  it.entry += (tiles - 1 - 2 * it.tile) * it.parts;
  it.tile = tiles - 1 - it.tile;
}

// A column of an item: its row and head, and the tokens [lo, hi) that it sees.
struct Column {
  bool real;
  int row, head, lo, hi;
};
__device__ __forceinline__ Column column_of(const AttentionArgs& a, const KvSeq& s, int kv_head, int c) {
  Column o;
  o.real = c < s.n * a.group;
  const int i = c / a.group, position = (int)((uint32_t)s.first + (uint32_t)i);  // past an int only where it is none
  o.row = s.start + i;
  o.head = kv_head * a.group + c % a.group;
  // A column that is none has nothing written, and does not make a tile take the masked path.
  o.hi = a.causal && o.real ? min(s.len, position + 1) : s.len;
  o.lo = o.real ? lowest(a, position) : 0;
  return o;
}

// The tokens [from, to) of an item's part, whole tiles of `step`: those that its tile's
// columns see, cut evenly.
__device__ __forceinline__ void part_of(const AttentionArgs& a, const KvSeq& s, const Item& it, int columns, int step,
                                        int& from, int& to) {
  const int c1 = min(s.n * a.group, (it.tile + 1) * columns) - 1;
  const int first = s.first + it.tile * columns / a.group, last = s.first + c1 / a.group;
  const int hi = a.causal ? min(s.len, last + 1) : s.len;
  const int lo = lowest(a, first) / step * step;
  const int each = ((max(hi - lo, 0) + it.parts - 1) / it.parts + step - 1) / step * step;
  from = min(lo + it.part * each, max(hi, 0));
  to = min(from + each, hi);
}

// Eight elements of q as halves, times 2^e where they are bf16.
template <bool F16>
__device__ __forceinline__ f16x8_t q_halves(const uint4& u, float factor) {
  if constexpr (F16) return __builtin_bit_cast(f16x8_t, u);
  f16x8_t r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = word_of(u, j);
    r[2 * j] = (_Float16)(lo_bf(w) * factor);
    r[2 * j + 1] = (_Float16)(hi_bf(w) * factor);
  }
  return r;
}
__device__ __forceinline__ uint32_t abs_most(const uint4& u, uint32_t most) {  // of bf16, as fp32 bits
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = word_of(u, j);
    most = max(most, max(w << 16 & 0x7fffffffu, w & 0x7fff0000u));
  }
  return most;
}
// 2^e with the largest of a row in [2^14, 2^15), and 2^-e; both are normal numbers.
__device__ __forceinline__ void row_factor(uint32_t most, float& factor, float& inverse) {
  const uint32_t field = min(253u, 268u - (most >> 23));
  factor = __uint_as_float(field << 23);
  inverse = __uint_as_float((254u - field) << 23);
}

// A negative scale goes into q, so that products' units are positive.
__device__ __forceinline__ uint4 flip_signs(uint4 u, uint32_t bits) {
  return make_uint4(u.x ^ bits, u.y ^ bits, u.z ^ bits, u.w ^ bits);
}
// What a product of halves is worth, in factors that stay in range where the whole does.
__device__ __forceinline__ float unit_of(float scale, float inverse) {
  static_assert(kKeyUnit == 0x1p24f, "two factors of 2^12");
  return fabsf(scale) * (inverse * 0x1p12f) * 0x1p12f;
}
// A unit so small that no score counts, but not zero: a hidden score, -inf, stays that. So for a
// page's value scale, which needs a logarithm and an inverse: a page never written holds zeros.
__device__ __forceinline__ float not_zero(float unit) { return unit < 0x1p-100f ? 0x1p-100f : unit; }

// Sum of eight halves times `each` on top of `sum`.
__device__ __forceinline__ float add_halves(const f16x8_t& h, float sum, float each = 1.0f) {
  const f16x2_t unit = {(_Float16)each, (_Float16)each};
#pragma unroll
  for (int j = 0; j < 4; ++j) sum = __builtin_amdgcn_fdot2(f16x2_t{h[2 * j], h[2 * j + 1]}, unit, sum, false);
  return sum;
}

__device__ __forceinline__ uint4 load16(const uint16_t* p) {
  uint4 u;
  __builtin_memcpy(&u, p, 16);
  return u;
}

template <bool F16>
__device__ __forceinline__ void put_out4(uint16_t* p, const float* v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_st2<F16>(v[0], v[1]), pack_st2<F16>(v[2], v[3]));
}

// The table's entry for a token of the sequence whose row it is; past the table's end, the
// last (no row sees such a token). It is looked at only where it is used: with a check here
// each load would be waited for on the spot, and all loads before it.
__device__ __forceinline__ int entry_of(const KvBatchArgs& g, const int32_t* row, int token) {
  return row[min(token >> g.page_shift, g.table_width - 1)];
}
__device__ __forceinline__ bool is_page(const KvBatchArgs& g, int id) { return (uint32_t)id < (uint32_t)g.pages; }
__device__ __forceinline__ int64_t place_of(const KvBatchArgs& g, int id, int kv_head) {
  return (int64_t)(is_page(g, id) ? id : 0) * g.kv_heads + kv_head;
}

// ---- few columns -------------------------------------------------------------

// 32 tokens of a wave, as loaded: lane (r = lane % 16, g = lane / 16) has bytes
// D/4 * g .. of key rows 8 (r / 4) + 4 t + r % 4, and bytes D/16 * r .. of value rows 8 g + j.
template <int D>
struct FewKeys {
  uint4 k[2][D / 64];
};
template <int D>
struct FewValues {
  uint32_t v[8][D / 64];
};
struct FewPages {
  int k, v;  // table entries of this lane's key rows and value rows
};
__device__ __forceinline__ FewPages few_pages(const AttentionArgs& a, const int32_t* table, int token) {
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  return FewPages{entry_of(a.b, table, token + 8 * (r >> 2)), entry_of(a.b, table, token + 8 * q)};
}
template <int D>
__device__ __forceinline__ void few_load_keys(const AttentionArgs& a, int kv_head, int token, int page, FewKeys<D>& t) {
  const KvBatchArgs& g = a.b;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int at = token + 8 * (r >> 2) + (r & 3);
  const int64_t place = place_of(g, page, kv_head);
  const int8_t* k = g.k + ((place << g.page_shift) + (at & ((1 << g.page_shift) - 1))) * D + (D / 4) * q;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < D / 64; ++j) t.k[i][j] = *reinterpret_cast<const uint4*>(k + 4 * i * D + 16 * j);
}
template <int D>
__device__ __forceinline__ void few_load_values(const AttentionArgs& a, int kv_head, int token, int page, FewValues<D>& t) {
  const KvBatchArgs& g = a.b;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int at = token + 8 * q;
  const int64_t place = place_of(g, page, kv_head);
  const int8_t* v = g.v + ((place << g.page_shift) + (at & ((1 << g.page_shift) - 1))) * D + (D / 16) * r;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (D == 128) {
      const uint2 w = *reinterpret_cast<const uint2*>(v + i * D);
      t.v[i][0] = w.x;
      t.v[i][1] = w.y;
    } else {
      t.v[i][0] = *reinterpret_cast<const uint32_t*>(v + i * D);
    }
  }
}
// The scales of the page that tokens 8 g .. lie in.
__device__ __forceinline__ float2 few_load_scales(const AttentionArgs& a, int kv_head, int page) {
  const int64_t place = place_of(a.b, page, kv_head);
  return make_float2(a.b.k_scales[place], a.b.v_scales[place]);
}

// Value operand of channels D/16 * r + N: byte N of the eight rows.
template <int N, int W>
__device__ __forceinline__ f16x8_t few_values(const uint32_t (&x)[8][W]) {
  f16x8_t o;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f16x2_t h = value_codes<N % 4>(x[2 * j][N / 4], x[2 * j + 1][N / 4]);
    o[2 * j] = h[0];
    o[2 * j + 1] = h[1];
  }
  return o;
}
template <int N, int NV, int NC, int W>
__device__ __forceinline__ void few_weigh(const uint32_t (&x)[8][W], const f16x8_t (&w)[NC], f32x4_t (&o)[NC][NV]) {
  if constexpr (N < NV) {
    const f16x8_t v = few_values<N>(x);
#pragma unroll
    for (int c = 0; c < NC; ++c) o[c][N] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w[c], o[c][N], 0, 0, 0);
    few_weigh<N + 1>(x, w, o);
  }
}

// NC * 16 columns a workgroup of four waves, which take the part's tiles of 32 tokens in turn; a
// wave has its next tile's codes on their way while it works, and no wave waits for another
// before the end, where their sums meet in LDS. Registers instead of LDS, because each code is
// used by one wave only; rows of an 8-bit product would be half the work, but the codes' bound is
// memory: 64 sequences (1.79 GB of codes) in 320 us are 5.6 TB/s, and one of 1407 tokens 6.8 us,
// of which a chain of loads (lengths, table, codes) is most. With more columns than fit one
// workgroup the chain of tiles decides: 512 rows of 16 heads of 128, 256 workgroups, 12.7 us.
template <bool F16, int D, int NC>
__global__ __launch_bounds__(256, D == 64 ? 7 - 2 * NC : 4 - NC) void attention_few_kernel(AttentionArgs a) {
  constexpr int COLS = 16 * NC, NK = D / 32, NV = D / 16, PAD = D + 4;
  __shared__ float joined[4][16][PAD];
  __shared__ float stat_m[4][COLS], stat_l[4][COLS];
  const int kv_head = blockIdx.x % a.b.kv_heads;
  int tiles_cut;
  Item it = find_item(a, COLS, blockIdx.x / a.b.kv_heads, tiles_cut);
  if (kv_head == 0) tell_join(a, it, COLS, tiles_cut);
  if (it.b < 0) return;
  const KvSeq& s = it.s;
  longest_first(a, COLS, it);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;

  // What the first tile needs is asked for before anything is waited for.
  uint4 raw[NC][NK];
  Column col[NC];
  const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    col[c] = column_of(a, s, kv_head, it.tile * COLS + 16 * c + r);
#pragma unroll
    for (int k = 0; k < NK; ++k)
      raw[c][k] = col[c].real ? load16(a.q + col[c].row * a.q_row + col[c].head * a.q_head + (D / 4) * g + 8 * k)
                              : make_uint4(0, 0, 0, 0);
  }
  int from, to;
  part_of(a, s, it, COLS, 32, from, to);
  // Keys of the next tile are asked for when this one's scores are done, values when
  // they are weighed; page numbers a tile earlier.
  const int32_t* table = a.b.table + (int64_t)it.b * a.b.table_width;
  FewKeys<D> t;
  FewValues<D> u;
  FewPages page{-1, -1}, next{-1, -1};
  float2 scale{};
  int token = from + 32 * wave;
  if (token < to) {
    page = few_pages(a, table, token);
    next = few_pages(a, table, token + 128);
    few_load_keys<D>(a, kv_head, token, page.k, t);
    few_load_values<D>(a, kv_head, token, page.v, u);
    scale = few_load_scales(a, kv_head, page.v);
  }

  f16x8_t q[NC][NK];
  float unit[NC];  // of a product of halves, times scale log2(e)
  float bias[NC];  // what the keys' 128 adds to one
  int all_lo = 0, all_hi = s.len;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
#pragma unroll
    for (int k = 0; k < NK; ++k) raw[c][k] = flip_signs(raw[c][k], flip);
    float factor = 1.0f;
    unit[c] = unit_of(a.scale, 1.0f);
    if constexpr (!F16) {
      uint32_t most = 0;
#pragma unroll
      for (int k = 0; k < NK; ++k) most = abs_most(raw[c][k], most);
      most = max(most, (uint32_t)__shfl_xor((int)most, 16, kWave));
      most = max(most, (uint32_t)__shfl_xor((int)most, 32, kWave));
      float inverse;
      row_factor(most, factor, inverse);
      unit[c] = unit_of(a.scale, inverse);
    }
#pragma unroll
    for (int k = 0; k < NK; ++k) q[c][k] = q_halves<F16>(raw[c][k], factor);
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < NK; ++k) sum = add_halves(q[c][k], sum);
    sum += __shfl_xor(sum, 16, kWave);
    sum += __shfl_xor(sum, 32, kWave);
    bias[c] = sum * (128.0f / kKeyUnit);
    all_lo = max(all_lo, col[c].lo);
    all_hi = min(all_hi, col[c].hi);
  }
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) {
    all_lo = max(all_lo, __shfl_xor(all_lo, m, kWave));
    all_hi = min(all_hi, __shfl_xor(all_hi, m, kWave));
  }
  all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  all_hi = __builtin_amdgcn_readfirstlane(all_hi);

  float m[NC], l[NC], seen[NC];  // seen: at most what all lanes of the column have in l
  f32x4_t o[NC][NV];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    m[c] = kLow;
    l[c] = 0.0f;
    seen[c] = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n) o[c][n] = f32x4_t{0, 0, 0, 0};
  }

  for (; token < to; token += 128) {
    const bool more = token + 128 < to;
    // Scores: keys 8 g + 4 i + e of the tile in element e of half i.
    f32x4_t z[NC][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int c = 0; c < NC; ++c) z[c][i] = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        const uint4& raw = t.k[i][k / 2];
        const uint32_t w0 = word_of(raw, 2 * (k & 1)) ^ 0x80808080u, w1 = word_of(raw, 2 * (k & 1) + 1) ^ 0x80808080u;
        const f16x2_t h[4] = {key_codes_lo(w0), key_codes_hi(w0), key_codes_lo(w1), key_codes_hi(w1)};
        const f16x8_t key = __builtin_bit_cast(f16x8_t, h);
#pragma unroll
        for (int c = 0; c < NC; ++c) z[c][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, q[c][k], z[c][i], 0, 0, 0);
      }
    }
    if (more) few_load_keys<D>(a, kv_head, token + 128, next.k, t);
    const float lv = __builtin_amdgcn_logf(not_zero(scale.y)), inverse_v = __builtin_amdgcn_rcpf(not_zero(scale.y));
    const bool there = is_page(a.b, page.v), whole = token >= all_lo && token + 32 <= all_hi && !__any(!there);
    f16x8_t w[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float unit_k = not_zero(unit[c] * scale.x), shift = __builtin_fmaf(-bias[c], unit_k, lv), inverse = inverse_v;
      if (!whole) {
        asm volatile("");  // a branch, not selects
        const int lo = col[c].lo - token - 8 * g, hi = there ? col[c].hi - token - 8 * g : 0;
        if (max(lo, 0) >= min(hi, 8)) {  // nothing of the page: nor of its scales, whatever they are
          unit_k = 1.0f;
          shift = 0.0f;
          inverse = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) z[c][e / 4][e % 4] = e >= lo && e < hi ? z[c][e / 4][e % 4] : -__builtin_inff();
      }
      auto score = [&](int e, float low) { return __builtin_fmaf(z[c][e / 4][e % 4], unit_k, low); };
      auto weight = [&](int e) { return exp2_fast(score(e, shift - m[c])); };
      auto held = [&](int e) { return exp2_fast(score(e, shift) - m[c]); };
      auto weigh = [&](auto&& by) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[c][e] = (_Float16)by(e);
        return add_halves(w[c], 0.0f, 1.0f / kLiftUnit);
      };
      float sum = weigh(weight);
      const bool again = __any(sum > kMost);
      if (again) {
        float top = kLow;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, score(e, shift));
        top = fmaxf(top, __shfl_xor(top, 16, kWave));
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        top = fmaxf(m[c], below(top));
        const float less = exp2_fast(m[c] - top);
        m[c] = top;
        l[c] *= less;
        seen[c] *= less;
#pragma unroll
        for (int n = 0; n < NV; ++n) o[c][n] *= less;
        sum = weigh(held);
      }
      if (__any(inverse > kLeast * seen[c])) {
        auto together = [&] {
          const float t = __builtin_fmaf(sum, inverse, l[c]);
          const float two = t + __shfl_xor(t, 16, kWave);
          return two + __shfl_xor(two, 32, kWave);
        };
        seen[c] = together();
        if (__any(inverse > kLeast * seen[c])) {  // the sum in fp32, whatever the halves lose
          sum = 0.0f;
          if (again) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += held(e);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += weight(e);
          }
          sum *= 1.0f / kLiftUnit;
          seen[c] = together();
        }
      }
      l[c] = __builtin_fmaf(sum, inverse, l[c]);
    }
    uint32_t x[8][D / 64];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < D / 64; ++j) x[i][j] = u.v[i][j] ^ 0x80808080u;
    few_weigh<0>(x, w, o);
    if (more) {
      few_load_values<D>(a, kv_head, token + 128, next.v, u);
      scale = few_load_scales(a, kv_head, next.v);
      page = next;
      next = few_pages(a, table, token + 256);
    }
  }

  // The waves' parts to one maximum, and together.
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    l[c] += __shfl_xor(l[c], 16, kWave);
    l[c] += __shfl_xor(l[c], 32, kWave);
    if (g == 0) {
      stat_m[wave][16 * c + r] = m[c];
      stat_l[wave][16 * c + r] = l[c];
    }
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int mine = 16 * c + r;
    const float most = fmaxf(fmaxf(stat_m[0][mine], stat_m[1][mine]), fmaxf(stat_m[2][mine], stat_m[3][mine]));
    const float less = exp2_fast(m[c] - most);
    if (c > 0) __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e)  // channels NV (4 g + e) ..
#pragma unroll
      for (int n = 0; n < NV; n += 4)
        *reinterpret_cast<f32x4_t*>(&joined[wave][r][NV * (4 * g + e) + n]) =
            f32x4_t{o[c][n][e] * less, o[c][n + 1][e] * less, o[c][n + 2][e] * less, o[c][n + 3][e] * less};
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (D / 4); i += 256) {
      const int cc = i / (D / 4), d = i % (D / 4) * 4, at = 16 * c + cc;
      const int column = it.tile * COLS + at;
      if (column >= s.n * a.group) continue;
      const float top = fmaxf(fmaxf(stat_m[0][at], stat_m[1][at]), fmaxf(stat_m[2][at], stat_m[3][at]));
      float total = 0.0f, v[4] = {0, 0, 0, 0};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        total = __builtin_fmaf(stat_l[x][at], exp2_fast(stat_m[x][at] - top), total);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += joined[x][cc][d + e];
      }
      if (it.parts == 1) {
        const float inverse = total == 0.0f ? 0.0f : kOutUnit / total;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= inverse;
        const int row = s.start + column / a.group, head = kv_head * a.group + column % a.group;
        put_out4<F16>(a.out + ((int64_t)row * a.heads + head) * D + d, v);
      } else {
        const int64_t slot = ((int64_t)(it.entry + it.part) * a.b.kv_heads + kv_head) * COLS + at;
        *reinterpret_cast<float4*>(a.part_out + slot * D + d) = make_float4(v[0], v[1], v[2], v[3]);
        if (d == 0) a.part_ml[slot] = make_float2(top, total);
      }
    }
  }
}

// ---- many columns ------------------------------------------------------------

// 32 columns a wave, WAVES (4 or 8) a workgroup; tiles of 16 tokens a wave in two LDS
// stages as halves: keys [tokens][D] and values transposed, [D][tokens], in 16-byte chunks
// whose places are XORed so that the 16 lanes of one access meet all banks.
template <int D>
__device__ __forceinline__ int key_at(int token, int chunk) {  // in chunks
  if constexpr (D == 128) return token * 16 + (chunk ^ ((token & 7) | (token >> 4 & 1) << 3));
  return token * 8 + (chunk ^ ((token >> 1 & 3) | (token >> 4 & 1) << 2));
}
template <int WAVES>
__device__ __forceinline__ int value_at(int channel, int chunk) {
  if constexpr (WAVES == 8) return channel * 16 + (chunk ^ ((channel ^ (channel >> 3)) & 15));
  return channel * 8 + (chunk ^ (((channel >> 1) ^ (channel >> 4)) & 7));
}

// What a wave brings of a tile: 16 of its tokens, which lie in one page, behind each other.
// Lanes take 16-byte pieces of key rows, and eight channels of D/32 value rows each: few and
// wide loads, since a compute unit takes about 12 cycles for each.
template <int D>
struct Staged {
  uint4 k[D / 64];
  uint2 v[D / 32];
  float ks, vs;
  bool there;
};

template <int D, int WAVES>
struct Stage {
  static constexpr int ROWS = D / 32;     // value rows a lane
  static constexpr int LOADS = D / 64 + ROWS;
  static constexpr int KEY_UNITS = D / 32;  // 16-byte chunks of halves a lane
  __device__ static int lane() { return threadIdx.x & 63; }
  __device__ static int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

  // Where the 16 tokens from `token` on start in a page whose table entry is `id`, in bytes of either array.
  __device__ static int64_t start(const AttentionArgs& a, int kv_head, int token, int id) {
    return ((place_of(a.b, id, kv_head) << a.b.page_shift) + (token & ((1 << a.b.page_shift) - 1))) * D;
  }
  __device__ static void load(const AttentionArgs& a, int64_t at, int piece, Staged<D>& t) {
    if (piece < D / 64)
      t.k[piece] = *reinterpret_cast<const uint4*>(a.b.k + at + 1024 * piece + 16 * lane());
    else if (piece < LOADS)
      t.v[piece - D / 64] = *reinterpret_cast<const uint2*>(a.b.v + at + (lane() / (D / 8) * ROWS + piece - D / 64) * D +
                                                            8 * (lane() % (D / 8)));
  }
  __device__ static void load_scales(const AttentionArgs& a, int kv_head, int id, Staged<D>& t) {
    const int64_t place = place_of(a.b, id, kv_head);
    t.ks = a.b.k_scales[place];
    t.vs = a.b.v_scales[place];
    t.there = is_page(a.b, id);
  }
  // Pieces on their way to a stage: unit of KEY_UNITS of keys, channel of 8 of values.
  __device__ static void store_keys(const Staged<D>& t, int unit, f16x8_t* to) {
    constexpr int lanes = D / 16;  // of a row
    const int h = unit % 2, token = 16 * wave() + unit / 2 * (64 / lanes) + lane() / lanes, chunk = 2 * (lane() % lanes) + h;
    const uint32_t w0 = word_of(t.k[unit / 2], 2 * h) ^ 0x80808080u, w1 = word_of(t.k[unit / 2], 2 * h + 1) ^ 0x80808080u;
    const f16x2_t c[4] = {key_codes_lo(w0), key_codes_hi(w0), key_codes_lo(w1), key_codes_hi(w1)};
    to[key_at<D>(token, chunk)] = __builtin_bit_cast(f16x8_t, c);
  }
  template <int N>
  __device__ static void store_value(const Staged<D>& t, f16x8_t* to) {
    const int channel = 8 * (lane() % (D / 8)) + N, token = ROWS * (lane() / (D / 8));  // of the wave's 16
    f16x2_t c[ROWS / 2];
#pragma unroll
    for (int j = 0; j < ROWS / 2; ++j) {
      const uint32_t x = N < 4 ? t.v[2 * j].x : t.v[2 * j].y, y = N < 4 ? t.v[2 * j + 1].x : t.v[2 * j + 1].y;
      c[j] = value_codes<N % 4>(x ^ 0x80808080u, y ^ 0x80808080u);
    }
    f16x8_t* chunk = to + value_at<WAVES>(channel, 2 * wave() + token / 8);
    __builtin_memcpy(reinterpret_cast<char*>(chunk) + token % 8 * 2, c, sizeof c);
  }
  __device__ static void store_values(const Staged<D>& t, int channel, f16x8_t* to) {
    if (channel == 0) store_value<0>(t, to);
    if (channel == 1) store_value<1>(t, to);
    if (channel == 2) store_value<2>(t, to);
    if (channel == 3) store_value<3>(t, to);
    if (channel == 4) store_value<4>(t, to);
    if (channel == 5) store_value<5>(t, to);
    if (channel == 6) store_value<6>(t, to);
    if (channel == 7) store_value<7>(t, to);
  }
  // float4 of the wave's 16 tokens: key scale, log2 of the value scale, its inverse, whether there is a page.
  __device__ static void store_scales(const Staged<D>& t, float4* to) {
    // The same from every lane: no branch among the matrix instructions.
    const float vs = not_zero(t.vs);
    to[wave()] = make_float4(t.ks, __builtin_amdgcn_logf(vs), __builtin_amdgcn_rcpf(vs), t.there ? 1.0f : 0.0f);
  }
  __device__ static void store(const Staged<D>& t, f16x8_t* keys_to, f16x8_t* values_to, float4* scales) {
#pragma unroll
    for (int unit = 0; unit < KEY_UNITS; ++unit) store_keys(t, unit, keys_to);
#pragma unroll
    for (int channel = 0; channel < 8; ++channel) store_values(t, channel, values_to);
    store_scales(t, scales);
  }
};

__device__ __forceinline__ f32x16_t zeros16() {
  f32x16_t z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}

// A workgroup's waves own 32 columns each and share tiles of 16 * WAVES tokens, which all of them
// convert to halves in LDS, once for all columns: two buffers, one barrier a tile. Within 64
// tokens the products of one half of the keys run beside the exponentials of the other, and the
// next tile's loads, conversions and stores stand between them, one a step; operands come from
// LDS four steps ahead. 32 x 32 x 16 products, since a wave's 32 columns then read each operand
// once.
// PAIRS: two waves share 32 columns, and each takes one half of every 64 tokens: for prompts
// whose columns are too few to fill the card otherwise, where the chain of tiles is what lasts
// (three of 200 rows and 16 heads 13.5 to 10.8 us).
//
// Bound: the matrix cores. 8192 rows of 16 heads of 128, causal, take 297 us (0.93 PFLOP/s; 290 to
// 298 by the card). With weights as they are, not lifted, they took 285 to 293, of which
// exponentials were 36, conversions 17 and reads of LDS 17.
template <bool F16, int D, int WAVES, bool PAIRS>
__global__ __launch_bounds__(64 * WAVES, 2) void attention_tile_kernel(AttentionArgs a) {
  static_assert(!PAIRS || WAVES == 4, "a pair's places in LDS are those of 64 tokens");
  constexpr int COLS = 32 * WAVES / (PAIRS ? 2 : 1), NK = D / 16, NV = D / 32;
  constexpr int TILE = 16 * WAVES, SUBS = TILE / 64;  // tokens, worked on 64 at a time
  constexpr int HALVES = PAIRS ? 1 : 2;               // of those 64, in turn
  __shared__ f16x8_t keys[2][TILE * D / 8];
  __shared__ f16x8_t values[2][TILE * D / 8];
  __shared__ float4 scales[2][WAVES];
  const int kv_head = blockIdx.x % a.b.kv_heads;
  int tiles_cut;
  Item it = find_item(a, COLS, blockIdx.x / a.b.kv_heads, tiles_cut);
  if (kv_head == 0) tell_join(a, it, COLS, tiles_cut);
  if (it.b < 0) return;
  const KvSeq& s = it.s;
  longest_first(a, COLS, it);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, g = lane >> 5;
  const int half = PAIRS ? __builtin_amdgcn_readfirstlane(wave >> 1) : 0;  // the one that this wave takes

  const Column col = column_of(a, s, kv_head, it.tile * COLS + 32 * (PAIRS ? wave & 1 : wave) + r);
  // What the first tile needs is asked for before anything is waited for.
  uint4 u[NK];  // channels 16 k + 8 g ..
#pragma unroll
  for (int k = 0; k < NK; ++k)
    u[k] = col.real ? load16(a.q + col.row * a.q_row + col.head * a.q_head + 16 * k + 8 * g) : make_uint4(0, 0, 0, 0);
  int from, to;
  part_of(a, s, it, COLS, TILE, from, to);
  const int32_t* table = a.b.table + (int64_t)it.b * a.b.table_width;
  using St = Stage<D, WAVES>;
  Staged<D> staged;
  const int mine = 16 * St::wave();  // of a tile's tokens, those that this wave brings
  // Table entry of the next tile's, one for the wave, but in a vector register: as a scalar
  // it would be waited for where it is loaded.
  int next = 0, mine_v = mine;
  asm("" : "+v"(mine_v));
  if (from < to) {
    const int id = entry_of(a.b, table, from + mine);
    next = entry_of(a.b, table, from + TILE + mine_v);
    const int64_t at = St::start(a, kv_head, from + mine, id);
#pragma unroll
    for (int i = 0; i < St::LOADS; ++i) St::load(a, at, i, staged);
    St::load_scales(a, kv_head, id, staged);
  }
  f16x8_t q[NK];
  float unit = unit_of(a.scale, 1.0f), bias = 0.0f;  // of a product of halves; what the keys' 128 adds to one
  {
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0;
#pragma unroll
    for (int k = 0; k < NK; ++k) u[k] = flip_signs(u[k], flip);
    float factor = 1.0f;
    if constexpr (!F16) {
      uint32_t most = 0;
#pragma unroll
      for (int k = 0; k < NK; ++k) most = abs_most(u[k], most);
      most = max(most, (uint32_t)__shfl_xor((int)most, 32, kWave));
      float inverse;
      row_factor(most, factor, inverse);
      unit = unit_of(a.scale, inverse);
    }
#pragma unroll
    for (int k = 0; k < NK; ++k) q[k] = q_halves<F16>(u[k], factor);
#pragma unroll
    for (int k = 0; k < NK; ++k) bias = add_halves(q[k], bias);
    bias = (bias + __shfl_xor(bias, 32, kWave)) * (128.0f / kKeyUnit);
  }
  int all_lo = col.lo, all_hi = col.hi, any_lo = col.lo, any_hi = col.hi;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    all_lo = max(all_lo, __shfl_xor(all_lo, m, kWave));
    all_hi = min(all_hi, __shfl_xor(all_hi, m, kWave));
    any_lo = min(any_lo, __shfl_xor(any_lo, m, kWave));
    any_hi = max(any_hi, __shfl_xor(any_hi, m, kWave));
  }
  all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  all_hi = __builtin_amdgcn_readfirstlane(all_hi);
  any_lo = __builtin_amdgcn_readfirstlane(any_lo);
  any_hi = __builtin_amdgcn_readfirstlane(any_hi);
  // The key row that this lane's row of a product stands for: lanes of half g then hold tokens 16 g .. in order.
  const int key_row = 16 * (r >> 2 & 1) + 4 * (r >> 3) + (r & 3);

  float m = kLow, l = 0.0f, seen = 0.0f;  // seen: at most what both lanes of the column have in l
  f32x16_t o[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) o[n] = zeros16();

  if (from < to) St::store(staged, keys[0], values[0], scales[0]);
  __syncthreads();
  // Places of this lane's operands, in bytes: an XOR away from each other, and the other stage's by one more.
  constexpr int STAGE = TILE * D * 2;
  int key_place[NK], value_place[8];
#pragma unroll
  for (int k = 0; k < NK; ++k) key_place[k] = 16 * key_at<D>(32 * half + key_row, 2 * k + g);
#pragma unroll
  for (int c = 0; c < 8; ++c) value_place[c] = 16 * value_at<WAVES>(r, (WAVES == 8 ? c / 2 * 4 + c % 2 : c) ^ (2 * g) ^ (4 * half));
  const char* key_base = reinterpret_cast<const char*>(keys);
  const char* value_base = reinterpret_cast<const char*>(values);
  int stage = 0;
  for (int token = from; token < to; token += TILE, stage ^= 1) {
    // The next tile's loads (behind the last one's, its own again, which nobody uses).
    const int ahead = token + TILE < to ? token + TILE : token;
    const int id = __builtin_amdgcn_readfirstlane(next);
    const int64_t at = St::start(a, kv_head, ahead + mine, id);
    St::load_scales(a, kv_head, id, staged);
    next = entry_of(a.b, table, ahead + TILE + mine_v);
    f16x8_t* keys_to = keys[stage ^ 1];
    f16x8_t* values_to = values[stage ^ 1];
#pragma unroll
    for (int t = 0; t < SUBS; ++t) {
      // Of the next tile's way into LDS, a unit of keys and a channel of values for each step
      // (with two halves of a tile keys in the first, values in the second).
      auto store_step = [&](int v) {
        if (t == 0 && v < St::KEY_UNITS) St::store_keys(staged, v, keys_to);
        if (t == SUBS - 1) {
#pragma unroll
          for (int channel = 4 / NV * v; channel < 4 / NV * (v + 1); ++channel) St::store_values(staged, channel, values_to);
          if (v == 2 * NV - 1) St::store_scales(staged, scales[stage ^ 1]);
        }
      };
      const int base = token + 64 * t + 32 * half;  // the first token that this wave works on
      if (base >= any_hi || base + 32 * HALVES <= any_lo) {  // no column of the wave sees them
        if (t == 0)
#pragma unroll
          for (int i = 0; i < St::LOADS; ++i) St::load(a, at, i, staged);
#pragma unroll
        for (int v = 0; v < 2 * NV; ++v) store_step(v);
        continue;
      }
      // Matrix instructions and the rest go side by side, in steps that the scheduler keeps:
      // the scores of the second 32 tokens beside the weights of the first, those weighed
      // beside the second weights, those weighed beside the next tile's way into LDS.
      // Operands are read from LDS four steps ahead.
      f16x8_t ring[4];
      auto fetch = [&](int j) {
        if (j < HALVES * NK) {
          ring[j % 4] = *reinterpret_cast<const f16x8_t*>(key_base + key_place[j % NK] + (64 * t + 32 * (j / NK)) * D * 2);
        } else if (j < HALVES * (NK + 2 * NV)) {
          // Chunk 8 t + 4 i + 2 g + h of channel 32 n + r, for i, h = c / 2, c % 2.
          const int v = j - HALVES * NK, n = v % NV, c = v / NV;
          const int chunk = (8 * t + 4 * (c / 2) + c % 2) ^ (WAVES == 8 ? 4 * n : 2 * n & 7);
          ring[j % 4] = *reinterpret_cast<const f16x8_t*>(value_base + value_place[WAVES == 8 ? chunk / 4 * 2 + chunk % 2 : chunk] + 32 * TILE * 2 * n);
        }
      };
      float4 sc[2];
#pragma unroll
      for (int i = 0; i < HALVES; ++i) sc[i] = scales[stage][4 * t + 2 * (half + i) + g];
      if (PAIRS) sc[1] = sc[0];
#pragma unroll
      for (int j = 0; j < 4; ++j) fetch(j);
      f32x16_t z[2] = {zeros16(), zeros16()};
      f16x8_t w[2][2];
      float unit_k[2], shift[2], inverse[2], sum[2];
      auto scores = [&](int i, int k) {
        const int j = i * NK + k;
        z[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[j % 4], q[k], z[i], 0, 0, 0);
        fetch(j + 4);
      };
      auto weighed = [&](int i, int v) {
        const int j = HALVES * NK + 2 * NV * i + v;
        o[v % NV] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[j % 4], w[i][v / NV], o[v % NV], 0, 0, 0);
        fetch(j + 4);
      };
      auto weight = [&](int i, int e) { return exp2_fast(__builtin_fmaf(z[i][e], unit_k[i], shift[i] - m)); };
      auto held = [&](int i, int e) { return exp2_fast(__builtin_fmaf(z[i][e], unit_k[i], shift[i]) - m); };
      auto weigh_by = [&](int i, int from_e, int to_e, auto&& by) {
        const f16x2_t unit = {(_Float16)(1.0f / kLiftUnit), (_Float16)(1.0f / kLiftUnit)};
#pragma unroll
        for (int e = from_e; e < to_e; e += 2) {
          const f16x2_t p = {(_Float16)by(i, e), (_Float16)by(i, e + 1)};
          w[i][e / 8][e % 8] = p[0];
          w[i][e / 8][e % 8 + 1] = p[1];
          sum[i] = __builtin_amdgcn_fdot2(p, unit, e ? sum[i] : 0.0f, false);
        }
      };
      auto weigh = [&](int i, int from_e, int to_e) { weigh_by(i, from_e, to_e, weight); };
#pragma unroll
      for (int i = 0; i < HALVES; ++i) {
        unit_k[i] = not_zero(unit * sc[i].x);
        shift[i] = __builtin_fmaf(-bias, unit_k[i], sc[i].y);
        inverse[i] = sc[i].z;
      }
      const bool partly = base < all_lo || base + 32 * HALVES > all_hi || __any(sc[0].w * sc[1].w == 0.0f);
      auto hide = [&](int i) {
        if (!partly) return;
        asm volatile("");  // a branch: as selects this would be most of the tile's instructions
        const int at = base + 32 * i + 16 * g, lo = col.lo - at, hi = sc[i].w != 0.0f ? col.hi - at : 0;
        if (max(lo, 0) >= min(hi, 16)) {  // nothing of the page: nor of its scales, whatever they are
          unit_k[i] = 1.0f;
          shift[i] = 0.0f;
          inverse[i] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) z[i][e] = e >= lo && e < hi ? z[i][e] : -__builtin_inff();
      };
      auto settle = [&](int i) {
        const bool again = __any(sum[i] > kMost);
        if (again) {
          float top = kLow;
#pragma unroll
          for (int e = 0; e < 16; ++e) top = fmaxf(top, __builtin_fmaf(z[i][e], unit_k[i], shift[i]));
          top = fmaxf(top, __shfl_xor(top, 32, kWave));
          top = fmaxf(m, below(top));
          const float less = exp2_fast(m - top);
          m = top;
          l *= less;
          seen *= less;
#pragma unroll
          for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[n][e] *= less;
          weigh_by(i, 0, 16, held);
        }
        if (__any(inverse[i] > kLeast * seen)) {
          auto together = [&] {
            const float t = __builtin_fmaf(sum[i], inverse[i], l);
            return t + __shfl_xor(t, 32, kWave);
          };
          seen = together();
          if (__any(inverse[i] > kLeast * seen)) {  // the sum in fp32, whatever the halves lose
            sum[i] = 0.0f;
            if (again) {
#pragma unroll
              for (int e = 0; e < 16; ++e) sum[i] += held(i, e);
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) sum[i] += weight(i, e);
            }
            sum[i] *= 1.0f / kLiftUnit;
            seen = together();
          }
        }
        l = __builtin_fmaf(sum[i], inverse[i], l);
      };
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        scores(0, k);
        if (t == 0 && k < St::LOADS) St::load(a, at, k, staged);
        __builtin_amdgcn_sched_barrier(0);
      }
      hide(0);
      if constexpr (PAIRS) {
        weigh(0, 0, 16);
        settle(0);
      } else {
#pragma unroll
        for (int k = 0; k < NK; ++k) {
          scores(1, k);
          weigh(0, 16 / NK * k, 16 / NK * (k + 1));
          __builtin_amdgcn_sched_barrier(0);
        }
        settle(0);
        hide(1);
#pragma unroll
        for (int v = 0; v < 2 * NV; ++v) {
          weighed(0, v);
          weigh(1, 8 / NV * v, 8 / NV * (v + 1));
          __builtin_amdgcn_sched_barrier(0);
        }
        settle(1);
      }
#pragma unroll
      for (int v = 0; v < 2 * NV; ++v) {
        weighed(HALVES - 1, v);
        store_step(v);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int k = 0; k < NK; ++k) key_place[k] ^= STAGE;
#pragma unroll
    for (int c = 0; c < 8; ++c) value_place[c] ^= STAGE;
    __syncthreads();
  }

  l += __shfl_xor(l, 32, kWave);
  if constexpr (PAIRS) {  // the second half's sums to the first's wave, through LDS that nobody reads now
    float* sums = reinterpret_cast<float*>(keys) + (wave & 1) * NV * 16 * 64 + lane;
    float2* stats = reinterpret_cast<float2*>(values) + (wave & 1) * 64 + lane;
    if (half) {
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) sums[(n * 16 + e) * 64] = o[n][e];
      *stats = make_float2(m, l);
    }
    __syncthreads();
    if (half) return;
    const float2 other = *stats;
    const float most = fmaxf(m, other.x), mine_less = exp2_fast(m - most), other_less = exp2_fast(other.x - most);
    m = most;
    l = l * mine_less + other.y * other_less;
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[n][e] = o[n][e] * mine_less + sums[(n * 16 + e) * 64] * other_less;
  }
  // Found again: kept across the tiles it would take registers that those are short of.
  int thread = threadIdx.x;  // of the first COLS * 2
  asm volatile("" : "+v"(thread));
  const Column column = column_of(a, s, kv_head, it.tile * COLS + thread / 64 * 32 + thread % 32);
  if (!column.real) return;
  if (it.parts == 1) {
    const float inverse = l == 0.0f ? 0.0f : kOutUnit / l;
    uint16_t* out = a.out + ((int64_t)column.row * a.heads + column.head) * D;
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {  // channels 32 n + 8 (e / 4) + 4 g ..
        const float v[4] = {o[n][e] * inverse, o[n][e + 1] * inverse, o[n][e + 2] * inverse, o[n][e + 3] * inverse};
        put_out4<F16>(out + 32 * n + 2 * e + 4 * g, v);
      }
  } else {
    const int64_t slot = ((int64_t)(it.entry + it.part) * a.b.kv_heads + kv_head) * COLS + thread / 64 * 32 + thread % 32;
    float* out = a.part_out + slot * D;
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<float4*>(out + 32 * n + 2 * e + 4 * g) = make_float4(o[n][e], o[n][e + 1], o[n][e + 2], o[n][e + 3]);
    if (g == 0) a.part_ml[slot] = make_float2(m, l);
  }
}

// ---- parts together ----------------------------------------------------------

// Of one value a thread over aligned groups of GROUP threads (32, or all 256 by way of `part`).
template <int GROUP, typename F>
__device__ __forceinline__ float group_reduce(float v, float* part, F&& f) {
#pragma unroll
  for (int m = 1; m < (GROUP < 64 ? GROUP : 64); m <<= 1) v = f(v, __shfl_xor(v, m, kWave));
  if constexpr (GROUP > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = f(f(part[0], part[1]), f(part[2], part[3]));
  }
  return v;
}

// A workgroup for EACH columns (1 or 8) of a tile that was cut into parts, `blocks` of them a
// tile: a column's threads first look at a part's maximum and sum each, then teams of D/4
// threads read the parts' sums.
constexpr int kJoinParts = 256;  // parts whose factors are held at once
template <bool F16, int D, int EACH>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionArgs a, int columns, int blocks) {
  constexpr int GROUP = 256 / EACH, LANES = D / 4, WAYS = GROUP / LANES, AHEAD = 4;
  __shared__ float factors[EACH][kJoinParts];
  __shared__ float4 sums[256];
  __shared__ float part0[4], part1[4];
  const int kv_head = blockIdx.y, tile = blockIdx.x / blocks;
  const int count = a.cut[0].x;
  const int4 info = a.cut[1 + tile];  // first row, first column, columns of the sequence, parts
  const int entry = a.cut_entry[tile];
  if (tile >= count || info.w == 1) return;
  const int of = threadIdx.x / GROUP, t = threadIdx.x % GROUP, way = t / LANES, d = t % LANES * 4;
  const int64_t step = (int64_t)a.b.kv_heads * columns;
  const int at = blockIdx.x % blocks * EACH + of, column = info.y + at;
  const int parts = column < info.z ? info.w : 0;  // none where there is no column
  const int64_t slot = ((int64_t)entry * a.b.kv_heads + kv_head) * columns + at;
  const float* sums_at = a.part_out + slot * D + d;
  float4 ahead[AHEAD];  // asked for with the statistics
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (way + i * WAYS < parts) ahead[i] = *reinterpret_cast<const float4*>(sums_at + (way + i * WAYS) * step * D);
  float most = kLow;
  for (int p = t; p < parts; p += GROUP) most = fmaxf(most, a.part_ml[slot + p * step].x);
  most = group_reduce<GROUP>(most, part0, [](float x, float y) { return fmaxf(x, y); });
  float total = 0.0f;
  float4 v = make_float4(0, 0, 0, 0);
  for (int p0 = 0; p0 < info.w; p0 += kJoinParts) {
    const int n = min(kJoinParts, parts - p0);
    for (int p = t; p < n; p += GROUP) {
      const float2 ml = a.part_ml[slot + (p0 + p) * step];
      const float f = exp2_fast(ml.x - most);
      factors[of][p] = f;
      total = __builtin_fmaf(ml.y, f, total);
    }
    __syncthreads();
    auto add = [&](const float4& x, float f) {
      v.x = __builtin_fmaf(x.x, f, v.x);
      v.y = __builtin_fmaf(x.y, f, v.y);
      v.z = __builtin_fmaf(x.z, f, v.z);
      v.w = __builtin_fmaf(x.w, f, v.w);
    };
    if (p0 == 0) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (way + i * WAYS < n) add(ahead[i], factors[of][way + i * WAYS]);
    }
#pragma unroll 4
    for (int p = way + (p0 == 0 ? AHEAD * WAYS : 0); p < n; p += WAYS)
      add(*reinterpret_cast<const float4*>(sums_at + (p0 + p) * step * D), factors[of][p]);
    __syncthreads();
  }
  total = group_reduce<GROUP>(total, part1, [](float x, float y) { return x + y; });
  if (WAYS > 1) {
    sums[threadIdx.x] = v;
    __syncthreads();
  }
  if (way || !parts) return;
#pragma unroll
  for (int w = 1; w < WAYS; ++w) {
    const float4 o = sums[threadIdx.x + w * LANES];
    v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
  }
  const float inverse = total == 0.0f ? 0.0f : kOutUnit / total;
  const float x[4] = {v.x * inverse, v.y * inverse, v.z * inverse, v.w * inverse};
  const int row = info.x + column / a.group, head = kv_head * a.group + column % a.group;
  put_out4<F16>(a.out + ((int64_t)row * a.heads + head) * D + d, x);
}

template <bool F16, int D>
void launch_as(const AttentionPlan& p, const AttentionArgs& a, hipStream_t s) {
  const dim3 grid((uint32_t)p.items * a.b.kv_heads);
  auto* kernel = p.columns == 16    ? attention_few_kernel<F16, D, 1>
                 : p.columns == 32  ? attention_few_kernel<F16, D, 2>
                 : p.columns == 64  ? attention_tile_kernel<F16, D, 4, true>
                 : p.columns == 128 ? attention_tile_kernel<F16, D, 4, false>
                                    : attention_tile_kernel<F16, D, 8, false>;
  tfm_launch(kernel, grid, dim3(p.columns == 256 ? 512 : 256), 0, s, a);
  check_hip(hipGetLastError(), "cache_attention launch");
  if (!p.split) return;
  // Tiles of columns that can be cut: fewer than the target.
  const int64_t tiles = (int64_t)a.b.rows * a.group / p.columns + a.b.sequences;
  const int cut = (int)std::min<int64_t>(tiles, p.target);
  const int used = std::min(p.columns, a.b.max_rows * a.group);
  auto join = [&](auto* kernel, int each) {
    const int blocks = (used + each - 1) / each;
    tfm_launch(kernel, dim3(cut * blocks, a.b.kv_heads), dim3(256), 0, s, a, p.columns, blocks);
  };
  // Few columns in all: a workgroup each; many: several share one (1280 x 8 columns of 5 drafted rows 9.5 to 4.6 us).
  if ((int64_t)cut * used * a.b.kv_heads <= 1024)
    join(attention_join_kernel<F16, D, 1>, 1);
  else
    join(attention_join_kernel<F16, D, 8>, 8);
  check_hip(hipGetLastError(), "cache_attention join launch");
}

}  // namespace

// Whether the few kernel takes many columns sooner than the tile kernel. Its waves wait for nobody
// and each takes its own tokens, 32 columns a workgroup, so a call lasts a quarter of the chain of
// tiles while its workgroups are there at once or nearly; but each brings and converts its tokens
// for 32 columns only, which is most of the work with heads of 128. Measured, us, tile and few (as are
// the figures below, before weights were lifted, which in prompts and chunks costs either 2 to 7 %):
// - 16 heads of 128: a prompt of 400 rows 16.2 and 12.3, 700 behind 100 tokens 21.7 and 16.6, behind
//   1500 37.7 and 33.9, behind 3000 46.7 and 54.5; 8 of 60 rows behind 1000 30 and 19.5; 16 of 50
//   behind 100 11.9 and 13.2, behind 1500 49 and 30.5; 8 of 150 behind 500 23.9 and 26.2, behind 1000
//   44 and 34; 1300 behind 100 40.5 and 32.3, behind 1500 58.7 and 58.1; 4 of 1000 44 and 62.
// - 24 heads of 64 over 8: 400 rows behind 500 18.5 and 12.7, behind 3000 32.0 and 32.4; 16 of 50
//   behind 1000 32 and 19; 8 of 150 behind 100 11.7 and 14.6, behind 500 19.5 and 19.7, behind 3000 73
//   and 56; 4 of 300 behind 1500 46 and 30; 1300 behind 1000 45 and 37; 3 of 1000 behind 500 45 and 49.
static bool few_suffice(int head_dim, int64_t n32, int64_t capacity) {
  if (n32 <= 512) return (n32 <= 256 || capacity >= 400) && n32 * capacity <= (head_dim == 64 ? 1200000 : 1000000);
  if (head_dim == 64) return n32 <= 1536 && capacity >= 600;
  return n32 <= 1024 && capacity > 1024 && n32 * capacity <= 1500000;
}

// Sequences of a batch past which none is cut, since each workgroup of one that may be looks at all of
// them. One key head of 64, us, cut and whole: 8 sequences of 20000 tokens among 1000 empty ones 40 and 103,
// 2000 75 and 104, 4000 127 and 104; 2000 and 4000 of 30 tokens 43 and 12, 127 and 21.
constexpr int kMaxCutSequences = 2048;

// How a call is cut. Measured on one card, us:
// - 32 columns at most, least tokens of a part: 1 x 1407 tokens of 16 heads 9.8 with 128, 10.5 with
//   256, 13.5 with 512 (one part 16.1).
// - The same, tokens from which on a sequence is cut, by the workgroups without (a launch and the join
//   cost 3 to 5): 16 heads of 128, one token after 500 9.9 cut and 8.3 whole, after 800 9.8 and 10.9;
//   16 sequences after 1100 19.3 and 15.4, after 2000 27 and 27; 32 after 3000 62 and 60; 24 heads of
//   64 over 8, one after 800 9.8 and 8.5, after 1500 9.6 and 11.6; 64 after 2000 25.8 and 24.0; 300 rows
//   behind 900 19.0 and 14.0, 512 behind 1500 25.8 and 22.3.
// - many columns: four waves (two workgroups a compute unit) or eight (one, which brings and
//   converts a tile for twice the columns, at 1.15 of the rate: 8192 rows of 16 heads 335 against
//   289). Eight where a sequence's columns do not leave 1 / 1.15 of its tiles empty, and either
//   there are two rounds of them, or less than the rounds of four come to (7 chunks of 129 to 815
//   rows 45 against 63), or tiles are cut along many tokens (800 rows behind 30000 tokens, 32
//   heads: 438 against 507; behind 500: 43 against 42).
// - many columns, two waves to 32 of them (64 a workgroup): where 128 a workgroup would leave most
//   compute units without one and their chain of tiles is short. Three of 200 rows and 16 heads 13.5
//   to 10.8, 8 of 60 rows behind 200 tokens, 4 key heads of 128, 16.0 to 13.0, 8 of 64 11.9 to 10.1;
//   16 of 40 rows behind none 10.0 to 11.4 and 7.4 to 6.8; with 240 workgroups of 128, 12.4 to 14.4.
// - many columns, least tokens of a part: 48 rows behind 4000 tokens 25 with 512, 36 with 1024.
// - more columns in the few kernel, least tokens of a part: 5 rows of 32 heads over 4 behind 1500 16.0
//   with 512, 13.9 with 256; 48 rows of them behind 1500 16.6 and 19.9, behind 4000 23.1 and 23.8.
// - tiles, tokens from which on they are cut: 24 heads of 64 over 8, 8 of 60 rows behind 500 17.4 cut and
//   13.4 whole; 700 rows behind 100 19.5 and 17.1; of 128, 4 key heads, 16 of 50 behind 500 30 and 23.
AttentionPlan attention_plan(int64_t rows, int group, int kv_heads, int head_dim, int sequences, int max_rows,
                             int64_t capacity) {
  AttentionPlan p{};
  const int64_t most = (int64_t)max_rows * group, all = rows * group;
  const int64_t n32 = (all + 31) / 32 * kv_heads, n128 = (all + 127) / 128 * kv_heads, n256 = (all + 255) / 256 * kv_heads;
  int64_t whole;  // tokens from which on a sequence may be cut
  int resident;   // workgroups that the card holds at once
  if (most <= 32 || few_suffice(head_dim, n32, capacity)) {
    p.columns = most <= 16 ? 16 : 32;
    resident = 256 * (head_dim == 64 ? 7 - p.columns / 8 : 4 - p.columns / 16);
    p.min_chunk = most <= 32 ? 128 : n32 * capacity <= 56000 ? 256 : 512;
    const int64_t uncut = std::min<int64_t>(all / p.columns + sequences, sequences * ((most + p.columns - 1) / p.columns)) * kv_heads;
    whole = head_dim == 64 ? 900 + 4 * uncut : 600 + 5 * uncut;
  } else {
    const int64_t rest = n128 % 512;
    const bool fits = 20 * ((most + 255) / 256 * 2) <= 23 * ((most + 127) / 128);
    const bool even = n256 >= 512 || (n256 < 256 ? capacity >= 4096
                                                 : 20 * ((n256 + 255) / 256) <= 23 * (n128 / 512) + (rest > 256 ? 23 : rest ? 13 : 0));
    p.columns = fits && even ? 256 : n128 <= 192 && capacity <= 1024 ? 64 : 128;
    resident = p.columns == 256 ? 256 : 512;
    p.min_chunk = 512;
    whole = 1024;
  }
  p.target = std::max(1, resident / kv_heads);
  const int64_t tiles = std::min<int64_t>(all / p.columns + sequences, all);
  // Where the rows by themselves make enough tiles, or one workgroup reads so few tokens, none is cut.
  p.split = capacity > whole && all / p.columns < p.target && sequences <= kMaxCutSequences;
  p.items = (int)std::max<int64_t>(1, p.split ? std::max<int64_t>(tiles, p.target) : tiles);
  return p;
}

void launch_cache_attention(bool f16, int head_dim, const AttentionPlan& p, const AttentionArgs& a, hipStream_t s) {
  if (head_dim == 64)
    f16 ? launch_as<true, 64>(p, a, s) : launch_as<false, 64>(p, a, s);
  else
    f16 ? launch_as<true, 128>(p, a, s) : launch_as<false, 128>(p, a, s);
}

}  // namespace tfm
