// Attention of a few query tokens of each sequence over its paged FP8 cache: decode, trees of drafted tokens, chunks
// of a prompt. gfx950 only.
//
// Row (t, h): query token t of a sequence, query head h of a kv head's group. The sequence's last T positions are its T
// query tokens, the ctx = len - T before them are seen by every row, and token t sees token j where mask[t][j] (without
// a mask: j <= t). With codes c and scales s of keys and values, in base 2:
//   x_p = (q . ck_p) * (sk_p * softmax_scale * log2 e),  m = max x_p,  l = sum 2^(x_p - m),
//   o = sum (2^(x_p - m) * sv_p) cv_p / l.
// A scale belongs to a token, so it multiplies a column of the scores and of the weights, never the codes: codes turn
// into bf16 (keys into fp16 against fp16 queries) exactly, two an instruction, and the products run on matrix units.
// The weights times sv become bf16 for that, whatever the queries' type: fp16's range would hold neither a value that fp16
// does not, nor the weights of a row that one position draws to itself. Up to 32 rows, where memory is the bound, and for
// fp16 queries they are two bf16 pieces (what is lost is at most 2^-16 of a term); for bf16 ones in tiles of more rows,
// which the products bound, they are one (2^-8, half a step of the output's type): 2048 tokens of two prompts over 8192 take
// 581 us with one and 731 with two. (One fp16 piece, whose range needs the scales in the codes' conversions, took 742.)
// Scores, maxima, sums and outputs stay in fp32. Products of codes with e4m3 pieces of q would need no conversions of
// keys, but a chain of them sums to 2^-15 of its size on this hardware (bf16 and fp16 products to 2^-23), which a log of a
// sum shows.
#include "common.h"

AKLR_SCALAR_FP32_BEGIN

namespace aklr {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4, kThreads = 256;
constexpr int kUnit = 128;  // tokens a workgroup takes in one step: 32 a wave
// Weights are 2^(x - m) for a reference m that is set kHead above the largest score so far and set again once a score
// is kRise above it. Floating-point sums lose nothing by that, and a row's reference rises at most every kHead + kRise
// powers of two: once for all where no score is 2^40 times the first ones'. Weights below 2^20 leave bf16 values to 2^100.
constexpr float kHead = 20.0f, kRise = 20.0f;
constexpr float kNone = -3e38f;   // the reference in a partial result of a row that saw nothing

struct AttnArgs {
  const void* q;
  int64_t q_token, q_head;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  int64_t code_page, scale_page;  // bytes from one page to the next, of keys and of values
  const int32_t* table;
  int64_t table_row;
  const int32_t *lens, *starts;
  const uint8_t* mask;
  int64_t mask_row;
  void* out;
  float* lse;
  float* part;        // partial results, and before them the arrival words
  uint64_t* word;
  uint32_t page_magic;  // 2^32 / (page / 8), rounded up
  int table_cols, mask_cols, total, batch, hq, hkv, group, page, pages;
  // Work items a kv head is cut into: as many as run at once where its tiles are few, else `target` beside one a tile
  int slots, target;
  int dim;     // of a head
  int wide;    // page % 32 == 0
  int held;    // partial results a kv head can have
  int words;   // tiles of rows a kv head can have: arrival words
  int joiners;  // workgroups of a kernel of its own that join a tile's partial results; 0: the last of those that wrote them does
  float scale_log2;
};

// What one workgroup does. Every workgroup works it out from the lengths on the device, so no length has to be known
// to the host and a captured launch serves other lengths: rows are cut into tiles of R, a sequence's tokens into
// chunks of `chunk` units, the same for all sequences and so that the items come to about `target`.
struct Item {
  int b, tiles, tile, split, splits, chunk;
  int q0, count, len;  // the sequence's first query token, how many, its positions
  int row_tile;        // the tile's number over all sequences
  int slot;            // of the partial result of the tile's first split, where there are several
  bool ok;
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Item `index` of a kv head: items are the tiles of each sequence's first chunk, of its second, ..., then the next
// sequence's. TILE: the first item of tile `index` of a kv head. Wave-wide: lane i looks at sequence i of each 64.
template <int R, bool TILE = false>
__device__ __forceinline__ Item find(const AttnArgs& a, int index) {
  const int lane = threadIdx.x & 63;
  const int64_t most = (int64_t)a.table_cols * a.page;
  struct One {
    int q0, count, len, tiles, units;
  };
  auto look = [&](int b) {
    One s{0, 0, 0, 0, 0};
    if (b < a.batch) {
      s.q0 = min(max(a.starts[b], 0), a.total);
      s.count = min(max(a.starts[b + 1], s.q0), a.total) - s.q0;
      s.len = (int)min((int64_t)max(a.lens[b], 0), most);
      s.tiles = (int)(((int64_t)s.count * a.group + R - 1) / R);
      s.units = max(1, (s.len + kUnit - 1) / kUnit);
    }
    return s;
  };
  One s = look(lane);
  int64_t work = (int64_t)s.tiles * s.units;
  int all_tiles = s.tiles;
  for (int b0 = 64; b0 < a.batch; b0 += 64) {
    const One x = look(b0 + lane);
    work += (int64_t)x.tiles * x.units;
    all_tiles += x.tiles;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    work += __shfl_xor(work, d, 64);
    all_tiles += __shfl_xor(all_tiles, d, 64);
  }
  Item r{};
  const int target = all_tiles > 0 && 2 * all_tiles <= a.slots ? a.slots - all_tiles : a.target;
  r.chunk = uniform((int)fmin((double)work / target, (double)(1 << 23)) + 1);
  int items_before = 0, tiles_before = 0, held_before = 0;  // of the 64 sequences at hand
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (b0) s = look(b0 + lane);
    const int splits = (s.units + r.chunk - 1) / r.chunk;
    // inclusive sums over the lanes; only a tile of several splits has partial results
    int items = s.tiles * splits, tiles = s.tiles, held = splits > 1 ? items : 0;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(items, d, 64), y = __shfl_up(tiles, d, 64), z = __shfl_up(held, d, 64);
      if (lane >= d) items += x, tiles += y, held += z;
    }
    const uint64_t past = __ballot(TILE ? tiles_before + tiles > index : items_before + items > index);
    if (past) {
      const int at = __builtin_ctzll(past);
      auto take = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
      r.b = b0 + at;
      r.tiles = take(s.tiles);
      r.splits = take(splits);
      r.chunk = (take(s.units) + r.splits - 1) / r.splits;  // of even length
      r.slot = held_before + take(held) - r.tiles * r.splits;
      r.row_tile = tiles_before + take(tiles) - r.tiles;
      const int nth = TILE ? index - r.row_tile : index - (items_before + take(items) - r.tiles * r.splits);
      r.split = TILE ? 0 : nth / r.tiles;
      r.tile = nth - r.split * r.tiles;
      r.tile = r.tiles - 1 - r.tile;  // the last first: under causal masks it sees the most
      r.slot += r.tile;
      r.row_tile += r.tile;
      r.q0 = take(s.q0);
      r.count = take(s.count);
      r.len = take(s.len);
      // starts that do not ascend can make more of all than there is room for, or than an int counts
      r.ok = (unsigned)r.tile < (unsigned)r.tiles && (unsigned)r.split < (unsigned)r.splits &&
             (unsigned)r.row_tile < (unsigned)a.words &&
             (r.splits == 1 || (r.slot >= 0 && r.slot + (int64_t)(r.splits - 1) * r.tiles < a.held));
      return r;
    }
    items_before += __builtin_amdgcn_readlane(items, 63);
    tiles_before += __builtin_amdgcn_readlane(tiles, 63);
    held_before += __builtin_amdgcn_readlane(held, 63);
  }
  return r;
}

// A block table is read by scalar loads: a vector load's wait would also wait for the codes that are on their way.
typedef const int32_t __attribute__((address_space(4))) const_i32;
__device__ __forceinline__ const_i32* row_of(const int32_t* table, int64_t at) {
  return (const_i32*)reinterpret_cast<uintptr_t>(table + at);
}

template <typename F>
__device__ __forceinline__ float across(float v, F f) {  // f over the four 16-lane groups, in every lane
  const uint32_t u = __float_as_uint(v);
  const auto x = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  v = f(__uint_as_float(x[0]), __uint_as_float(x[1]));
  const uint32_t w = __float_as_uint(v);
  const auto y = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  return f(__uint_as_float(y[0]), __uint_as_float(y[1]));
}

template <bool F16, bool HIGH>
__device__ __forceinline__ uint32_t two(uint32_t codes) {  // two e4m3 codes of a word as bf16 (fp16)
  if constexpr (F16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, HIGH));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, HIGH));
}

template <bool F16>
__device__ __forceinline__ f32x4 mfma32(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// What follows for steps at an edge works on bit masks and selects by them, not by conditions: it stands beside the hot
// loops, which need the registers.
__device__ __forceinline__ uint32_t spread(uint32_t bits, int i) {  // bit i in all 32
  return (uint32_t)__builtin_amdgcn_sbfe((int)bits, i, 1);
}
__device__ __forceinline__ uint32_t sign(int v) { return (uint32_t)v >> 31; }

// Which of a lane's N tokens its row sees, four consecutive ones every STEP from the j0-th past the context, as bits.
template <int N, int STEP>
__device__ __forceinline__ uint32_t seen_by(const AttnArgs& a, uint32_t held, int j0, int row_t, int q0) {
  uint32_t sees = 0;
  if (a.mask) {
    const uint8_t* row = a.mask + (int64_t)(q0 + row_t) * a.mask_row;
#pragma unroll 1
    for (int b = 0; b < N / 4; ++b) {
      uint32_t four = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = j0 + STEP * b + i;
        const uint32_t on = a.mask_cols ? row[min(max(j, 0), a.mask_cols - 1)] : 0;
        four |= (sign(j) | (min(on, 1u) & sign(j - a.mask_cols))) << i;
      }
      sees |= four << (4 * b);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) sees |= sign(j0 + STEP * (i / 4) + i % 4 - row_t - 1) << i;
  }
  return sees & held;
}

// Which of a lane's N tokens are there: positions below `left` of those from its first, in 16-token blocks that are.
template <int N, int STEP>
__device__ __forceinline__ uint32_t held_by(int first, int left, uint32_t lo, uint32_t hi) {
  uint32_t held = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int token = first + STEP * (i / 4) + i % 4;
    held |= (sign(token - left) & (STEP * (i / 4) < 16 ? lo : hi)) << i;
  }
  return held;
}

// The words of a lane's N tokens as an edge needs them: what is not there is zero, and a token with a NaN code anywhere
// (the LANES lanes of a group hold its codes) gets a NaN scale in place of it, which only rows that see it multiply by.
template <int N, int LANES, int VW>
__device__ __forceinline__ void clean(uint32_t (*v)[VW], f32x4* s, uint32_t held) {
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint32_t nan = 0;
#pragma unroll
    for (int w = 0; w < VW; ++w) nan |= ((v[i][w] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
    bad |= min(nan, 1u) << i;
  }
#pragma unroll
  for (int d = 1; d < LANES; d *= 2) bad |= (uint32_t)__shfl_xor((int)bad, d, 64);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i / 4][i % 4] = __uint_as_float(__float_as_uint(s[i / 4][i % 4]) | (spread(bad, i) & 0x7FC00000u));
#pragma unroll
    for (int w = 0; w < VW; ++w) v[i][w] &= spread(held & ~bad, i);
  }
}

__device__ __forceinline__ float masked(float x, uint32_t sees, int i) {  // -infinity where bit i is not set
  const uint32_t on = spread(sees, i);
  return __uint_as_float((__float_as_uint(x) & on) | (0xFF800000u & ~on));
}
__device__ __forceinline__ float masked_weight(float w, uint32_t sees, int i) {  // 0 there, whatever it is
  return __uint_as_float(__float_as_uint(w) & spread(sees, i));
}

// Scores of a lane's NQ rows and 8 tokens become exponents, x - m. `limit` is kRise, or -infinity in a row that has
// seen nothing. True where some row of the wave has to lift its reference first; elsewhere nothing has to shrink, and
// the four lane groups that share a row need not agree on a maximum.
template <int NQ>
__device__ __forceinline__ bool relate(f32x4 (&x)[NQ][2], const f32x4 (&ks)[2], bool edge, const uint32_t (&sees)[NQ],
                                       const float (&m)[NQ], const float (&limit)[NQ]) {
  bool rise = false;
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int i = 0; i < 8; ++i) x[n][i / 4][i % 4] = fmaf(x[n][i / 4][i % 4], ks[i / 4][i % 4], -m[n]);
  if (edge) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[n][i / 4][i % 4] = masked(x[n][i / 4][i % 4], sees[n], i);
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, x[n][i / 4][i % 4]);
    rise |= top > limit[n];
  }
  return __ballot(rise) != 0;
}

// What the rows summed so far shrinks to their new references.
template <int NQ, int DT>
__device__ __forceinline__ void lift(f32x4 (&x)[NQ][2], float (&m)[NQ], float (&limit)[NQ], float (&l)[NQ],
                                     f32x4 (&o)[NQ][DT]) {
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float top = x[n][0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, x[n][i / 4][i % 4]);
    top = across(top, [](float u, float v) { return fmaxf(u, v); });
    const bool first = limit[n] != kRise;
    if (top > (first ? -__builtin_inff() : 0.0f)) {
      top += kHead;
      limit[n] = kRise;
    } else {
      top = 0.0f;
    }
    const float by = first ? 1.0f : __builtin_amdgcn_exp2f(-top);
    m[n] += top;
    l[n] *= by;
#pragma unroll
    for (int i = 0; i < DT; ++i) o[n][i] *= by;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[n][i / 4][i % 4] -= top;
  }
}

// Two weights as bf16, and what that leaves of them, as another two.
__device__ __forceinline__ uint32_t pieces(float a, float b, uint32_t& rest) {
  const uint32_t two = pack_bf16x2(a, b);
  rest = pack_bf16x2(a - bf16_lo(two), b - bf16_hi(two));
  return two;
}

// The weights, as the second product's operands. A bf16 keeps 8 bits of one, so what that leaves goes into a second: an
// output is then as near as its type lets it be, and where memory is the bound the matrix unit has the time for both (64
// sequences of up to 8192 tokens, group 8: 128.1 us with one bf16, 128.6 with two).
template <int NQ>
__device__ __forceinline__ void weigh(const f32x4 (&x)[NQ][2], const f32x4 (&vs)[2], bool edge,
                                      const uint32_t (&sees)[NQ], float (&l)[NQ], u32x4 (&hi)[NQ], u32x4 (&lo)[NQ]) {
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = __builtin_amdgcn_exp2f(x[n][i / 4][i % 4]);
      l[n] += e;
      w[i] = e * vs[i / 4][i % 4];
    }
    if (edge) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = masked_weight(w[i], sees[n], i);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t rest;
      hi[n][i] = pieces(w[2 * i], w[2 * i + 1], rest);
      lo[n][i] = rest;
    }
  }
}

// Four tokens' words of four codes turned over: out[e] holds dimension e of the four, two values a word.
__device__ __forceinline__ void turn_over(uint32_t a, uint32_t b, uint32_t c, uint32_t d, u32x2 (&out)[4]) {
  const uint32_t l0 = __builtin_amdgcn_perm(b, a, 0x05010400), l1 = __builtin_amdgcn_perm(d, c, 0x05010400);
  const uint32_t h0 = __builtin_amdgcn_perm(b, a, 0x07030602), h1 = __builtin_amdgcn_perm(d, c, 0x07030602);
  out[0] = u32x2{two<false, false>(l0), two<false, false>(l1)};
  out[1] = u32x2{two<false, true>(l0), two<false, true>(l1)};
  out[2] = u32x2{two<false, false>(h0), two<false, false>(h1)};
  out[3] = u32x2{two<false, true>(h0), two<false, true>(h1)};
}

// The same for two codes of a token.
__device__ __forceinline__ void turn_over2(uint32_t a, uint32_t b, uint32_t c, uint32_t d, u32x2 (&out)[2]) {
  const uint32_t l0 = __builtin_amdgcn_perm(b, a, 0x05010400), l1 = __builtin_amdgcn_perm(d, c, 0x05010400);
  out[0] = u32x2{two<false, false>(l0), two<false, false>(l1)};
  out[1] = u32x2{two<false, true>(l0), two<false, true>(l1)};
}

// Partial results: for each slot, o [R][D] not yet divided by l, then (m, l, -, -) [R].
template <int D, int R>
__device__ __forceinline__ rsrc_t slot_at(const AttnArgs& a, int head, int slot) {
  return make_rsrc(a.part + ((int64_t)head * a.held + slot) * (R * (D + 4)), R * (D + 4) * 4);
}

template <bool F16, int N>
__device__ __forceinline__ void store_row(void* out, int64_t at, const float (&v)[N], float by) {
  uint32_t* p = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(out) + at);
#pragma unroll
  for (int i = 0; i < N / 2; ++i)
    p[i] = pack_out2(v[2 * i] * by, v[2 * i + 1] * by, F16 ? AKLR_OUT_F16 : AKLR_OUT_BF16);
}

template <int N, bool F16>
__device__ __forceinline__ void finish(const AttnArgs& a, const Item& it, int head, int row, int d, float best, float total,
                                       const float (&v)[N]) {
  const int t = row / a.group, h = row - t * a.group;
  const int64_t at = (int64_t)(it.q0 + t) * a.hq + head * a.group + h;
  store_row<F16>(a.out, at * (a.dim) + d, v, total == 0.0f ? 0.0f : 1.0f / total);
  if (a.lse && d == 0) a.lse[at] = total == 0.0f ? -__builtin_inff() : (best + __log2f(total)) * 0.69314718f;
}

// Joins the splits of a tile's rows from `first` to `left`, by a workgroup. 16 lanes take a row; where there are fewer
// rows than 16-lane groups, the groups left over take every second, fourth, ... split each, and their sums meet in LDS
// (`sum`, a row of D + 4 floats for each group). Always in the same order.
template <int D, int R, bool F16>
__device__ __forceinline__ void join(const AttnArgs& a, const Item& it, int head, int first, int left, int r0, float* sum) {
  constexpr int DT = D / 16;
  const int all = blockDim.x >> 4;  // 16-lane groups
  const int chunk = (threadIdx.x & 15) * DT;
  int at_once = all;
  while (at_once > 1 && at_once / 2 >= left - first) at_once /= 2;
  const int groups = all / at_once, r = (threadIdx.x >> 4) % at_once, part = (threadIdx.x >> 4) / at_once;
  for (int base = first; base < left; base += at_once) {
    const int row = base + r;
    float best = kNone, total = 0.0f, v[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) v[i] = 0.0f;
    auto take = [&](float m, float s, const f32x4* x) {
      const float now = fmaxf(best, m);
      const float old = best == now ? 1.0f : __builtin_amdgcn_exp2f(best - now), by = m == now ? 1.0f : __builtin_amdgcn_exp2f(m - now);
      best = now;
      total = total * old + s * by;
#pragma unroll
      for (int i = 0; i < DT; ++i) v[i] = v[i] * old + x[i / 4][i % 4] * by;
    };
    if (row < left) {
#pragma unroll 4
      for (int s = part; s < it.splits; s += groups) {
        const rsrc_t from = slot_at<D, R>(a, head, it.slot + s * it.tiles);
        const f32x4 ml = load_partial4(from, R * D + 4 * row);
        f32x4 x[DT / 4];
#pragma unroll
        for (int i = 0; i < DT / 4; ++i) x[i] = load_partial4(from, row * D + chunk + 4 * i);
        take(ml[0], ml[1], x);
      }
    }
    if (groups > 1) {
      __syncthreads();
      float* mine = sum + (threadIdx.x >> 4) * (D + 4);
#pragma unroll
      for (int i = 0; i < DT; i += 4) *reinterpret_cast<f32x4*>(mine + chunk + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
      if (chunk == 0) mine[D] = best, mine[D + 1] = total;
      __syncthreads();
      if (part == 0) {
        for (int o = 1; o < groups; ++o) {
          const float* other = sum + (o * at_once + r) * (D + 4);
          f32x4 x[DT / 4];
#pragma unroll
          for (int i = 0; i < DT / 4; ++i) x[i] = *reinterpret_cast<const f32x4*>(other + chunk + 4 * i);
          take(other[D], other[D + 1], x);
        }
      }
    }
    if (part == 0 && row < left) finish<DT, F16>(a, it, head, r0 + row, chunk, best, total, v);
  }
}

// Joins all tiles of rows, `joiners` workgroups a tile.
template <int D, int R, bool F16>
__global__ __launch_bounds__(kThreads) void join_kernel(const AttnArgs a) {
  __shared__ float sum[kThreads / 16][D + 4];
  const int head = blockIdx.x % a.hkv, index = blockIdx.x / a.hkv;
  const Item it = find<R, true>(a, index / a.joiners);
  if (!it.ok || it.splits == 1) return;
  const int r0 = it.tile * R, left = min(R, it.count * a.group - r0), each = (R + a.joiners - 1) / a.joiners;
  const int first = index % a.joiners * each;
  join<D, R, F16>(a, it, head, first, min(left, first + each), r0, sum[0]);
}

// Up to 32 rows, or more in tiles of those: bound by memory, and where there is little by one chain of loads and a join.
// 64 sequences of up to 8192 tokens, 8 kv heads of 128, group 8: 129 us, 5.0 TB/s; 156 with codes loaded into registers.
// One sequence of 2048, group 4: 11.8 us.
//
// Rows by the 16 * NQ, tokens by the 32 of a wave. S^T = K Q^T puts a row in a lane (column c of the
// accumulator) and tokens 4g..4g+3 of each 16 in lane group g, which is just what the second product wants of its
// operand P^T, so the weights never move between lanes: O^T = V^T P^T sums over k in any order as long as both
// operands agree, and lane group g holds its own 4 + 4 tokens' values. The order of the head's dimension is free too: a
// lane loads head_dim / 16 consecutive codes of each of its tokens (a token's 16 lanes a whole line), turns them over
// in registers, and ends with head_dim / 4 consecutive outputs of its row.
template <int D, int NQ, bool F16>
__global__ __launch_bounds__(kThreads, 2) void stream_kernel(const AttnArgs a) {
  constexpr int R = 16 * NQ, VW = D / 64;  // VW: words of a lane's codes of a token
  constexpr int KL = D / 64;               // 16-byte loads of a key row a lane (D = 64: one)
  constexpr int QS = D / 32;               // steps of 32 along the head
  constexpr int DT = D / 16;               // output tiles along the head
  constexpr int C = D / 16;                // 16-byte pieces of a row of codes
  constexpr int ND = D / 64;               // 1 KiB direct loads of 16 rows
  constexpr int kStage = 2 * 32 * D + 256;  // bytes of 32 tokens: keys, values, their scales
  constexpr int S = D == 64 ? 4 : 2;  // what LDS holds for two workgroups (D = 256: one)
  const int head = blockIdx.x % a.hkv;
  const int index = blockIdx.x / a.hkv;
  const Item it = find<R>(a, index);
  if (!it.ok) return;
  uint64_t* const word = a.word + (int64_t)head * a.words + it.row_tile;
  uint64_t seen = 0;
  const bool joins = NQ == 1 && !a.joiners;  // the last workgroup of a tile; 32 rows have the other kernel for it
  if (threadIdx.x == 0 && it.splits > 1 && joins) seen = splitk_peek(word);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int rows = it.count * a.group, r0 = it.tile * R, ctx = it.len - it.count;
  const int last_t = (min(r0 + R, rows) - 1) / a.group, first_t = r0 / a.group;
  // positions any row of the tile sees, and those all of its rows see
  const int visible = a.mask ? it.len : min(it.len, ctx + last_t + 1);
  const int from = it.split * it.chunk * kUnit;  // below len
  const int end = (int)min((int64_t)visible, from + (int64_t)it.chunk * kUnit);
  const int clear = min(end, ctx + (a.mask ? 0 : first_t + 1));

  u32x4 q[NQ][QS];
  int row_t[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = r0 + 16 * n + c, t = min(r, rows - 1) / a.group, h = min(r, rows - 1) - t * a.group;
    row_t[n] = t;
    const uint16_t* p = static_cast<const uint16_t*>(a.q) + (it.q0 + t) * a.q_token + (head * a.group + h) * a.q_head;
#pragma unroll
    for (int s = 0; s < QS; ++s)  // the order of a key lane's codes: 32 (D = 64: 16) at a time
      q[n][s] = D == 64 ? ld16(p + 16 * g + 8 * s) : ld16(p + 128 * (s / 4) + 32 * g + 8 * (s % 4));
  }

  // A wave's own ring of S stages in LDS. Codes go there straight from memory (no registers, so several steps are on
  // their way at once), a row's pieces by consecutive lanes, so that one line serves eight of them; an operand wants 16
  // rows in consecutive lanes, and loaded in that order into registers each of a wave's 64 lanes asked for a line of its
  // own. Piece u of key row r lies at place u ^ (r * C / 16), and value row t at row t ^ (t / 4 % 4), which puts what the
  // lanes of one read take on different banks.
  __shared__ __align__(1024) uint8_t ring[kWaves][S][kStage];
  uint32_t from_k[ND], from_v[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    const int row = (64 * i + lane) / C, place = (64 * i + lane) % C;
    from_k[i] = row * D + (place ^ (row * C / 16)) * 16;
    from_v[i] = (row ^ ((row >> 2) & 3)) * D + place * 16;
  }
  uint32_t at_k[KL], at_v[4];
#pragma unroll
  for (int i = 0; i < KL; ++i) at_k[i] = c * D + (((D == 64 ? g : 8 * (i / 2) + 2 * g + i % 2) ^ (c * C / 16)) * 16);
#pragma unroll
  for (int j = 0; j < 4; ++j) at_v[j] = 32 * D + (4 * g + (j ^ g)) * D + c * (D / 16);

  struct Pages {
    int id[2];  // of positions p.. and p + 16..
  };
  const_i32* const table = row_of(a.table, it.b * a.table_row);
  // positions are multiples of 16 below 2^28, so the quotient is exact
  auto page_of = [&](int pos) { return (int)__umulhi((uint32_t)pos >> 3, a.page_magic); };
  auto look = [&](int p) {
    Pages x{{-1, -1}};
    if (p < end) {
      x.id[0] = table[page_of(p)];
      x.id[1] = a.wide ? x.id[0] : table[min(page_of(p + 16), a.table_cols - 1)];
    }
    return x;
  };
  auto is_page = [&](int id) { return (uint32_t)id < (uint32_t)a.pages; };
  const int64_t head_codes = (int64_t)head * a.page * D, head_scales = (int64_t)head * a.page * 4;
  const uint64_t kc = (uint64_t)(a.kc + head_codes), vc = (uint64_t)(a.vc + head_codes);
  const uint64_t ks = (uint64_t)a.ks + head_scales, vs = (uint64_t)a.vs + head_scales;
  const uint32_t lds = uniform(lds_addr(&ring[wave][0][0]));
  // Stage `slot` for the 32 tokens from p: always kLoads loads; what is no token's reads as zeros.
  constexpr int kLoads = 4 * ND + 4;
  auto issue = [&](int slot, int p, const Pages& x) {
    const uint32_t to = lds + slot * kStage;
    auto block = [&](int h, uint64_t codes, uint64_t scales, bool real) {
      auto words = [&](uint64_t base, uint32_t bytes) {
        return i32x4{(int)(uint32_t)base, (int)(uint32_t)(base >> 32), real ? (int)bytes : 0, 0x00020000};
      };
      const i32x4 k = words(kc + codes, 16 * D), v = words(vc + codes, 16 * D);
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        lds_dma16(k, to + 16 * D * h + 1024 * i, from_k[i]);
        lds_dma16(v, to + 32 * D + 16 * D * h + 1024 * i, from_v[i]);
      }
      if (lane < 16) {
        lds_dma4(words(ks + scales, 64), to + 64 * D + 64 * h, 4 * lane);
        lds_dma4(words(vs + scales, 64), to + 64 * D + 128 + 64 * h, 4 * lane);
      }
    };
    const bool real = is_page(x.id[0]);
    const uint32_t page = real ? x.id[0] : 0;
    const int off = p - page_of(p) * a.page;
    const uint64_t codes = (uint64_t)page * (uint32_t)a.code_page + (uint32_t)(off * D);
    const uint64_t scales = (uint64_t)page * (uint32_t)a.scale_page + (uint32_t)(off * 4);
    block(0, codes, scales, real);
    if (a.wide) {  // pages of whole 32 tokens
      block(1, codes + 16 * D, scales + 64, real);
    } else {
      const bool real1 = is_page(x.id[1]);
      const uint32_t page1 = real1 ? x.id[1] : 0;
      const int off1 = p + 16 - page_of(p + 16) * a.page;
      block(1, (uint64_t)page1 * (uint32_t)a.code_page + (uint32_t)(off1 * D),
            (uint64_t)page1 * (uint32_t)a.scale_page + (uint32_t)(off1 * 4), real1);
    }
  };
  struct Values {
    uint32_t v[8][VW];
    f32x4 s[2];
  };
  auto read_values = [&](const uint8_t* stage) {
    Values t;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint8_t* w = stage + at_v[j] + 16 * D * h;
        if constexpr (VW == 1) {
          t.v[4 * h + j][0] = *reinterpret_cast<const uint32_t*>(w);
        } else if constexpr (VW == 2) {
          const u32x2 y = *reinterpret_cast<const u32x2*>(w);
          t.v[4 * h + j][0] = y[0];
          t.v[4 * h + j][1] = y[1];
        } else {
          const u32x4 y = *reinterpret_cast<const u32x4*>(w);
#pragma unroll
          for (int i = 0; i < 4; ++i) t.v[4 * h + j][i] = y[i];
        }
      }
      t.s[h] = *reinterpret_cast<const f32x4*>(stage + 64 * D + 128 + 64 * h + 16 * g);
    }
    return t;
  };

  f32x4 o[NQ][DT];
  float m[NQ], l[NQ], limit[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = l[n] = 0.0f;
    limit[n] = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < DT; ++i) o[n][i] = f32x4{0, 0, 0, 0};
  }

  // One step of 32 tokens: scores as exponents; then weights and their sum with the values.
  f32x4 x[NQ][2];
  uint32_t sees[NQ] = {};
  auto first = [&](const uint8_t* stage, bool edge) {
    f32x4 scale[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) x[n][h] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(stage + at_k[i] + 16 * D * h);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const u32x4 k = {two<F16, false>(w[2 * e]), two<F16, true>(w[2 * e]), two<F16, false>(w[2 * e + 1]), two<F16, true>(w[2 * e + 1])};
#pragma unroll
          for (int n = 0; n < NQ; ++n) x[n][h] = mfma32<F16>(k, q[n][2 * i + e], x[n][h]);
        }
      }
      scale[h] = *reinterpret_cast<const f32x4*>(stage + 64 * D + 64 * h + 16 * g) * a.scale_log2;
    }
    return relate<NQ>(x, scale, edge, sees, m, limit);
  };
  auto second = [&](Values& t, bool edge) {
    u32x4 w_hi[NQ], w_lo[NQ];
    weigh<NQ>(x, t.s, edge, sees, l, w_hi, w_lo);
#pragma unroll
    for (int w = 0; w < VW; ++w) {  // a word holds 4 dimensions of a token; an operand wants one, of 8 tokens
      u32x2 lo[4], hi[4];
      turn_over(t.v[0][w], t.v[1][w], t.v[2][w], t.v[3][w], lo);
      turn_over(t.v[4][w], t.v[5][w], t.v[6][w], t.v[7][w], hi);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const u32x4 v = {lo[e][0], lo[e][1], hi[e][0], hi[e][1]};
          o[n][4 * w + e] = mfma32<false>(v, w_hi[n], o[n][4 * w + e]);
          o[n][4 * w + e] = mfma32<false>(v, w_lo[n], o[n][4 * w + e]);
        }
    }
  };

  // Steps that every row sees whole. Where a row lifts its reference the loop is left for that and entered again: with
  // the sums touched by products alone inside it, they stay where the matrix unit has them.
  int p = from + 32 * wave, slot = 0;
  Pages at[S + 1];
#pragma unroll
  for (int i = 0; i <= S; ++i) at[i] = look(p + i * kUnit);
#pragma unroll
  for (int i = 0; i < S; ++i) issue(i, p + i * kUnit, at[i]);
  auto plain = [&] { return p + 32 <= clear && is_page(at[0].id[0]) && is_page(at[0].id[1]); };
  // the oldest stage has arrived; loads after it stay in flight
  auto arrive = [&] { asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * kLoads) : "memory"); };
  auto move = [&] {  // its reads are over: the stage takes the tokens S steps ahead
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    issue(slot, p + S * kUnit, at[S]);
    slot = slot + 1 == S ? 0 : slot + 1;
    p += kUnit;
#pragma unroll
    for (int i = 0; i < S; ++i) at[i] = at[i + 1];
    at[S] = look(p + S * kUnit);
  };
  while (plain()) {
    do {
      arrive();
      const uint8_t* stage = ring[wave][slot];
      if (first(stage, false)) break;
      Values t = read_values(stage);
      second(t, false);
      move();
    } while (plain());
    if (!plain()) break;
    lift<NQ, DT>(x, m, limit, l, o);
    Values t = read_values(ring[wave][slot]);
    second(t, false);
    move();
  }
  // And those at an edge, one or two at most where pages are in order: some row does not see some of their positions, or
  // they hold no token. Nothing in them may reach a row that does not see them, NaN included: scores are replaced, and
  // because a weight of zero times a NaN would still be one, a value's NaN code moves into its token's scale, which only
  // rows that see it multiply by.
  while (p < end) {
    arrive();
    const uint8_t* stage = ring[wave][slot];
    const uint32_t held = held_by<8, 16>(4 * g, end - p, is_page(at[0].id[0]), is_page(at[0].id[1]));
#pragma unroll
    for (int n = 0; n < NQ; ++n) sees[n] = seen_by<8, 16>(a, held, p + 4 * g - ctx, row_t[n], it.q0);
    if (first(stage, true)) lift<NQ, DT>(x, m, limit, l, o);
    Values t = read_values(stage);
    clean<8, 16, VW>(t.v, t.s, held);
    second(t, true);
    move();
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing is on its way into the ring any more
  __syncthreads();

  // The waves' sums meet in LDS, in wave order; rows padded by 4 floats, which spreads 8 rows over the banks
  __shared__ float wave_m[kWaves][R], wave_l[kWaves][R];
  static_assert(sizeof(ring) >= sizeof(float) * kWaves * 16 * (D + 4), "the waves' sums fit the ring");
  auto& sum = *reinterpret_cast<float(*)[kWaves][16][D + 4]>(&ring[0][0][0]);
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] = across(l[n], [](float u, float v) { return u + v; });
    if (limit[n] != kRise) m[n] = kNone;
    if (g == 0) wave_m[wave][16 * n + c] = m[n], wave_l[wave][16 * n + c] = l[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float top = wave_m[0][16 * n + c];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, wave_m[w][16 * n + c]);
    const float by = m[n] == top ? 1.0f : __builtin_amdgcn_exp2f(m[n] - top);
    if (n) __syncthreads();
#pragma unroll
    for (int rr = 0; rr < 4; ++rr)
#pragma unroll
      for (int i = 0; i < DT; i += 4) {
        float* to = &sum[wave][c][DT * (4 * g + rr) + i];
        *reinterpret_cast<f32x4*>(to) = f32x4{o[n][i][rr], o[n][i + 1][rr], o[n][i + 2][rr], o[n][i + 3][rr]} * by;
      }
    __syncthreads();
    const int r = threadIdx.x >> 4, d = (threadIdx.x & 15) * DT, row = r0 + 16 * n + r;
    float best = wave_m[0][16 * n + r], total = 0.0f, v[DT];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) best = fmaxf(best, wave_m[w][16 * n + r]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mw = wave_m[w][16 * n + r];
      total += wave_l[w][16 * n + r] * (mw == best ? 1.0f : __builtin_amdgcn_exp2f(mw - best));
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) v[i] = sum[0][r][d + i];
#pragma unroll
    for (int w = 1; w < kWaves; ++w)
#pragma unroll
      for (int i = 0; i < DT; ++i) v[i] += sum[w][r][d + i];
    if (it.splits > 1) {
      if (row < rows) {  // past the XCD's own cache: the workgroup that joins may sit on another
        const rsrc_t to = slot_at<D, R>(a, head, it.slot + it.split * it.tiles);
#pragma unroll
        for (int i = 0; i < DT; i += 4)
          store_partial4(to, (16 * n + r) * D + d + i, f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]});
        if (d == 0) store_partial4(to, R * D + 4 * (16 * n + r), f32x4{best, total, 0, 0});
      }
    } else if (row < rows) {
      finish<DT, F16>(a, it, head, row, d, best, total, v);
    }
  }
  if constexpr (NQ == 1) {
    if (it.splits == 1 || !joins) return;
    __shared__ unsigned arrived;
    if (splitk_arrive(word, seen, it.splits, &arrived)) join<D, R, F16>(a, it, head, 0, min(R, rows - r0), r0, &sum[0][0][0]);
  }
}

template <bool F16>
__device__ __forceinline__ f32x16 mfma16(const u32x4& a, const u32x4& b, const f32x16& c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Many rows: bound by the vector unit's issue beside the matrix unit's time. A step of 32 rows and tokens is 16 products
// (512 cycles) and about 195 vector instructions, 64 of them conversions; counters show the vector unit's issue two thirds
// and the matrix unit 37 % of the time busy, two waves on a SIMD. 2048 tokens of each of two prompts over 8192, 8 kv heads
// of 128, group 4: 577 to 606 us by the card, 815 to 856 TFLOP/s; without the raised priority of the second products 30 us more. fp16
// queries, whose weights are two bf16 (24 products): 735 us.
//
// The W waves of a workgroup take 32 rows each and share a ring of S stages of 64 tokens' codes in LDS, which
// come straight from memory, 16 tokens a load. One barrier a stage: a wave waits for its own loads, the barrier for the
// others', and behind it the stage before is free for the loads S - 1 stages ahead.
//
// 32 x 32 x 16 products: the matrix unit is busy for 32 cycles with one, in which the SIMD issues other instructions all
// the same; beside the 16 cycles of a 16 x 16 x 32 product it hardly does (measured: a product and three fused
// multiply-adds take 26 cycles there, one of 32 x 32 and four of them 31). Conversions and exponentials are as much work
// here as the products, so that is worth more than the smaller tiles' fit. Row c of the lane's half of the wave, hf, and
// tokens 8b + 4hf + 0..3 of each 32 in the four accumulator groups b: again what the second product wants.
template <int D, int W, bool F16>
__global__ __launch_bounds__(64 * W, D > 128 ? 1 : 2) void tile_kernel(const AttnArgs a) {
  constexpr int R = 32 * W, QS = D / 16, DT = D / 32, C = D / 16, KL = D / 32, ND = D / 64;
  constexpr bool kTwo = F16;  // bf16 pieces of a weight
  constexpr int kStep = 64, S = W == 2 ? 2 : 3, kStage = 2 * kStep * D + 8 * kStep, kBlocks = 4 / W;  // blocks of 16 a wave loads
  const int head = blockIdx.x % a.hkv, index = blockIdx.x / a.hkv;
  const Item it = find<R>(a, index);
  if (!it.ok) return;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), c = lane & 31, hf = lane >> 5;
  const int rows = it.count * a.group, r0 = it.tile * R, rw = r0 + 32 * wave, ctx = it.len - it.count;
  const int last_t = (min(r0 + R, rows) - 1) / a.group;
  const int visible = a.mask ? it.len : min(it.len, ctx + last_t + 1);
  const int from = it.split * it.chunk * kUnit;  // below len
  const int end = (int)min((int64_t)visible, from + (int64_t)it.chunk * kUnit);
  // the wave's own rows: positions some of them see, and those all of them see
  const int own = rw >= rows ? 0 : a.mask ? end : min(end, ctx + (min(rw + 32, rows) - 1) / a.group + 1);
  const int clear = min(end, ctx + (a.mask ? 0 : rw / a.group + 1));

  u32x4 q[QS];
  const int row_t = min(rw + c, rows - 1) / a.group;
  {
    const int h = min(rw + c, rows - 1) - row_t * a.group;
    const uint16_t* p = static_cast<const uint16_t*>(a.q) + (it.q0 + row_t) * a.q_token + (head * a.group + h) * a.q_head + (D / 2) * hf;
#pragma unroll
    for (int s = 0; s < QS; ++s) q[s] = ld16(p + 8 * s);
  }

  // [keys of 64 tokens][values][key scales][value scales]. Piece u of key row r lies at u ^ (r * C / 16), value row t at
  // t ^ (t / 4 % 2): what the lanes of one read take is on different banks.
  __shared__ __align__(1024) uint8_t ring[S][kStage];
  __shared__ __align__(16) int here[S][4];  // whether 16 tokens' page is one
  uint32_t from_k[ND], from_v[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    const int row = (64 * i + lane) / C, place = (64 * i + lane) % C;
    from_k[i] = row * D + (place ^ (row * C / 16)) * 16;
    from_v[i] = (row ^ ((row >> 2) & 1)) * D + place * 16;
  }
  uint32_t at_k[KL], at_v[4];
#pragma unroll
  for (int i = 0; i < KL; ++i) at_k[i] = c * D + (((C / 2) * hf + i) ^ ((c & 15) * C / 16)) * 16;
#pragma unroll
  for (int j = 0; j < 4; ++j) at_v[j] = kStep * D + (4 * hf + (j ^ hf)) * D + c * (D / 32);

  const_i32* const table = row_of(a.table, it.b * a.table_row);
  auto page_of = [&](int pos) { return (int)__umulhi((uint32_t)pos >> 3, a.page_magic); };
  struct Pages {
    int id[kBlocks];
  };
  auto look = [&](int p) {
    Pages x;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const int pos = p + 16 * (wave + W * b);
      x.id[b] = pos < end ? table[min(page_of(pos), a.table_cols - 1)] : -1;
    }
    return x;
  };
  const uint64_t kc = (uint64_t)(a.kc + (int64_t)head * a.page * D), vc = (uint64_t)(a.vc + (int64_t)head * a.page * D);
  const uint64_t ks = (uint64_t)(a.ks + (int64_t)head * a.page), vs = (uint64_t)(a.vs + (int64_t)head * a.page);
  const uint32_t lds = uniform(lds_addr(&ring[0][0]));
  constexpr int kLoads = kBlocks * (2 * ND + 2);
  auto issue = [&](int slot, int p, const Pages& x) {  // always kLoads loads; what is no token's reads as zeros
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const int block = wave + W * b, pos = p + 16 * block;
      const bool real = (uint32_t)x.id[b] < (uint32_t)a.pages;
      const uint32_t page = real ? x.id[b] : 0, off = pos - page_of(pos) * a.page;
      const uint64_t codes = (uint64_t)page * (uint32_t)a.code_page + off * D;
      const uint64_t scales = (uint64_t)page * (uint32_t)a.scale_page + off * 4;
      auto words = [&](uint64_t base, uint32_t bytes) {
        return i32x4{(int)(uint32_t)base, (int)(uint32_t)(base >> 32), real ? (int)bytes : 0, 0x00020000};
      };
      const i32x4 k = words(kc + codes, 16 * D), v = words(vc + codes, 16 * D);
      const uint32_t to = lds + slot * kStage + 16 * D * block;
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        lds_dma16(k, to + 1024 * i, from_k[i]);
        lds_dma16(v, to + kStep * D + 1024 * i, from_v[i]);
      }
      const uint32_t to_s = lds + slot * kStage + 2 * kStep * D + 64 * block;
      if (lane < 16) {
        lds_dma4(words(ks + scales, 64), to_s, 4 * lane);
        lds_dma4(words(vs + scales, 64), to_s + 4 * kStep, 4 * lane);
      }
      if (lane == 0) here[slot][block] = real;
    }
  };

  f32x16 o[DT], x;
  float m, l, limit;
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.0f;
  m = l = 0.0f;
  limit = -__builtin_inff();

  auto across = [](float v, auto f) {  // over the two halves that share a row
    const uint32_t u = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return f(__uint_as_float(s[0]), __uint_as_float(s[1]));
  };
  // 32 tokens from p, at `stage` (already past the tokens before them)
  constexpr int VB = D / 32, VN = VB > 4 ? VB / 4 : 1;  // codes of a token a lane, and words
  struct Read {  // what a step takes from LDS
    u32x4 k[KL];
    f32x4 ks[4], vs[4];
    uint32_t v[4][4][VN];  // [8 tokens][token 4hf + j of them]
  };
  auto read = [&](const uint8_t* codes, const uint8_t* scale) {
    Read t;
#pragma unroll
    for (int i = 0; i < KL; ++i) t.k[i] = *reinterpret_cast<const u32x4*>(codes + at_k[i]);
#pragma unroll
    for (int b = 0; b < 4; ++b) t.ks[b] = *reinterpret_cast<const f32x4*>(scale + 32 * b + 16 * hf);
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      t.vs[b] = *reinterpret_cast<const f32x4*>(scale + 4 * kStep + 32 * b + 16 * hf);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint8_t* w = codes + at_v[j] + 8 * b * D;
        if constexpr (VB == 2) {
          t.v[b][j][0] = *reinterpret_cast<const uint16_t*>(w);
        } else if constexpr (VB == 4) {
          t.v[b][j][0] = *reinterpret_cast<const uint32_t*>(w);
        } else {
          const u32x2 y = *reinterpret_cast<const u32x2*>(w);
          t.v[b][j][0] = y[0];
          t.v[b][j][1] = y[1];
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // all of it on its way before the first use waits
    return t;
  };
  uint32_t sees = 0;
  auto scores = [&](const Read& t, bool edge) {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const u32x4 w = t.k[i];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const u32x4 k = {two<F16, false>(w[2 * e]), two<F16, true>(w[2 * e]), two<F16, false>(w[2 * e + 1]), two<F16, true>(w[2 * e + 1])};
        x = mfma16<F16>(k, q[2 * i + e], x);
      }
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const f32x4 s = t.ks[b] * a.scale_log2;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * b + i] = fmaf(x[4 * b + i], s[i], -m);
    }
    if (edge) {
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = masked(x[r], sees, r);
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, x[r]);
    return __ballot(top > limit) != 0;
  };
  auto rise = [&] {
    float top = x[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
    top = across(top, [](float u, float v) { return fmaxf(u, v); });
    const bool first = limit != kRise;
    if (top > (first ? -__builtin_inff() : 0.0f)) {
      top += kHead;
      limit = kRise;
    } else {
      top = 0.0f;
    }
    const float by = first ? 1.0f : __builtin_amdgcn_exp2f(-top);
    m += top;
    l *= by;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] *= by;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] -= top;
  };
  auto sums = [&](Read& t, bool edge) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {  // 16 tokens: 16kk + 8b + 4hf + 0..3
      auto& v = reinterpret_cast<uint32_t(&)[2][4][VN]>(t.v[2 * kk]);
      const f32x4 s[2] = {t.vs[2 * kk], t.vs[2 * kk + 1]};
      u32x4 pt, rest;
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = __builtin_amdgcn_exp2f(x[8 * kk + i]);
        l += e;
        w[i] = e * s[i / 4][i % 4];
      }
      if (edge) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = masked_weight(w[i], sees, 8 * kk + i);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t left;
        pt[i] = pieces(w[2 * i], w[2 * i + 1], left);
        if constexpr (kTwo) rest[i] = left;
      }
      if (kk == 0) __builtin_amdgcn_s_setprio(1);
      constexpr int E = VB == 2 ? 2 : 4;  // dimensions of a word
#pragma unroll
      for (int y = 0; y < VN; ++y) {
        u32x2 y4[2][E];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if constexpr (E == 2)
            turn_over2(v[b][0][0], v[b][1][0], v[b][2][0], v[b][3][0], y4[b]);
          else
            turn_over(v[b][0][y], v[b][1][y], v[b][2][y], v[b][3][y], y4[b]);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const u32x4 z = {y4[0][e][0], y4[0][e][1], y4[1][e][0], y4[1][e][1]};
          o[E * y + e] = mfma16<false>(z, pt, o[E * y + e]);
          if constexpr (kTwo) o[E * y + e] = mfma16<false>(z, rest, o[E * y + e]);
        }
      }
    }
  };

  int p = from, slot = 0;
  Pages next;
#pragma unroll
  for (int i = 0; i < S - 1; ++i) issue(i, from + i * kStep, look(from + i * kStep));
  next = look(from + (S - 1) * kStep);
  // Steps of 32 tokens. As in the other kernel the inner loop is left where a row lifts its reference, and for an edge.
  int half = 0;
  i32x4 pages;
  while (p < end) {
    bool lifts = false;
    const uint8_t *codes = nullptr, *scale = nullptr;
    do {
      if (half == 0) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * kLoads) : "memory");
        stage_barrier();
        issue(slot == 0 ? S - 1 : slot - 1, p + (S - 1) * kStep, next);  // into the stage before this one
        pages = *reinterpret_cast<const i32x4*>(here[slot]);
      }
      codes = ring[slot] + 32 * D * half;
      scale = ring[slot] + 2 * kStep * D + 128 * half;
      if (p < own) {
        if (p + 32 > clear || !uniform(half ? pages[2] & pages[3] : pages[0] & pages[1])) break;
        Read t = read(codes, scale);
        __builtin_amdgcn_s_setprio(0);
        lifts = scores(t, false);
        if (half == 0) next = look(p + S * kStep);
        if (lifts) break;
        sums(t, false);
      } else if (half == 0) {
        next = look(p + S * kStep);
      }
      p += 32;
      slot = half == 0 ? slot : slot + 1 == S ? 0 : slot + 1;
      half ^= 1;
    } while (p < end);
    if (p >= end) break;
    Read t = read(codes, scale);
    const bool edge = !lifts;
    if (edge) {
      const uint32_t held = held_by<16, 8>(4 * hf, end - p, pages[2 * half] != 0, pages[2 * half + 1] != 0);
      sees = seen_by<16, 8>(a, held, p + 4 * hf - ctx, row_t, it.q0);
      clean<16, 32, VN>(&t.v[0][0], t.vs, held);
      lifts = scores(t, true);
      if (half == 0) next = look(p + S * kStep);
    }
    if (lifts) rise();
    sums(t, edge);
    p += 32;
    slot = half == 0 ? slot : slot + 1 == S ? 0 : slot + 1;
    half ^= 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing is on its way into the ring any more

  const rsrc_t to = slot_at<D, R>(a, head, it.slot + it.split * it.tiles);
  l = across(l, [](float u, float v) { return u + v; });
  if (limit != kRise) m = kNone;
  const int row = rw + c;
  if (row < rows) {  // DT consecutive dimensions of it for each of the accumulators' 16 rows
#pragma unroll
    for (int r = 0; r < 16; r += (DT < 4 ? 2 : 1)) {
      const int d = DT * (8 * (r / 4) + 4 * hf + r % 4);
      constexpr int N = DT < 4 ? 4 : DT;
      float v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = o[i % DT][r + i / DT];
      if (it.splits > 1) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
          store_partial4(to, (row - r0) * D + d + i, f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]});
      } else {
        finish<N, F16>(a, it, head, row, d, m, l, v);
      }
    }
    if (it.splits > 1 && hf == 0) store_partial4(to, R * D + 4 * (row - r0), f32x4{m, l, 0, 0});
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Workgroups a call is cut into: as many as run at once (two a CU, four of two waves, half of that with heads of 256) where
// the tiles of rows are at most half of those. 16 sequences of 64 rows over 8 k tokens take 94 us in 512 workgroups of two
// waves and 76 in 1024, one row over 16 k with heads of 256 36 us in 512 and 27 in 256. Where tiles are more, half as many
// again beside them let short and long ones even out: 64 sequences and 8 kv heads took 142 us with 512, 127 with 768, 136
// with 1024 (more partial results), and 144 with 2048.
//
// Joining: the last workgroup of a tile does it in the same launch where there is little to join, else a kernel of its
// own with up to a workgroup for four rows. A launch costs 2 us more (one row of each of 16 sequences of 1000 tokens and
// 8 kv heads of 4: 14.0 us joined by the last, 16.4 apart), and the last workgroup alone is bound by how long its loads
// take (one sequence of 16000: 23.8 and 20.8; of 2000 with 16 rows of one kv head 14.3 and 11.8, of 16000 61.8 and 24.1;
// 64 rows of each of 8 kv heads 165 and 37).
constexpr int kCus = 256, kJoinGroups = 2048, kApart = 240;
constexpr int kMostSplits = 254;  // an arrival word counts to 255

struct AttnPlan {
  int rows;     // a workgroup's
  int64_t slots, target, tiles;
  int64_t cap, held;  // items a kv head can have, and partial results
  int64_t joiners;
  size_t words, bytes;
};

bool plan_attention(int64_t total, int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t capacity, AttnPlan* p) {
  const int64_t group = hq / hkv, rows = (total * group + batch - 1) / batch;  // of a sequence, on the mean
  const int64_t units = (capacity + kUnit - 1) / kUnit;
  // Tiles of many rows where there is much to do, else more workgroups of fewer: a step of 128 tokens for 128 rows is
  // the unit, a tile of 64 rows half of one, over as many tokens as the table has room for. In us with tiles of 128 (64) and
  // with 32, contexts ragged between half and all of what is named:
  //   heads of 128, 128 rows: 2048 units (32 sequences of 1000, 8 kv heads) 50 and 42, (8 of 4000) 49 and 43; 4096 (16 of
  //     4000) 63 and 66; 4032 (32 of 8000, 2 kv heads) 62 and 84; 8000 (8 of 16000) 95 and 118; 64512 (32 of 8000, 32) 566 and 676;
  //   trees of up to 33 tokens, group 4 (101 rows): 12, 14, 16 and 20 over 2000 (up to 2560) 49 49 52 60 and 42 43 47 50; over
  //     16384 4 (4128) 68 and 59, 6 84 and 85, 12, 14, 15, 16 and 17 142 159 173 173 193 and 158 172 207 233 231;
  //   64 rows: 1024 (8 of 4000) 43 and 30, 4000 (8 of 16000) 71 and 69, 8000 (16) 118 and 126;
  //   heads of 64, 128 rows: 2048 (8 of 4000) 34 and 35, 8000 (8 of 16000) 76 and 90;
  //   heads of 256 (16 rows beside 128): 512 (8 of 1000) 48 and 35, 1024 (4 of 4000) 60 and 56, 2048 (8) 80 and 89.
  // Where a sequence's rows leave much of their last tile empty more would be better (132 of them 94 and 72 at 8192 units).
  // 32 rows of 16 sequences in tiles of 64 64.8, of 32 52.9, of 16 56.9; 4 rows of one in 32 50.5, of 16 44.3.
  const int64_t half_tiles = batch * hkv * units * (rows > 64 ? 2 * ((rows + 127) / 128) : 1);
  const bool many = rows > 32 && half_tiles >= (d == 256 ? 2000 : 8000);
  p->rows = many ? rows > 64 ? 128 : 64 : rows > 16 && d < 256 ? 32 : 16;
  const int64_t slots = kCus * (p->rows == 64 ? 4 : 2) / (d == 256 ? 2 : 1), target = slots * 3 / 2;
  p->target = (target + hkv - 1) / hkv < kMostSplits ? (target + hkv - 1) / hkv : kMostSplits;
  p->slots = (slots + hkv - 1) / hkv < kMostSplits ? (slots + hkv - 1) / hkv : kMostSplits;
  p->tiles = total * group / p->rows + (batch < total ? batch : total);
  // With chunk > work / target, the sum over sequences of tiles * units / chunk stays below the target. Rounded up to whole
  // splits that is a tile each more; of the sequences of several, at most twice as many, which are the partial results.
  p->cap = p->tiles + (units > 1 ? p->target : 0);
  p->held = p->cap < 2 * p->target ? p->cap : 2 * p->target;
  const int64_t tiles = batch * ((rows + p->rows - 1) / p->rows);  // at the mean; with the most splits a tile can have
  const int64_t splits = units < p->slots / tiles ? units : p->slots / tiles;
  p->joiners = 0;
  if (units > 1 && (p->rows > 16 || splits * (rows + 8) >= kApart)) {
    const int64_t most = p->rows / 4, each = kJoinGroups / (p->tiles * hkv);
    p->joiners = each < 1 ? 1 : each > most ? most : each;
  }
  if (p->cap * hkv > 0xFFFFFF) return false;  // a launch has fewer than 2^32 threads
  p->words = ((size_t)(p->tiles * hkv) * 8 + 15) / 16 * 16;
  p->bytes = units > 1 ? p->words + (size_t)(p->held * hkv * p->rows * (d + 4)) * sizeof(float) : 0;
  return true;
}

template <int D, bool F16>
int launch_attention(const AttnArgs& a, const AttnPlan& p, hipStream_t stream) {
  const auto go = [&](auto kernel, auto rows, int threads) {
    constexpr int R = decltype(rows)::value;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(p.cap * a.hkv)), dim3(threads), 0, stream, a);
    AKLR_LAUNCH_CHECK();
    if (!a.joiners) return AKLR_OK;
    hipLaunchKernelGGL((join_kernel<D, R, F16>), dim3((unsigned)(p.tiles * a.joiners * a.hkv)), dim3(kThreads), 0, stream, a);
    AKLR_LAUNCH_CHECK();
    return AKLR_OK;
  };
  if (p.rows == 128) return go(tile_kernel<D, 4, F16>, IC<128>{}, 256);
  if (p.rows == 64) return go(tile_kernel<D, 2, F16>, IC<64>{}, 128);
  if constexpr (D < 256)
    if (p.rows == 32) return go(stream_kernel<D, 2, F16>, IC<32>{}, kThreads);
  return go(stream_kernel<D, 1, F16>, IC<16>{}, kThreads);
}

bool attention_shape_ok(int64_t total, int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t capacity) {
  return total >= 0 && batch >= 0 && batch <= 65536 && hkv >= 1 && hkv <= 1024 && hq >= hkv && hq % hkv == 0 &&
         hq <= 65536 && total * (hq / hkv) <= 0x3FFFFFFF && (d == 64 || d == 128 || d == 256) && capacity >= 0 &&
         capacity <= (1 << 28);
}

}  // namespace aklr

using namespace aklr;

extern "C" size_t aklr_tree_attention_fp8_workspace_bytes(int64_t total_q, int64_t batch, int64_t q_heads,
                                                          int64_t kv_heads, int64_t head_dim, int64_t capacity) {
  AttnPlan p;
  if (!attention_shape_ok(total_q, batch, q_heads, kv_heads, head_dim, capacity) || total_q == 0 || batch == 0 ||
      !plan_attention(total_q, batch, q_heads, kv_heads, head_dim, capacity, &p))
    return 0;
  return p.bytes;
}

extern "C" int aklr_tree_attention_fp8_rows(int64_t total_q, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                            int64_t head_dim, int64_t capacity, int* joiners) {
  AttnPlan p;
  if (!attention_shape_ok(total_q, batch, q_heads, kv_heads, head_dim, capacity) || total_q == 0 || batch == 0 ||
      !plan_attention(total_q, batch, q_heads, kv_heads, head_dim, capacity, &p))
    return 0;
  if (joiners) *joiners = (int)p.joiners;
  return p.rows;
}

extern "C" int aklr_tree_attention_fp8(const void* q, int64_t q_token, int64_t q_head, const void* k_codes,
                                       const void* v_codes, const float* k_scales, const float* v_scales,
                                       int64_t code_page, int64_t scale_page,
                                       const int32_t* block_table, int64_t table_stride, int64_t table_cols,
                                       const int32_t* seq_lens, const int32_t* starts, const void* mask,
                                       int64_t mask_stride, int64_t mask_cols, void* out, float* lse, int64_t total_q,
                                       int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                       int64_t pages, int64_t page_size, float softmax_scale, int dtype, void* workspace,
                                       size_t workspace_bytes, hipStream_t stream) {
  if (dtype != AKLR_OUT_BF16 && dtype != AKLR_OUT_F16) return AKLR_ERR_UNSUPPORTED;
  if (page_size < 16 || page_size > 1024 || page_size % 16 != 0 || pages < 1 || pages * page_size > 0x7FFFFFFF ||
      table_cols < 0 || table_cols > (1 << 24) || table_stride < table_cols ||
      !attention_shape_ok(total_q, batch, q_heads, kv_heads, head_dim, table_cols * page_size))
    return AKLR_ERR_INVALID_ARGUMENT;
  if (total_q == 0 || batch == 0) return AKLR_OK;
  if (!q || !k_codes || !v_codes || !k_scales || !v_scales || !seq_lens || !starts || !out || (table_cols && !block_table))
    return AKLR_ERR_INVALID_ARGUMENT;
  if (!aklr_aligned16(q) || !aklr_aligned16(k_codes) || !aklr_aligned16(v_codes) || !aklr_aligned16(k_scales) ||
      !aklr_aligned16(v_scales) || !aklr_aligned16(out) || q_token % 8 != 0 || q_head % 8 != 0)
    return AKLR_ERR_INVALID_ARGUMENT;
  const int64_t page_codes = kv_heads * page_size * head_dim, page_scales = kv_heads * page_size;
  if (code_page < page_codes || scale_page < page_scales || code_page % 16 != 0 || scale_page % 4 != 0 ||
      code_page > 0xFFFFFFFFll || scale_page > 0x3FFFFFFFll)
    return AKLR_ERR_INVALID_ARGUMENT;
  if (mask && (mask_cols < 0 || mask_cols > 0x7FFFFFFF)) return AKLR_ERR_INVALID_ARGUMENT;
  AttnPlan p;
  if (!plan_attention(total_q, batch, q_heads, kv_heads, head_dim, table_cols * page_size, &p))
    return AKLR_ERR_INVALID_ARGUMENT;
  if (p.bytes && (workspace_bytes < p.bytes || !workspace || !aklr_aligned16(workspace))) return AKLR_ERR_WORKSPACE;
  AttnArgs a{};
  a.q = q;
  a.q_token = q_token;
  a.q_head = q_head;
  a.kc = static_cast<const uint8_t*>(k_codes);
  a.vc = static_cast<const uint8_t*>(v_codes);
  a.ks = k_scales;
  a.vs = v_scales;
  a.code_page = code_page;
  a.scale_page = scale_page * 4;
  a.wide = page_size % 32 == 0;
  a.table = block_table;
  a.table_row = table_stride;
  a.lens = seq_lens;
  a.starts = starts;
  a.mask = static_cast<const uint8_t*>(mask);
  a.mask_row = mask_stride;
  a.out = out;
  a.lse = lse;
  a.word = static_cast<uint64_t*>(workspace);
  a.part = p.bytes ? reinterpret_cast<float*>(static_cast<char*>(workspace) + p.words) : nullptr;
  a.page_magic = (uint32_t)(((1ull << 32) + page_size / 8 - 1) / (page_size / 8));
  a.table_cols = (int)table_cols;
  a.mask_cols = (int)mask_cols;
  a.total = (int)total_q;
  a.batch = (int)batch;
  a.hq = (int)q_heads;
  a.hkv = (int)kv_heads;
  a.group = (int)(q_heads / kv_heads);
  a.page = (int)page_size;
  a.pages = (int)pages;
  a.target = (int)p.target;
  a.slots = (int)p.slots;
  a.held = (int)p.held;
  a.words = (int)p.tiles;
  a.joiners = (int)p.joiners;
  a.scale_log2 = softmax_scale * 1.44269504f;
  a.dim = (int)head_dim;
  const auto go = [&](auto d) {
    constexpr int D = decltype(d)::value;
    return dtype == AKLR_OUT_F16 ? launch_attention<D, true>(a, p, stream) : launch_attention<D, false>(a, p, stream);
  };
  return head_dim == 64 ? go(IC<64>{}) : head_dim == 128 ? go(IC<128>{}) : go(IC<256>{});
}

AKLR_SCALAR_FP32_END
