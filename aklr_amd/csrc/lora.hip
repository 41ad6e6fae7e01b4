// Low-rank adapters of many requests beside a projection that all share: out[t] = base[t] + s_a (x[t] A_a^T) B_a^T with
// a = adapters[t], A_a [rank, K], B_a [N, rank]. gfx950 only.
//
// Two launches over tiles of up to 16 * MT tokens of one adapter, so that its weights are read once a tile (what many
// workgroups of the second would convert again is joined by one between them):
//   shrink  v[t, r] = sum_k x[t, k] A[r, k], K split over workgroups (fp32 parts in the workspace) and over a workgroup's
//           four waves, on 16x16x32 products with the adapter's rows as one operand and tokens as the other;
//   expand  the parts added in their order, v in 16-bit pieces (three for bf16, which hold all 24 bits of it; two for fp16,
//           off by 2^-23 of it or 2^-39 of the token's largest), products with B's rows, base added in fp32, one rounding.
// Only the first reads x, so out may lie where x and base do.
// Up to 256 tokens a workgroup finds its tile by itself, from all tokens' adapters; more are put in the adapters' order by a
// launch before. A token's row of a tile changes no result: the products' columns do not meet.
//
// Bound by memory in long prompts, by x, base and out, and in the second product of batches, by B; the first of batches up to
// 256 tokens has 2.5 TB/s of A behind its search for a tile, and a few tokens are two chains of loads (figures at plan_lora).
#include "common.h"
#include "scan.h"

AKLR_SCALAR_FP32_BEGIN

namespace aklr {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kScan = 256;  // tokens that a workgroup looks through by itself
constexpr int kMostAdapters = 4096;  // what the sort counts in LDS

template <bool F16>
__device__ __forceinline__ f32x4 product(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

struct Tile {
  int adapter;  // `adapters`: tokens without one
  int first;    // in `order`
  int count;    // 0: no tile
  int pad;
};

struct LoraArgs {
  const uint16_t *x, *a, *b, *base;
  uint16_t* out;
  int64_t x_row, a_adapter, a_row, b_adapter, b_row, base_row, out_row;  // elements
  const void* ids;
  const float* scales;
  const int32_t* ranks;
  float* part;  // [splits][tokens][rank rounded up to the products' rows]
  uint16_t* joined;  // [pieces][tokens][..], and powers [tokens], of many tokens
  int32_t* powers;
  int32_t* order;
  Tile* tiles;
  int tokens, k, n, rank, adapters, ids64, splits, k_split, n_group, copies, part_row;
};

// A token's adapter, `adapters` where it has none.
__device__ __forceinline__ int adapter_of(const LoraArgs& a, int t) {
  const uint32_t* const p = static_cast<const uint32_t*>(a.ids);
  const uint32_t i = p[(int64_t)t << a.ids64];
  if (a.ids64 && p[2 * (int64_t)t + 1] != 0) return a.adapters;
  return i < (uint32_t)a.adapters ? (int)i : a.adapters;
}

__device__ __forceinline__ int rank_of(const LoraArgs& a, int adapter) {
  if (adapter >= a.adapters) return 0;
  return a.ranks ? min(max(a.ranks[adapter], 0), a.rank) : a.rank;
}

// Tile number `id` from the workspace: its tokens in `rows`, the first repeated behind them. False: there is none.
template <int TM>
__device__ __forceinline__ bool read_tile(const LoraArgs& a, int id, int (&rows)[TM], int& adapter, int& count) {
  const Tile tile = a.tiles[id];
  adapter = tile.adapter;
  count = tile.count;
  if (count == 0) return false;
  if ((int)threadIdx.x < TM) rows[threadIdx.x] = a.order[tile.first + ((int)threadIdx.x < count ? threadIdx.x : 0)];
  __syncthreads();
  return true;
}

// The same with few tokens, by each wave for itself (no wave waits for another): which tokens have a lane's adapter follows
// from ballots over the bits of all tokens' numbers. A tile begins at each token that has a whole number of tiles' tokens of
// its adapter before it, and the tiles are counted in the order of where they begin. `writes`: puts it into the workspace, for
// the second launch.
template <int TM>
__device__ __forceinline__ bool find_tile(const LoraArgs& a, int id, int (&rows)[TM], int& adapter, int& count, bool writes) {
  constexpr int kChunks = kScan / 64;
  const int lane = threadIdx.x & 63, bits = 32 - __builtin_clz(a.adapters), chunks = (a.tokens + 63) / 64;
  const uint64_t below = (1ull << lane) - 1;
  int own[kChunks], before[kChunks];
  uint64_t same[kChunks][kChunks];  // of a token of chunk c: the tokens of chunk d with its adapter
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int t = c * 64 + lane;
    own[c] = t < a.tokens ? adapter_of(a, t) : a.adapters;
#pragma unroll
    for (int d = 0; d <= c; ++d) same[c][d] = __ballot(d * 64 + lane < a.tokens);
  }
#pragma unroll 1
  for (int i = 0; i < bits; ++i) {
    uint64_t b[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (c >= chunks) break;
      b[c] = __ballot(own[c] >> i & 1);
      const uint64_t flip = (uint64_t)(own[c] >> i & 1) - 1;
#pragma unroll
      for (int d = 0; d <= c; ++d) same[c][d] &= b[d] ^ flip;
    }
  }
  int left = id, first = -1;
  adapter = -1;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    before[c] = __popcll(same[c][c] & below);
#pragma unroll
    for (int d = 0; d < c; ++d) before[c] += __popcll(same[c][d]);
    const bool begins = c * 64 + lane < a.tokens && before[c] % TM == 0;
    const uint64_t all = __ballot(begins), chosen = __ballot(begins && __popcll(all & below) == left);
    left -= __popcll(all);
    if (chosen) {
      const int at = __ffsll((unsigned long long)chosen) - 1;
      adapter = __builtin_amdgcn_readlane(own[c], at);
      first = __builtin_amdgcn_readlane(before[c], at);
    }
  }
  if (adapter < 0) {
    if (writes && threadIdx.x == 0) a.tiles[id] = {0, 0, 0, 0};
    return false;
  }
  count = 0;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int at = before[c] - first;
    const bool in = c * 64 + lane < a.tokens && own[c] == adapter && at >= 0 && at < TM;
    count += __popcll(__ballot(in));
    if (in) rows[at] = c * 64 + lane;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if (lane >= count && lane < TM) rows[lane] = rows[0];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if (writes && (int)threadIdx.x < count) a.order[id * TM + threadIdx.x] = rows[threadIdx.x];
  if (writes && threadIdx.x == 0) a.tiles[id] = {adapter, id * TM, count, 0};
  return true;
}

// Tokens in the order of their adapters, those without one last, and the tiles of that order: one workgroup. Within an
// adapter the order is that of arrival; no result depends on it. Consecutive tokens are mostly of one adapter: a wave whose
// tokens all are counts them at once. Up to 8192 tokens are read once.
constexpr int kSort = 1024, kHeld = 8;
__global__ __launch_bounds__(kSort) void sort_kernel(const LoraArgs a, const int tm, const int most) {
  extern __shared__ int32_t counts[];  // [adapters + 1], then where each one's next token goes
  __shared__ int2 sums[kSort / 64];  // tokens, tiles
  const int groups = a.adapters + 1, lane = threadIdx.x & 63;
  int32_t* const next = counts + groups;
  int g[kHeld];
  const auto read = [&](int t0) {  // -1 past the last token
    const uint32_t* const p = static_cast<const uint32_t*>(a.ids);
    uint32_t high[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int64_t t = min(t0 + i * kSort + (int)threadIdx.x, a.tokens - 1);
      g[i] = (int)p[t << a.ids64];
      high[i] = p[a.ids64 ? 2 * t + 1 : t];
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const bool is = (uint32_t)g[i] < (uint32_t)a.adapters && !(a.ids64 && high[i]);
      g[i] = t0 + i * kSort + (int)threadIdx.x >= a.tokens ? -1 : is ? g[i] : a.adapters;
    }
  };
  read(0);
  for (int i = threadIdx.x; i < groups; i += kSort) counts[i] = 0;
  __syncthreads();
  for (int t0 = 0; t0 < a.tokens; t0 += kHeld * kSort) {
    if (t0 > 0) read(t0);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int g0 = __builtin_amdgcn_readfirstlane(g[i]);
      const uint64_t same = __ballot(g[i] == g0);
      if (g0 >= 0 && lane == 0) atomicAdd(counts + g0, __popcll(same));
      if (g[i] >= 0 && g[i] != g0) atomicAdd(counts + g[i], 1);
    }
  }
  __syncthreads();
  int tokens_before = 0, tiles_before = 0;
#pragma unroll 1
  for (int g0 = 0; g0 < groups; g0 += kSort) {
    const int id = g0 + threadIdx.x, c = id < groups ? counts[id] : 0, tiles = (c + tm - 1) / tm;
    const int c_upto = sum_upto<true>(c), tiles_upto = sum_upto<true>(tiles), wave = threadIdx.x >> 6;
    __syncthreads();  // the last round's reads are done
    if (lane == 63) sums[wave] = int2{c_upto, tiles_upto};
    __syncthreads();
    int at = tokens_before + c_upto - c, tile = tiles_before + tiles_upto - tiles;
#pragma unroll
    for (int w = 0; w < kSort / 64; ++w) {
      const int2 x = sums[w];
      at += w < wave ? x.x : 0;
      tile += w < wave ? x.y : 0;
      tokens_before += x.x;
      tiles_before += x.y;
    }
    if (id < groups) {
      next[id] = at;
#pragma unroll 1
      for (int i = 0; i < tiles; ++i) a.tiles[tile + i] = {id, at + i * tm, min(tm, c - i * tm), 0};
    }
  }
  for (int i = tiles_before + threadIdx.x; i < most; i += kSort) a.tiles[i] = {0, 0, 0, 0};
  __syncthreads();
  for (int t0 = 0; t0 < a.tokens; t0 += kHeld * kSort) {
    if (a.tokens > kHeld * kSort) read(t0);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int g0 = __builtin_amdgcn_readfirstlane(g[i]);
      const uint64_t same = __ballot(g[i] == g0);
      int at = 0;
      if (g0 >= 0 && lane == 0) at = atomicAdd(next + g0, __popcll(same));
      at = __builtin_amdgcn_readfirstlane(at) + __popcll(same & ((1ull << lane) - 1));
      if (g[i] >= 0 && g[i] != g0) at = atomicAdd(next + g[i], 1);
      if (g[i] >= 0) a.order[at] = t0 + i * kSort + threadIdx.x;
    }
  }
}

// Sixteen rows of 64 columns, two 16-byte loads or stores a lane. An operand of the products wants columns 8 g .. + 7 and
// 32 + 8 g .. + 7 of row li from a lane; half a line of a row an instruction, that is 4.3 TB/s of a copy. As they go to and
// from memory a lane has the same columns of rows li % 8 and li % 8 + 8, 8 * (g + 4 * (li / 8)) .. + 7, whole lines of eight
// rows: 4.9 TB/s. The lanes of one and the other trade places by a rotation of their sixteen.
__device__ __forceinline__ u32x4 other_eight(const u32x4& x) {
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x[i], 0x128, 0xF, 0xF, true);  // row_ror:8
  return y;
}
__device__ __forceinline__ u32x4 either(bool first, const u32x4& x, const u32x4& y) {
  u32x4 z;
#pragma unroll
  for (int i = 0; i < 4; ++i) z[i] = first ? x[i] : y[i];
  return z;
}
__device__ __forceinline__ void to_operands(u32x4& x, u32x4& y) {  // from lines: rows li % 8, li % 8 + 8
  const bool low = !(threadIdx.x & 8);
  const u32x4 got = other_eight(either(low, y, x));
  const u32x4 first = either(low, x, got);
  y = either(low, got, y);
  x = first;
}
__device__ __forceinline__ void to_lines(u32x4& x, u32x4& y) { to_operands(x, y); }  // its own inverse

// Which tile and which part of it a workgroup takes. Above rank 32, where weights are much of what is read, the tiles of one
// part follow each other on one XCD, whose L2 then has their adapters' weights: 1000 tokens of 4096 x 4096, rank 64: 25.8 us
// (29.7 as workgroups come), rank 128: 34.0 (39.4), 600 of 8192 x 8192 and 16 adapters, rank 128: 41.0 (47.8). With fewer
// parts (LEAST) XCDs would share them unevenly: 5000 of 8192 x 2048, rank 64: 54.4 (52.9). 1500 of 8192 x 8192,
// rank 64, lose: 48.0 (45.9). Of rank 16 and 32 it gave nothing.
struct Spot {
  int tile, part;
};
template <bool WEIGHTS, int LEAST>
__device__ __forceinline__ Spot spot() {
  if (!WEIGHTS || gridDim.y < LEAST) return {(int)blockIdx.x, (int)blockIdx.y};
  const uint32_t id = xcd_remap_any(blockIdx.x + gridDim.x * blockIdx.y, gridDim.x * gridDim.y), part = id / gridDim.x;
  return {(int)(id - part * gridDim.x), (int)part};
}

// v's part of a tile, a range of K and up to 64 rows of A (ranges of K first along blockIdx.y). A wave takes 64 of K at a
// time (whole lines of x's and A's rows), every fourth such piece; NR * 16 rows of A against MT * 16 tokens, straight from
// memory into the products. The four waves' sums meet in LDS, in a fixed order. Where a SIMD has few waves, or a wave few
// pieces (decode), the next one's loads are on their way during one's products; else the other waves' are. Bound by memory:
// 8191 tokens of 8192, 134 MB of x, in 33 us, 4.1 TB/s.
template <int MT, int NR, bool F16>
__global__ __launch_bounds__(kThreads, MT == 1 ? 1 : MT * NR <= 8 ? 4 : 2) void shrink_kernel(const LoraArgs a) {
  const Spot at = spot<(MT > 1 && NR == 4), 8>();
  constexpr int TM = 16 * MT;
  __shared__ int all_rows[MT == 1 ? kThreads / 64 : 1][TM];
  __shared__ f32x4 meet[2][NR][MT][64];
  int adapter, count;
  int(&rows)[TM] = all_rows[MT == 1 ? threadIdx.x >> 6 : 0];
  if constexpr (MT == 1) {
    if (!find_tile<TM>(a, at.tile, rows, adapter, count, at.part == 0)) return;
  } else {
    if (!read_tile<TM>(a, at.tile, rows, adapter, count)) return;
  }
  constexpr bool kGroups = MT == 1 ? NR == 2 : NR == 4;  // of rows of A there may be more than one
  const int rank_group = kGroups ? at.part / a.splits : 0, split = at.part - rank_group * a.splits;
  const int r0 = rank_group * 16 * NR, rank = rank_of(a, adapter) - r0;
  if (rank <= 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4;
  const int k0 = split * a.k_split, k1 = min(k0 + a.k_split, a.k);
  const int own = 8 * (g + 4 * (li >> 3));  // the lane's columns of a line
  const uint16_t *xr[MT][2], *ar[NR][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int m = 0; m < MT; ++m) xr[m][h] = a.x + rows[m * 16 + (li & 7) + 8 * h] * a.x_row + own;
#pragma unroll
    for (int r = 0; r < NR; ++r)  // rows past the rank repeat its last; what they give is not used
      ar[r][h] = a.a + adapter * a.a_adapter + (r0 + min(r * 16 + (li & 7) + 8 * h, rank - 1)) * a.a_row + own;
  }
  const int used = (rank + 15) / 16;
  struct Piece {
    u32x4 x[MT][2], w[NR][2];
  };
  const auto fetch = [&](int k, Piece& p) {
    const bool on = k + own < k1;  // k % 8 == 0: eight values are inside or past the end
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int r = 0; r < NR; ++r)
        p.w[r][h] = on && r < used ? (MT == 1 ? ld16_nt(ar[r][h] + k) : ld16(ar[r][h] + k)) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int m = 0; m < MT; ++m) p.x[m][h] = on ? (MT == 1 ? ld16(xr[m][h] + k) : ld16_nt(xr[m][h] + k)) : u32x4{0, 0, 0, 0};
    }
  };
  f32x4 acc[NR][MT] = {};
  const auto multiply = [&](Piece& p) {
#pragma unroll
    for (int r = 0; r < NR; ++r) to_operands(p.w[r][0], p.w[r][1]);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      to_operands(p.x[m][0], p.x[m][1]);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < NR; ++r) acc[r][m] = product<F16>(p.w[r][h], p.x[m][h], acc[r][m]);
    }
  };
  int k = k0 + wave * 64;
  if constexpr (MT == 1 || MT * NR > 8) {
    Piece now;
    if (k < k1) fetch(k, now);
    while (k < k1) {
      Piece next;
      const int after = k + 256;
      if (after < k1) fetch(after, next);
      multiply(now);
      now = next;
      k = after;
    }
  } else {
#pragma unroll 1
    for (; k < k1; k += 256) {
      Piece p;
      fetch(k, p);
      multiply(p);
    }
  }
  if (wave >= 2) {
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int m = 0; m < MT; ++m) meet[wave - 2][r][m][lane] = acc[r][m];
  }
  __syncthreads();
  if (wave < 2) {
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[r][m] += meet[wave][r][m][lane];
  }
  __syncthreads();
  if (wave == 1) {
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int m = 0; m < MT; ++m) meet[0][r][m][lane] = acc[r][m];
  }
  __syncthreads();
  if (wave == 0) {  // a lane has rows 16 r + 4 g .. + 3 of token li
    float* const to = a.part + (int64_t)split * a.tokens * a.part_row + r0;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m * 16 + li >= count) continue;
      const int64_t row = (int64_t)rows[m * 16 + li] * a.part_row + 4 * g;
#pragma unroll
      for (int r = 0; r < NR; ++r) *reinterpret_cast<f32x4*>(to + row + 16 * r) = acc[r][m] + meet[0][r][m][lane];
    }
  }
}

// x as a sum of 16-bit pieces, the largest first. bf16 holds 8 bits: three pieces, each what is left cut to its first 8 bits,
// are x itself (down to bf16's least subnormal), and a finite x has none that is not. fp16 holds 11: two pieces leave 2^-23 of
// x, or half its least subnormal, 2^-25. What is not finite is the first piece, with nothing behind it.
constexpr int pieces_of(bool f16) { return f16 ? 2 : 3; }

template <bool F16>
__device__ __forceinline__ void pieces(float x, uint32_t (&to)[pieces_of(F16)]) {
  const bool finite = __builtin_isfinite(x);
  if constexpr (F16) {
    const _Float16 h = (_Float16)x;
    to[0] = __builtin_bit_cast(uint16_t, h);
    to[1] = f32_to_f16_bits(finite ? x - (float)h : 0.0f);
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const uint32_t first = __float_as_uint(x) & 0xFFFF0000u;
      to[i] = first >> 16;
      x = finite ? x - __uint_as_float(first) : 0.0f;
    }
  }
}

template <bool F16>
__device__ __forceinline__ float from16(uint32_t bits) {
  if constexpr (F16)
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  else
    return bf16_lo(bits);
}

// Four values of v of a token from r on, their parts added in order, each piece of the four side by side. fp16 has no room for
// every v: the largest of a token's becomes 2^14 to 2^15, by a power of two, so that 2^-25 is 2^-39 of it and the small ones
// keep their bits too. R / 4 lanes side by side have one token.
template <int R, bool F16>
__device__ __forceinline__ void join_four(const LoraArgs& a, int token, int r, int rank, u32x2 (&to)[pieces_of(F16)],
                                          int& power) {
  f32x4 v = {0, 0, 0, 0};
  if (r < rank) {
    const float* from = a.part + (int64_t)token * R + r;
    const int64_t step = (int64_t)a.tokens * R;
    constexpr int kAhead = 8;
#pragma unroll 1
    for (int s = 0; s < a.splits; s += kAhead) {
      f32x4 y[kAhead];
#pragma unroll
      for (int e = 0; e < kAhead; ++e) y[e] = *reinterpret_cast<const f32x4*>(from + min(s + e, a.splits - 1) * step);
#pragma unroll
      for (int e = 0; e < kAhead; ++e) v += s + e < a.splits ? y[e] : f32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (r + e >= rank) v[e] = 0.0f;
  }
  power = 0;
  if constexpr (F16) {
    float top = 0.0f;  // of the finite ones
#pragma unroll
    for (int j = 0; j < 4; ++j) top = fmaxf(top, __builtin_isfinite(v[j]) ? fabsf(v[j]) : 0.0f);
#pragma unroll
    for (int d = 1; d < R / 4; d *= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
    power = top > 0.0f ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __builtin_amdgcn_ldexpf(v[j], -power);
  }
  uint32_t w[4][pieces_of(F16)];
#pragma unroll
  for (int e = 0; e < 4; ++e) pieces<F16>(v[e], w[e]);
#pragma unroll
  for (int i = 0; i < pieces_of(F16); ++i) to[i] = u32x2{w[0][i] | w[1][i] << 16, w[2][i] | w[3][i] << 16};
}

// Where many workgroups need the same parts of v: joined once, not by each of them.
template <int NR, bool F16>
__global__ __launch_bounds__(kThreads) void join_kernel(const LoraArgs a) {
  constexpr int R = 16 * NR;
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int token = (int)min(id / (R / 4), (int64_t)a.tokens - 1), r = (int)(id % (R / 4)) * 4;
  u32x2 v[pieces_of(F16)];
  int power;
  join_four<R, F16>(a, token, r, rank_of(a, adapter_of(a, token)), v, power);
  if (id >= (int64_t)a.tokens * (R / 4)) return;
#pragma unroll
  for (int i = 0; i < pieces_of(F16); ++i)
    *reinterpret_cast<u32x2*>(a.joined + ((int64_t)i * a.tokens + token) * R + r) = v[i];
  if (F16 && r == 0) a.powers[token] = power;
}

// The outputs of a tile for n_group columns. A wave takes 64 columns at a time, four products' rows: row i of the q-th is
// column 32 (q / 2) + 8 (i / 4) + 4 (q % 2) + i % 4, so that a lane ends with twice eight columns side by side of one token,
// which go to memory as whole lines. B's rows stay in registers for all the tile's tokens; base comes sixteen tokens ahead,
// the first of it and of B before v. Bound by memory: 8191 tokens of 10240, 336 MB of base and out, in 76 us, 4.4 TB/s.
enum Mode : int { kParts, kJoined, kStreamed };  // v from its parts, joined, and with base and out passing the caches by

template <int MT, int NR, bool F16, Mode MODE>
__global__ __launch_bounds__(kThreads) void expand_kernel(const LoraArgs a) {
  const Spot at = spot<(MT > 1 && NR >= 4), 16>();
  constexpr int TM = 16 * MT, R = 16 * NR, kSteps = (R + 31) / 32, kRow = kSteps * 32 + 8;  // a row of pieces: 16 bytes more
  constexpr int kPieces = pieces_of(F16);
  constexpr bool kStream = MODE == kStreamed;
  __shared__ int rows[TM];
  __shared__ __align__(16) uint16_t piece[kPieces][TM][kRow];
  __shared__ int power[TM];
  int adapter, count;
  if (!read_tile<TM>(a, at.tile, rows, adapter, count)) return;
  const int rank = rank_of(a, adapter);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4;
  const int c0 = at.part * a.n_group, c1 = min(c0 + a.n_group, a.n);
  if (rank == 0) {
    if (!a.copies) return;
    constexpr int kAhead = 4;
    const int units = (c1 - c0) / 8, all = count * units;  // n % 8 == 0
    for (int u0 = threadIdx.x; u0 < all; u0 += kAhead * kThreads) {
      u32x4 held[kAhead];
      uint16_t* to[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int u = min(u0 + i * kThreads, all - 1), t = rows[u / units], c = c0 + u % units * 8;
        held[i] = ld16(a.base + t * a.base_row + c);
        to[i] = a.out + t * a.out_row + c;
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (u0 + i * kThreads < all) *reinterpret_cast<u32x4*>(to[i]) = held[i];
    }
    return;
  }
  const int steps = (rank + 31) / 32, own = 8 * (g + 4 * (li >> 3));  // the lane's columns of a line
  u32x4 w[kSteps][4], old[2];
  const auto load_w = [&](int c) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int r0 = s * 32 + g * 8;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        // those past the end are not stored
        const int n = min(c + (q >> 1) * 32 + (li >> 2) * 8 + (q & 1) * 4 + (li & 3), a.n - 1);
        w[s][q] = r0 < rank ? ld16(a.b + adapter * a.b_adapter + n * a.b_row + r0) : u32x4{0, 0, 0, 0};
      }
    }
  };
  const auto load_old = [&](int c, int m, u32x4 (&o)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = m * 16 + (li & 7) + 8 * h;
      o[h] = u32x4{0, 0, 0, 0};
      if (t >= count || c + own >= c1) continue;
      const uint16_t* const from = a.base + rows[t] * a.base_row + c + own;
      o[h] = kStream ? ld16_nt(from) : ld16(from);
    }
  };
  int c = c0 + wave * 64;
  if (c < c1) {
    load_w(c);
    load_old(c, 0, old);
  }
  if constexpr (MODE == kParts) {
    constexpr int kLanes = R / 4;
#pragma unroll
    for (int i = 0; i < (TM * kLanes + kThreads - 1) / kThreads; ++i) {
      const int id = i * kThreads + threadIdx.x, t = id / kLanes, r = id % kLanes * 4;
      if (TM * kLanes % kThreads != 0 && t >= TM) break;
      u32x2 v[kPieces];
      int e;
      join_four<R, F16>(a, rows[t], r, t < count ? rank : 0, v, e);
#pragma unroll
      for (int p = 0; p < kPieces; ++p) *reinterpret_cast<u32x2*>(&piece[p][t][r]) = v[p];
      if (r == 0) power[t] = e;
    }
  } else {
    constexpr int kEach = TM * R / 8;  // 16 bytes each
#pragma unroll
    for (int i = 0; i < (kPieces * kEach + kThreads - 1) / kThreads; ++i) {
      const int id = i * kThreads + threadIdx.x, p = id / kEach, t = id % kEach / (R / 8), r = id % (R / 8) * 8;
      if (kPieces * kEach % kThreads != 0 && p >= kPieces) break;
      *reinterpret_cast<u32x4*>(&piece[p][t][r]) = ld16(a.joined + ((int64_t)p * a.tokens + rows[t]) * R + r);
    }
    if (F16 && (int)threadIdx.x < TM) power[threadIdx.x] = a.powers[rows[threadIdx.x]];
  }
  if (R < 32 && (int)threadIdx.x < TM) {  // the products' K is 32
#pragma unroll
    for (int i = 0; i < 2 * kPieces; ++i)
      *reinterpret_cast<u32x4*>(&piece[i / 2][threadIdx.x][R + i % 2 * 8]) = u32x4{0, 0, 0, 0};
  }
  __syncthreads();
  const float scale = a.scales ? a.scales[adapter] : 1.0f;
  while (c < c1) {
    const int after = c + kThreads;
    if (rank % 8) {  // what lies behind the rank may be anything
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (s * 32 + g * 8 + e >= rank) {
#pragma unroll
            for (int q = 0; q < 4; ++q) w[s][q][e / 2] &= e % 2 ? 0x0000FFFFu : 0xFFFF0000u;
          }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      u32x4 next[2];
      if (m + 1 < MT)
        load_old(c, m + 1, next);
      else if (after < c1)
        load_old(after, 0, next);
      f32x4 acc[4] = {};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (s >= steps) break;
#pragma unroll
        for (int p = kPieces - 1; p >= 0; --p) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(&piece[p][m * 16 + li][s * 32 + g * 8]);
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[q] = product<F16>(w[s][q], v, acc[q]);
        }
      }
      if (m + 1 == MT && after < c1) load_w(after);
      const int e = F16 ? power[m * 16 + li] : 0;
      to_operands(old[0], old[1]);
      u32x4 word[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float y[2];
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const int at = 8 * h + 2 * j + z;
            float d = acc[at / 4][at % 4];
            if constexpr (F16) d = __builtin_amdgcn_ldexpf(d, e);
            y[z] = fmaf(d, scale, from16<F16>(z ? old[h][j] >> 16 : old[h][j] & 0xFFFFu));
          }
          word[h][j] = pack_out2(y[0], y[1], F16 ? AKLR_OUT_F16 : AKLR_OUT_BF16);
        }
      to_lines(word[0], word[1]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = m * 16 + (li & 7) + 8 * h;
        if (t >= count || c + own >= c1) continue;
        u32x4* const to = reinterpret_cast<u32x4*>(a.out + rows[t] * a.out_row + c + own);
        if (kStream)
          __builtin_nontemporal_store(word[h], to);
        else
          *to = word[h];
      }
      old[0] = next[0];
      old[1] = next[1];
    }
    c = after;
  }
}

}  // namespace aklr

using namespace aklr;

namespace {

// Rows of A, in sixteens, that a workgroup of the first product takes: others take the rest of a larger rank.
constexpr int shrink_nr(int mt, int nr) { return mt == 1 && nr > 2 ? 2 : nr > 4 ? 4 : nr; }

struct Plan {
  int mt, nr;         // tiles of 16 tokens, of 16 rank rows
  int64_t tiles;      // workgroups along x: the most tiles there can be
  int64_t splits, k_split, n_group, rank_groups;
  bool joins;         // v's parts by a launch of their own
  size_t order, tile, part, joined, powers, bytes;  // offsets in the workspace
};

int64_t up(int64_t v, int64_t q) { return (v + q - 1) / q * q; }

// The plan of a call, from its sizes alone. Measured on 8 adapters, bf16, us (both sides of each choice, with two pieces of v;
// the third takes 0.5 to 2 % more, 3 at rank 128 and 8191 tokens):
// - up to 256 tokens each wave looks for its tile: 120 tokens of 4096 x 4096, rank 16: 9.6 (sorted: 14.8), 250: 11.0 (15.7).
// - 64 tokens a tile from 7168 tokens on, 32 below: 8191 of 8192 x 10240, rank 32: 120 (32 a tile: 131), rank 64: 142
//   (163); 6000 of 4096 x 4096, rank 16: 46 (64 a tile: 53), 6269 of 840 x 5512: 55 (57), 3000 and fewer the same. Above
//   rank 32, where a tile's weights are more than its tokens, from 2560 on: 5000 of 8192 x 2048, rank 64: 52.9 (60.9), rank
//   128: 78 (101), 2600 of 4096 x 4096, rank 128: 51 (56); 2000 of 8192 x 2048, rank 64: 36.5 (64 a tile: 40.7).
// - up to 256 tokens 32 rows of A a workgroup: 4 tokens of 7168 x 2112, rank 64: 10.2 (64 rows: 12.3, 16: 9.9), 64 of 7168
//   x 4608, rank 128: 17.7 (19.3, 18.6), 200 of 2048 x 8192, rank 64: 15.6 (17.7, 15.9).
// - as many ranges of K as make the workgroups that run at once, of at least 512; up to 256 tokens six workgroups a CU: 192
//   tokens of 48 adapters, 8192 x 10240, rank 64: 27.6 (four a CU: 28.4, eight: 30.1).
// - 256 columns a workgroup, 512 where that makes more than 2048: the same call 27.6 (256: 1.2 more, 1024: 2.3), 8191 of
//   8192 x 10240 120 (256: 123, 1024: 122).
// - v joined by a launch of its own (3 to 5 us) where workgroups would read and convert much of it again and again, a
//   conversion about as much as eight parts' reads: 8191 of 8192 x 10240, rank 32: 120 (from its parts 129), of 4096 x
//   4096, rank 128: 107 (114), 3000 of 4096 x 4096, rank 64: 42.5 (joined 43.9), rank 16: 30.9 (34.4).
Plan plan_lora(int64_t tokens, int64_t k, int64_t n, int64_t rank, int64_t adapters) {
  Plan p{};
  p.nr = rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8;
  const bool sorts = tokens > kScan;
  p.mt = !sorts ? 1 : tokens < (p.nr < 4 ? 7168 : 2560) ? 2 : 4;
  p.rank_groups = p.nr / shrink_nr(p.mt, p.nr);
  const int64_t tm = 16 * p.mt, groups = adapters + 1 < tokens ? adapters + 1 : tokens;
  const int64_t most = (tokens + tm - 1) / tm + groups;  // sum of ceil(c / tm) over groups of c tokens
  p.tiles = most < tokens ? most : tokens;
  // what registers leave room for, and for one token a tile more, since their work is uneven
  int64_t splits = 256 * (p.mt == 1 ? 6 : p.nr < 4 ? 4 : p.mt < 4 ? 3 : 2) / (p.tiles * p.rank_groups);
  if (splits > (k + 511) / 512) splits = (k + 511) / 512;
  if (splits < 1) splits = 1;
  p.k_split = up((k + splits - 1) / splits, 256);
  p.splits = (k + p.k_split - 1) / p.k_split;
  p.n_group = p.tiles * ((n + 255) / 256) > 2048 ? 512 : 256;
  p.joins = sorts && tokens * 16 * p.nr * ((n + p.n_group - 1) / p.n_group) * (p.splits + 8) > 70000000;
  size_t at = 0;
  p.order = at;
  at += up(4 * (sorts ? tokens : p.tiles * tm), 256);
  p.tile = at;
  at += up(16 * p.tiles, 256);
  p.part = at;
  at += up(4 * p.splits * tokens * 16 * p.nr, 256);
  p.joined = at;
  if (p.joins) at += up(2 * pieces_of(false) * tokens * 16 * p.nr, 256);
  p.powers = at;
  if (p.joins) at += up(4 * tokens, 256);
  p.bytes = at;
  return p;
}

bool sizes_ok(int64_t tokens, int64_t k, int64_t n, int64_t rank, int64_t adapters) {
  return tokens >= 1 && tokens <= (1 << 20) && k >= 8 && k <= 65536 && k % 8 == 0 && n >= 8 && n <= 262144 && n % 8 == 0 &&
         rank >= 8 && rank <= 128 && rank % 8 == 0 && adapters >= 1 && adapters <= kMostAdapters;
}

bool row_ok(const void* p, int64_t stride, int64_t least) {
  return p && aklr_aligned16(p) && stride % 8 == 0 && stride >= least;
}

}  // namespace

extern "C" size_t aklr_lora_project_workspace_bytes(int64_t tokens, int64_t k, int64_t n, int64_t rank, int64_t adapters) {
  return sizes_ok(tokens, k, n, rank, adapters) ? plan_lora(tokens, k, n, rank, adapters).bytes : 0;
}

extern "C" int aklr_lora_project(const void* x, int64_t x_stride, const void* a, int64_t a_adapter_stride,
                                 int64_t a_row_stride, const void* b, int64_t b_adapter_stride, int64_t b_row_stride,
                                 const void* adapters, int adapters_64, const float* scales, const int32_t* ranks,
                                 const void* base, int64_t base_stride, void* out, int64_t out_stride, int64_t tokens,
                                 int64_t k, int64_t n, int64_t rank, int64_t adapter_count, int dtype, void* workspace,
                                 size_t workspace_bytes, hipStream_t stream) {
  if (dtype != AKLR_OUT_BF16 && dtype != AKLR_OUT_F16) return AKLR_ERR_UNSUPPORTED;
  if (tokens == 0) return AKLR_OK;
  if (!sizes_ok(tokens, k, n, rank, adapter_count)) return AKLR_ERR_INVALID_ARGUMENT;
  if (!row_ok(x, x_stride, 0) || !row_ok(a, a_row_stride, 0) || a_adapter_stride % 8 || !row_ok(b, b_row_stride, 0) ||
      b_adapter_stride % 8 || !row_ok(base, base_stride, 0) || !row_ok(out, out_stride, tokens > 1 ? n : 0) || !adapters)
    return AKLR_ERR_INVALID_ARGUMENT;
  const Plan p = plan_lora(tokens, k, n, rank, adapter_count);
  if (!workspace || !aklr_aligned16(workspace) || workspace_bytes < p.bytes) return AKLR_ERR_WORKSPACE;
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  LoraArgs g{};
  g.x = static_cast<const uint16_t*>(x);
  g.a = static_cast<const uint16_t*>(a);
  g.b = static_cast<const uint16_t*>(b);
  g.base = static_cast<const uint16_t*>(base);
  g.out = static_cast<uint16_t*>(out);
  g.x_row = x_stride;
  g.a_adapter = a_adapter_stride;
  g.a_row = a_row_stride;
  g.b_adapter = b_adapter_stride;
  g.b_row = b_row_stride;
  g.base_row = base_stride;
  g.out_row = out_stride;
  g.ids = adapters;
  g.scales = scales;
  g.ranks = ranks;
  g.part = reinterpret_cast<float*>(ws + p.part);
  g.joined = reinterpret_cast<uint16_t*>(ws + p.joined);
  g.powers = reinterpret_cast<int32_t*>(ws + p.powers);
  g.order = reinterpret_cast<int32_t*>(ws + p.order);
  g.tiles = reinterpret_cast<Tile*>(ws + p.tile);
  g.tokens = (int)tokens;
  g.k = (int)k;
  g.n = (int)n;
  g.rank = (int)rank;
  g.adapters = (int)adapter_count;
  g.ids64 = adapters_64;
  g.splits = (int)p.splits;
  g.k_split = (int)p.k_split;
  g.n_group = (int)p.n_group;
  g.copies = base != out;
  g.part_row = 16 * p.nr;
  const auto whole_lines = [](const void* q, int64_t stride) {
    return reinterpret_cast<uintptr_t>(q) % 128 == 0 && stride % 64 == 0;
  };
  const bool streams = whole_lines(base, base_stride) && whole_lines(out, out_stride);
  if (tokens > kScan) {
    hipLaunchKernelGGL(sort_kernel, dim3(1), dim3(kSort), 8 * (adapter_count + 1), stream, g, 16 * p.mt, (int)p.tiles);
    AKLR_LAUNCH_CHECK();
  }
  const dim3 shrink((unsigned)p.tiles, (unsigned)(p.splits * p.rank_groups));
  const dim3 expand((unsigned)p.tiles, (unsigned)((n + p.n_group - 1) / p.n_group));
  const auto go = [&](auto mt, auto nr, auto f16) -> int {
    constexpr int MT = decltype(mt)::value, NR = decltype(nr)::value;
    constexpr bool F16 = decltype(f16)::value;
    hipLaunchKernelGGL((shrink_kernel<MT, shrink_nr(MT, NR), F16>), shrink, dim3(kThreads), 0, stream, g);
    AKLR_LAUNCH_CHECK();
    if constexpr (MT > 1) {
      if (p.joins) {
        const dim3 grid((unsigned)((tokens * NR * 4 + kThreads - 1) / kThreads));
        hipLaunchKernelGGL((join_kernel<NR, F16>), grid, dim3(kThreads), 0, stream, g);
        AKLR_LAUNCH_CHECK();
        if (MT == 4 && streams)
          hipLaunchKernelGGL((expand_kernel<MT, NR, F16, MT == 4 ? kStreamed : kJoined>), expand, dim3(kThreads), 0, stream, g);
        else
          hipLaunchKernelGGL((expand_kernel<MT, NR, F16, kJoined>), expand, dim3(kThreads), 0, stream, g);
        AKLR_LAUNCH_CHECK();
        return AKLR_OK;
      }
    }
    hipLaunchKernelGGL((expand_kernel<MT, NR, F16, kParts>), expand, dim3(kThreads), 0, stream, g);
    AKLR_LAUNCH_CHECK();
    return AKLR_OK;
  };
  const auto by_rank = [&](auto mt, auto f16) -> int {
    return p.nr == 1   ? go(mt, IC<1>{}, f16)
           : p.nr == 2 ? go(mt, IC<2>{}, f16)
           : p.nr == 4 ? go(mt, IC<4>{}, f16)
                       : go(mt, IC<8>{}, f16);
  };
  const auto by_rows = [&](auto f16) -> int {
    return p.mt == 1 ? by_rank(IC<1>{}, f16) : p.mt == 2 ? by_rank(IC<2>{}, f16) : by_rank(IC<4>{}, f16);
  };
  return dtype == AKLR_OUT_F16 ? by_rows(IC<1>{}) : by_rows(IC<0>{});
}

AKLR_SCALAR_FP32_END
