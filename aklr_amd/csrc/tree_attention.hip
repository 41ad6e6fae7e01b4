// Attention of a few query tokens of each sequence over its paged FP8 cache: decode, trees of drafted tokens, chunks
// of a prompt. gfx950 only.
//
// Row (t, h): query token t of a sequence, query head h of a kv head's group. The sequence's last T positions are its T
// query tokens, the ctx = len - T before them are seen by every row, and token t sees token j where mask[t][j] (without
// a mask: j <= t). With codes c and scales s of keys and values, in base 2:
//   x_p = (q . ck_p) * (sk_p * softmax_scale * log2 e),  m = max x_p,  l = sum 2^(x_p - m),
//   o = sum (2^(x_p - m) * sv_p) cv_p / l.
// A scale belongs to a token, so it multiplies a column of the scores and of the weights, never the codes: codes turn
// into bf16 (fp16 for fp16 queries against keys) exactly, two an instruction, and the products run on matrix units.
// The weights times sv are rounded to bf16 for that (half a step, at most 2^-8 of each term); scores, maxima, sums and outputs
// stay in fp32.
#include "common.h"

AKLR_SCALAR_FP32_BEGIN

namespace aklr {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4, kThreads = 256;
constexpr int kUnit = 128;  // tokens a workgroup takes in one step: 32 a wave

struct AttnArgs {
  const void* q;
  int64_t q_token, q_head;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  int64_t k_page, v_page, ks_page, vs_page;
  const int32_t* table;
  int64_t table_row;
  const int32_t *lens, *starts;
  const uint8_t* mask;
  int64_t mask_row;
  void* out;
  float* lse;
  float* part;
  uint64_t page_magic;  // 2^32 / (page / 16) + 1
  int table_cols, mask_cols, total, batch, hq, hkv, group, page, pages;
  int target;  // work items a kv head is cut into, beside one for each tile of rows
  int cap;     // items a kv head can have
  float scale_log2;
};

// What one workgroup does. Every workgroup works it out from the lengths on the device, so no length has to be known
// to the host and a captured launch serves other lengths: rows are cut into tiles of R, a sequence's tokens into
// chunks of `chunk` units, the same for all sequences and so that the items come to about `target`.
struct Item {
  int b, tiles, tile, split, splits, chunk;
  int q0, count, len;  // the sequence's first query token, how many, its positions
  int slot;            // TILES: of the partial result of the tile's first split
  bool ok;
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Item `index` of a kv head, or (TILES) tile `index`. Wave-wide: lane i looks at sequence i of each 64.
template <int R, bool TILES>
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
  for (int b0 = 64; b0 < a.batch; b0 += 64) {
    const One x = look(b0 + lane);
    work += (int64_t)x.tiles * x.units;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) work += __shfl_xor(work, d, 64);
  Item r{};
  r.chunk = uniform((int)fmin((double)work / a.target, (double)(1 << 23)) + 1);
  int base = 0, slots = 0;  // tiles (or items) and items before the 64 sequences at hand
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (b0) s = look(b0 + lane);
    const int splits = (s.units + r.chunk - 1) / r.chunk;
    const int items = s.tiles * splits;
    int before = items, tiles = s.tiles;  // inclusive sums over the lanes
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(before, d, 64), y = __shfl_up(tiles, d, 64);
      if (lane >= d) before += x, tiles += y;
    }
    const int mine = TILES ? tiles : before;
    const uint64_t past = __ballot(base + mine > index);
    if (past) {
      const int at = __builtin_ctzll(past);
      auto take = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
      r.b = b0 + at;
      r.tiles = take(s.tiles);
      r.splits = take(splits);
      const int within = index - base - (take(mine) - (TILES ? r.tiles : r.tiles * r.splits));
      r.split = TILES ? 0 : within / r.tiles;
      r.tile = TILES ? within : within - r.split * r.tiles;
      r.q0 = take(s.q0);
      r.count = take(s.count);
      r.len = take(s.len);
      r.slot = slots + take(before) - r.tiles * r.splits + r.split * r.tiles + r.tile;
      r.ok = true;
      return r;
    }
    base += __builtin_amdgcn_readlane(mine, 63);
    slots += __builtin_amdgcn_readlane(before, 63);
  }
  return r;
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
__device__ __forceinline__ uint32_t two(uint32_t codes) {  // two e4m3 codes of a word as bf16 (fp16), exactly
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

// Partial results: for each slot, o [R][D] not yet divided by l, then m [R] and l [R].
template <int D, int R>
__device__ __forceinline__ float* slot_at(const AttnArgs& a, int head, int slot) {
  return a.part + ((int64_t)head * a.cap + slot) * (R * (D + 2));
}

template <bool F16, int N>
__device__ __forceinline__ void store_row(void* out, int64_t at, const float (&v)[N], float by) {
  uint32_t* p = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(out) + at);
#pragma unroll
  for (int i = 0; i < N / 2; ++i)
    p[i] = pack_out2(v[2 * i] * by, v[2 * i + 1] * by, F16 ? AKLR_OUT_F16 : AKLR_OUT_BF16);
}

// Rows by the 16 * NQ, tokens by the 32 of a wave, all in registers. S^T = K Q^T puts a row in a lane (column c of the
// accumulator) and tokens 4g..4g+3 of each 16 in lane group g, which is just what the second product wants of its
// operand P^T, so the weights never move between lanes: O^T = V^T P^T sums over k in any order as long as both
// operands agree, and lane group g holds its own 4 + 4 tokens' values. The order of the head's dimension is free too: a
// lane loads head_dim / 16 consecutive codes of each of its tokens (a token's 16 lanes a whole line), turns them over
// in registers, and ends with head_dim / 4 consecutive outputs of its row.
template <int D, int NQ, bool F16>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void stream_kernel(const AttnArgs a) {
  constexpr int R = 16 * NQ, VW = D / 64;  // VW: words of a lane's codes of a token
  constexpr int KL = D / 64;               // 16-byte loads of a key row a lane (D = 64: one)
  constexpr int QS = D / 32;               // steps of 32 along the head
  constexpr int DT = D / 16;               // output tiles along the head
  const int head = blockIdx.x % a.hkv;
  const int index = blockIdx.x / a.hkv;
  const Item it = find<R, false>(a, index);
  if (!it.ok) return;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int rows = it.count * a.group, r0 = it.tile * R, ctx = it.len - it.count;
  const int last_t = (min(r0 + R, rows) - 1) / a.group, first_t = r0 / a.group;
  // positions any row of the tile sees, and those all of its rows see
  const int seen = a.mask ? it.len : min(it.len, ctx + last_t + 1);
  const int from = it.split * it.chunk * kUnit;  // below len
  const int end = (int)min((int64_t)seen, from + (int64_t)it.chunk * kUnit);
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

  struct Tile {
    u32x4 k[2][KL];
    uint32_t v[8][VW];
    f32x4 ks[2], vs[2];
    int pages[2];
  };
  const int32_t* table = a.table + it.b * a.table_row;
  auto page_of = [&](int pos) { return (int)(((uint64_t)(pos >> 4) * a.page_magic) >> 32); };
  auto look = [&](int p, int (&id)[2]) {  // the pages of positions p.. and p + 16..
#pragma unroll
    for (int h = 0; h < 2; ++h) id[h] = p < end ? table[min(page_of(p + 16 * h), a.table_cols - 1)] : 0;
  };
  auto load = [&](Tile& t, int p, const int (&id)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      t.pages[h] = id[h];
      const int64_t page = (uint32_t)id[h] < (uint32_t)a.pages ? id[h] : 0;
      const int off = p + 16 * h - page_of(p + 16 * h) * a.page;
      const int64_t token = (int64_t)head * a.page + off;
      const uint8_t* k = a.kc + page * a.k_page + token * D;
      const uint8_t* v = a.vc + page * a.v_page + token * D;
#pragma unroll
      for (int i = 0; i < KL; ++i)
        t.k[h][i] = ld16(k + c * D + (D == 64 ? 16 * g : 128 * (i / 2) + 32 * g + 16 * (i % 2)));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(v + (4 * g + j) * D + c * (D / 16));
        if constexpr (VW == 1) {
          t.v[4 * h + j][0] = w[0];
        } else if constexpr (VW == 2) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(w);
          t.v[4 * h + j][0] = x[0];
          t.v[4 * h + j][1] = x[1];
        } else {
          const u32x4 x = ld16(w);
#pragma unroll
          for (int i = 0; i < 4; ++i) t.v[4 * h + j][i] = x[i];
        }
      }
      t.ks[h] = *reinterpret_cast<const f32x4*>(a.ks + page * a.ks_page + token + 4 * g);
      t.vs[h] = *reinterpret_cast<const f32x4*>(a.vs + page * a.vs_page + token + 4 * g);
    }
  };

  f32x4 o[NQ][DT];
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = -__builtin_inff();
    l[n] = 0.0f;
#pragma unroll
    for (int i = 0; i < DT; ++i) o[n][i] = f32x4{0, 0, 0, 0};
  }

  auto compute = [&](Tile& t, int p) {
    f32x4 x[NQ][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) x[n][h] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < QS; ++s) {
        const uint32_t w0 = t.k[h][s / 2][2 * (s % 2)], w1 = t.k[h][s / 2][2 * (s % 2) + 1];
        const u32x4 k = {two<F16, false>(w0), two<F16, true>(w0), two<F16, false>(w1), two<F16, true>(w1)};
#pragma unroll
        for (int n = 0; n < NQ; ++n) x[n][h] = mfma32<F16>(k, q[n][s], x[n][h]);
      }
      t.ks[h] *= a.scale_log2;
#pragma unroll
      for (int n = 0; n < NQ; ++n) x[n][h] *= t.ks[h];
    }
    // Positions that some row does not see, or that hold no token: nothing in them may reach a row that does not see
    // them, NaN included. Scores are replaced; a weight of zero times a NaN would still be one, so a value's NaN code
    // moves into its token's scale, which only rows that see the token multiply by.
    const bool edge = p + 32 > clear || (uint32_t)t.pages[0] >= (uint32_t)a.pages || (uint32_t)t.pages[1] >= (uint32_t)a.pages;
    uint32_t sees[NQ];
    if (edge) {
      uint32_t held = 0;  // bit 4h + i: token p + 16h + 4g + i is there
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (p + 16 * h + 4 * g + i < end && (uint32_t)t.pages[h] < (uint32_t)a.pages) held |= 1u << (4 * h + i);
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        sees[n] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int j = p + 16 * (i / 4) + 4 * g + i % 4 - ctx;
          bool s = (held >> i) & 1;
          if (s && j >= 0) {
            if (a.mask)
              s = j < a.mask_cols && a.mask[(it.q0 + row_t[n]) * a.mask_row + j] != 0;
            else
              s = j <= row_t[n];
          }
          sees[n] |= (s ? 1u : 0u) << i;
          if (!s) x[n][i / 4][i % 4] = -__builtin_inff();
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t nan = 0;
#pragma unroll
        for (int w = 0; w < VW; ++w) nan |= ((t.v[i][w] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
        const bool bad = ((__ballot(nan != 0) >> (16 * g)) & 0xFFFF) != 0;
        if (bad) t.vs[i / 4][i % 4] = __uint_as_float(0x7FC00000u);
        if (bad || !((held >> i) & 1)) {
#pragma unroll
          for (int w = 0; w < VW; ++w) t.v[i][w] = 0;
        }
      }
    }
    u32x4 pt[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float top = x[n][0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, x[n][i / 4][i % 4]);
      top = across(top, [](float u, float v) { return fmaxf(u, v); });
      if (__ballot(top > m[n])) {  // some row has a new maximum: what it summed so far shrinks
        const float now = fmaxf(m[n], top);
        const float by = m[n] < now ? __builtin_amdgcn_exp2f(m[n] - now) : 1.0f;
        m[n] = now;
        l[n] *= by;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[n][i] *= by;
      }
      const float at = m[n] == -__builtin_inff() ? 0.0f : m[n];
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = __builtin_amdgcn_exp2f(x[n][i / 4][i % 4] - at);
        l[n] += e;
        w[i] = e * t.vs[i / 4][i % 4];
        if (edge && !((sees[n] >> i) & 1)) w[i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) pt[n][i] = pack_bf16x2(w[2 * i], w[2 * i + 1]);
    }
#pragma unroll
    for (int e = 0; e < DT / 2; ++e) {
      u32x4 lo, hi;  // dimensions 2e and 2e + 1 of this lane's, over its 8 tokens
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x0 = t.v[2 * j][e / 2], x1 = t.v[2 * j + 1][e / 2];
        const uint32_t b0 = e % 2 ? two<false, true>(x0) : two<false, false>(x0);
        const uint32_t b1 = e % 2 ? two<false, true>(x1) : two<false, false>(x1);
        lo[j] = __builtin_amdgcn_perm(b1, b0, 0x05040100);
        hi[j] = __builtin_amdgcn_perm(b1, b0, 0x07060302);
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        o[n][2 * e] = mfma32<false>(lo, pt[n], o[n][2 * e]);
        o[n][2 * e + 1] = mfma32<false>(hi, pt[n], o[n][2 * e + 1]);
      }
    }
  };

  // The next tile's codes are on their way while one is computed, and the pages of the one after it
  int p = from + 32 * wave, ahead[2];
  Tile x, y;
  look(p, ahead);
  if (p < end) load(x, p, ahead);
  look(p + kUnit, ahead);
  while (p < end) {
    if (p + kUnit < end) load(y, p + kUnit, ahead);
    look(p + 2 * kUnit, ahead);
    compute(x, p);
    p += kUnit;
    if (p >= end) break;
    if (p + kUnit < end) load(x, p + kUnit, ahead);
    look(p + 2 * kUnit, ahead);
    compute(y, p);
    p += kUnit;
  }

  // The waves' sums meet in LDS, in wave order; rows padded by 4 floats, which spreads 8 rows over the banks
  __shared__ float wave_m[kWaves][R], wave_l[kWaves][R];
  __shared__ __align__(16) float sum[kWaves][16][D + 4];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] = across(l[n], [](float u, float v) { return u + v; });
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
      float* to = slot_at<D, R>(a, head, index);
#pragma unroll
      for (int i = 0; i < DT; i += 4)
        *reinterpret_cast<f32x4*>(to + (16 * n + r) * D + d + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
      if (d == 0) to[R * D + 16 * n + r] = best, to[R * (D + 1) + 16 * n + r] = total;
    } else if (row < rows) {
      const int t = row / a.group, h = row - t * a.group;
      const int64_t at = (int64_t)(it.q0 + t) * a.hq + head * a.group + h;
      store_row<F16>(a.out, at * D + d, v, total == 0.0f ? 0.0f : 1.0f / total);
      if (a.lse && d == 0) a.lse[at] = total == 0.0f ? -__builtin_inff() : (best + __log2f(total)) * 0.69314718f;
    }
  }
}

// The splits of a tile of rows, in their order.
template <int D, int R, bool F16>
__global__ __launch_bounds__(kThreads) void join_kernel(const AttnArgs a) {
  constexpr int DT = D / 16;
  const int head = blockIdx.x % a.hkv;
  const Item it = find<R, true>(a, blockIdx.x / a.hkv);
  if (!it.ok || it.splits == 1) return;
  if (it.slot < 0 || it.slot + (int64_t)(it.splits - 1) * it.tiles >= a.cap) return;  // starts that do not ascend
  const int rows = it.count * a.group, d = (threadIdx.x & 15) * DT;
  for (int r = threadIdx.x >> 4; r < R; r += kThreads / 16) {
    const int row = it.tile * R + r;
    if (row >= rows) break;
    float best = -__builtin_inff(), total = 0.0f, v[DT];
    for (int s = 0; s < it.splits; ++s)
      best = fmaxf(best, slot_at<D, R>(a, head, it.slot + s * it.tiles)[R * D + r]);
#pragma unroll
    for (int i = 0; i < DT; ++i) v[i] = 0.0f;
    for (int s = 0; s < it.splits; ++s) {
      const float* p = slot_at<D, R>(a, head, it.slot + s * it.tiles);
      const float m = p[R * D + r], by = m == best ? 1.0f : __builtin_amdgcn_exp2f(m - best);
      total += p[R * (D + 1) + r] * by;
#pragma unroll
      for (int i = 0; i < DT; i += 4) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(p + r * D + d + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i + e] += x[e] * by;
      }
    }
    const int t = row / a.group, h = row - t * a.group;
    const int64_t at = (int64_t)(it.q0 + t) * a.hq + head * a.group + h;
    store_row<F16>(a.out, at * D + d, v, total == 0.0f ? 0.0f : 1.0f / total);
    if (a.lse && d == 0) a.lse[at] = total == 0.0f ? -__builtin_inff() : (best + __log2f(total)) * 0.69314718f;
  }
}

// ---------------------------------------------------------------------------------------------------------------
constexpr int kTarget = 512;  // workgroups a call is cut into beside one for each tile of rows: two for each CU

struct AttnPlan {
  int nq;
  int64_t target, tiles, cap;
  size_t bytes;
};

bool plan_attention(int64_t total, int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t capacity, AttnPlan* p) {
  const int64_t group = hq / hkv;
  p->nq = total * group > 16 * batch && d < 256 ? 2 : 1;  // more than 16 rows a sequence, on the mean
  const int64_t r = 16 * p->nq;
  p->target = (kTarget + hkv - 1) / hkv;
  p->tiles = total * group / r + (batch < total ? batch : total);
  const int64_t units = (capacity + kUnit - 1) / kUnit;
  p->cap = p->tiles + (units > 1 ? p->target : 0);
  if (p->cap * hkv > 0x7FFFFFFF) return false;
  p->bytes = units > 1 ? (size_t)(p->cap * hkv * r * (d + 2)) * sizeof(float) : 0;
  return true;
}

template <int D, int NQ, bool F16>
int launch_attention(const AttnArgs& a, const AttnPlan& p, hipStream_t stream) {
  hipLaunchKernelGGL((stream_kernel<D, NQ, F16>), dim3((unsigned)(p.cap * a.hkv)), dim3(kThreads), 0, stream, a);
  AKLR_LAUNCH_CHECK();
  if (p.bytes) {
    hipLaunchKernelGGL((join_kernel<D, 16 * NQ, F16>), dim3((unsigned)(p.tiles * a.hkv)), dim3(kThreads), 0, stream, a);
    AKLR_LAUNCH_CHECK();
  }
  return AKLR_OK;
}

bool attention_shape_ok(int64_t total, int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t capacity) {
  return total >= 0 && batch >= 0 && batch <= 65536 && hkv >= 1 && hkv <= 1024 && hq >= hkv && hq % hkv == 0 &&
         hq <= 65536 && total * (hq / hkv) <= 0x3FFFFFFF && (d == 64 || d == 128 || d == 256) && capacity >= 0 &&
         capacity <= (1 << 30);
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

extern "C" int aklr_tree_attention_fp8(const void* q, int64_t q_token, int64_t q_head, const void* k_codes,
                                       const void* v_codes, const float* k_scales, const float* v_scales,
                                       int64_t k_page, int64_t v_page, int64_t ks_page, int64_t vs_page,
                                       const int32_t* block_table, int64_t table_stride, int64_t table_cols,
                                       const int32_t* seq_lens, const int32_t* starts, const void* mask,
                                       int64_t mask_stride, int64_t mask_cols, void* out, float* lse, int64_t total_q,
                                       int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                       int64_t pages, int64_t page_size, float softmax_scale, int dtype, void* workspace,
                                       size_t workspace_bytes, hipStream_t stream) {
  if (dtype != AKLR_OUT_BF16 && dtype != AKLR_OUT_F16) return AKLR_ERR_UNSUPPORTED;
  if (page_size < 16 || page_size > 1024 || page_size % 16 != 0 || pages < 1 || pages * page_size > 0x7FFFFFFF ||
      table_cols < 0 || table_cols > (1 << 26) || table_stride < table_cols ||
      !attention_shape_ok(total_q, batch, q_heads, kv_heads, head_dim, table_cols * page_size))
    return AKLR_ERR_INVALID_ARGUMENT;
  if (total_q == 0 || batch == 0) return AKLR_OK;
  if (!q || !k_codes || !v_codes || !k_scales || !v_scales || !seq_lens || !starts || !out || (table_cols && !block_table))
    return AKLR_ERR_INVALID_ARGUMENT;
  if (!aklr_aligned16(q) || !aklr_aligned16(k_codes) || !aklr_aligned16(v_codes) || !aklr_aligned16(k_scales) ||
      !aklr_aligned16(v_scales) || !aklr_aligned16(out) || q_token % 8 != 0 || q_head % 8 != 0)
    return AKLR_ERR_INVALID_ARGUMENT;
  const int64_t page_codes = kv_heads * page_size * head_dim, page_scales = kv_heads * page_size;
  if (k_page < page_codes || v_page < page_codes || ks_page < page_scales || vs_page < page_scales || k_page % 16 != 0 ||
      v_page % 16 != 0 || ks_page % 4 != 0 || vs_page % 4 != 0)
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
  a.k_page = k_page;
  a.v_page = v_page;
  a.ks_page = ks_page;
  a.vs_page = vs_page;
  a.table = block_table;
  a.table_row = table_stride;
  a.lens = seq_lens;
  a.starts = starts;
  a.mask = static_cast<const uint8_t*>(mask);
  a.mask_row = mask_stride;
  a.out = out;
  a.lse = lse;
  a.part = static_cast<float*>(workspace);
  a.page_magic = (1ull << 32) / (uint64_t)(page_size / 16) + 1;
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
  a.cap = (int)p.cap;
  a.scale_log2 = softmax_scale * 1.44269504f;
  const auto go = [&](auto d, auto nq) {
    constexpr int D = decltype(d)::value, NQ = decltype(nq)::value;
    return dtype == AKLR_OUT_F16 ? launch_attention<D, NQ, true>(a, p, stream) : launch_attention<D, NQ, false>(a, p, stream);
  };
  if (head_dim == 256) return go(IC<256>{}, IC<1>{});
  if (head_dim == 128) return p.nq == 1 ? go(IC<128>{}, IC<1>{}) : go(IC<128>{}, IC<2>{});
  return p.nq == 1 ? go(IC<64>{}, IC<1>{}) : go(IC<64>{}, IC<2>{});
}

AKLR_SCALAR_FP32_END
