// Rotary positions and the FP8 key/value cache: the elementwise operators around an attention over it.
// gfx950 only.
//
// The cache holds, for keys and for values, e4m3fn codes [pages, kv heads, page, head_dim] and one fp32 scale per
// token and head [pages, kv heads, page]: a head's tokens of one page are contiguous, so the attention reads whole
// lines of them, and a token's write is one vector of head_dim bytes per head.
#include "common.h"

AKLR_SCALAR_FP32_BEGIN

namespace aklr {

constexpr int kThreads = 256;
constexpr int kManyGroups = 4096;
constexpr int64_t kMostGroups = 1 << 23;  // of one launch along x: it has fewer than 2^32 threads
constexpr int64_t kManyItems = 1 << 20;

// Eight consecutive values of T (bf16 bits, fp16 or fp32) as fp32, and back with one rounding to nearest even.
template <typename T>
struct Eight;
template <>
struct Eight<__bf16> {
  u32x4 w;
  __device__ __forceinline__ void load(const void* p) { w = ld16(p); }
  __device__ __forceinline__ void to(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = bf16_lo(w[i]), f[2 * i + 1] = bf16_hi(w[i]);
  }
  __device__ __forceinline__ static void store(void* p, const float (&f)[8]) {
    *static_cast<u32x4*>(p) = u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                                    pack_bf16x2(f[6], f[7])};
  }
};
template <>
struct Eight<_Float16> {
  typedef _Float16 h8 __attribute__((ext_vector_type(8)));
  u32x4 w;
  __device__ __forceinline__ void load(const void* p) { w = ld16(p); }
  __device__ __forceinline__ void to(float (&f)[8]) const {
    const h8 h = __builtin_bit_cast(h8, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
  }
  __device__ __forceinline__ static void store(void* p, const float (&f)[8]) {
    h8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)f[i];
    *static_cast<u32x4*>(p) = __builtin_bit_cast(u32x4, h);
  }
};
template <>
struct Eight<float> {
  f32x4 a, b;
  __device__ __forceinline__ void load(const void* p) {
    a = static_cast<const f32x4*>(p)[0];
    b = static_cast<const f32x4*>(p)[1];
  }
  __device__ __forceinline__ void to(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = a[i], f[4 + i] = b[i];
  }
  __device__ __forceinline__ static void store(void* p, const float (&f)[8]) {
    static_cast<f32x4*>(p)[0] = f32x4{f[0], f[1], f[2], f[3]};
    static_cast<f32x4*>(p)[1] = f32x4{f[4], f[5], f[6], f[7]};
  }
};

__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int is64) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

// One side of the cache (keys or values) and where its pages lie.
struct CacheSide {
  uint8_t* codes;
  float* scales;
  int64_t code_page, scale_page;  // elements from one page to the next
};

struct Heads {  // a strided [tokens, heads, head_dim] tensor, in elements; the last dimension is contiguous
  const void* in;
  void* out;
  int64_t in_token, in_head, out_token, out_head;
  int heads;
};

struct VecArgs {
  Heads q, k, v;         // rotary: q, k; write: k, v
  CacheSide kc, vc;      // write
  const void* positions;  // rotary
  const double* freq;
  const void* slots;  // write
  float magnitude;
  int first, tokens, per_wg;  // the launch's tokens from `first` to before `tokens`, and how many a workgroup takes at once
  int rot, interleaved, pos64, slot64;
  int kv_heads, page;
  int64_t slot_count;
};

// A vector of 16 values is a lane's item, D / 16 lanes hold one head of one token, and a workgroup walks the items of
// its tokens (blockIdx.x) and its share of their heads (blockIdx.y). ROT: q (and k) are rotated; WRITE: k and v are
// quantized into the cache.
//
// Rotation: a pair (a, b) at angle pos * f becomes (a cos - b sin, b cos + a sin). The angle is taken in 64 bits, in
// revolutions, and only its fraction goes on in 32, so far positions cost no accuracy (a position of 2^20 has
// 1.7e5 revolutions: an fp32 product would be off by 0.01 of one). A workgroup works each angle out once for all heads
// of its tokens: one lane, one pair, kept in LDS, while the items' loads are in flight. In the half layout a lane takes
// 8 values of each half, so that it holds whole pairs in both layouts.
//
// Quantization (the arithmetic of aklr_per_group_quant_fp8 at one group a head): s = max(amax, 1e-10) * fl32(1/448),
// code = e4m3(clamp(x * (1/s))). A rotated k goes from fp32 straight into its code. A vector that holds a NaN or an
// infinity gets zero codes under a NaN scale, so it reads as NaN throughout and no NaN code enters the cache.
//
// Bound by memory where there are many tokens (figures at launch_vec), by the launch and one chain of loads where few:
// 3.4 us for 64 tokens of 8 heads written, 3.5 for 16 tokens of 129 heads rotated, 3.9 for 8 of 80 rotated and written.
template <typename T, int D, bool ROT, bool WRITE>
__global__ __launch_bounds__(kThreads) void vec_kernel(const VecArgs a, const int head_dim) {
  const int dim = D ? D : head_dim;
  const int units = dim / 16;
  const int rot_units = ROT ? a.rot / 16 : 0;
  extern __shared__ float2 turn[];  // [per_wg][rot / 2] (cos, sin)
  const int t0 = a.first + blockIdx.x * a.per_wg;
  const int nt = min(a.per_wg, a.tokens - t0);
  const int heads = (ROT ? a.q.heads : 0) + a.k.heads + (WRITE ? a.v.heads : 0);
  const int row = heads * units;  // items a token
  const int items = nt * row;

  struct Item {
    const T* from;
    T* to;                // rotated only
    int t, u, head;       // token, unit, head of its tensor
    int at0, at1;         // where the item's two eights lie in the head
    int kind;             // 0 q, 1 k, 2 v
    bool turned, on;
  };
  auto locate = [&](int i) {
    Item m;
    m.on = i < items;
    i = m.on ? i : 0;
    m.t = i / row;
    const int r = i - m.t * row;
    int head = r / units;
    m.u = r - head * units;
    const int hq = ROT ? a.q.heads : 0;
    m.kind = head < hq ? 0 : head < hq + a.k.heads ? 1 : 2;
    head -= m.kind == 0 ? 0 : m.kind == 1 ? hq : hq + a.k.heads;
    m.head = head;
    m.turned = ROT && m.kind != 2 && m.u < rot_units;
    const bool half = m.turned && !a.interleaved;
    m.at0 = half ? 8 * m.u : 16 * m.u;
    m.at1 = half ? a.rot / 2 + 8 * m.u : 16 * m.u + 8;
    const int64_t t = t0 + m.t;
    const void* in = m.kind == 0 ? a.q.in : m.kind == 1 ? a.k.in : a.v.in;
    const int64_t in_token = m.kind == 0 ? a.q.in_token : m.kind == 1 ? a.k.in_token : a.v.in_token;
    const int64_t in_head = m.kind == 0 ? a.q.in_head : m.kind == 1 ? a.k.in_head : a.v.in_head;
    m.from = static_cast<const T*>(in) + t * in_token + head * in_head;
    m.to = nullptr;
    if (ROT) {
      const bool first = WRITE || m.kind == 0;
      m.to = static_cast<T*>(first ? a.q.out : a.k.out) + t * (first ? a.q.out_token : a.k.out_token) +
             head * (first ? a.q.out_head : a.k.out_head);
    }
    return m;
  };
  auto fetch = [&](const Item& m, Eight<T>& x, Eight<T>& y) {
    x.load(m.from + m.at0);
    y.load(m.from + m.at1);
  };
  const int step = gridDim.y * kThreads;
  int i = blockIdx.y * kThreads + threadIdx.x;
  const int last = (items + 63) / 64 * 64;  // whole waves go on, for the reductions over lanes
  Item m = locate(i);
  Eight<T> x, y;
  if (m.on) fetch(m, x, y);
  if (ROT) {
    const int pairs = a.rot / 2;
    for (int j = threadIdx.x; j < nt * pairs; j += kThreads) {
      const int t = j / pairs;
      const double pos = (double)load_index(a.positions, t0 + t, a.pos64);
      const double rev = pos * a.freq[j - t * pairs] * 0.15915494309189533577;  // 1 / (2 pi)
      float s, c;
      sincospif((float)(2.0 * (rev - __builtin_rint(rev))), &s, &c);
      turn[j] = float2{c * a.magnitude, s * a.magnitude};
    }
    __syncthreads();
  }
  while (i < last) {
    float f[8], g[8];
    if (m.on) {
      x.to(f);
      y.to(g);
    }
    const Item now = m;
    i += step;
    if (i < last) {  // the next item's loads, before this one's arithmetic
      m = locate(i);
      if (m.on) fetch(m, x, y);
    }
    if (!now.on) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = g[e] = 0.0f;
    }
    if (ROT && now.turned) {
      const float2* cs = turn + now.t * (a.rot / 2) + 8 * now.u;
      if (a.interleaved) {  // pairs (2e, 2e + 1): four in f, four in g
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 u = cs[e], w = cs[4 + e];
          const float f0 = f[2 * e], f1 = f[2 * e + 1], g0 = g[2 * e], g1 = g[2 * e + 1];
          f[2 * e] = f0 * u.x - f1 * u.y;
          f[2 * e + 1] = f1 * u.x + f0 * u.y;
          g[2 * e] = g0 * w.x - g1 * w.y;
          g[2 * e + 1] = g1 * w.x + g0 * w.y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 u = cs[e];
          const float f0 = f[e], g0 = g[e];
          f[e] = f0 * u.x - g0 * u.y;
          g[e] = g0 * u.x + f0 * u.y;
        }
      }
    }
    if (ROT && now.on && (!WRITE || now.kind == 0)) {
      Eight<T>::store(now.to + now.at0, f);
      Eight<T>::store(now.to + now.at1, g);
    }
    if constexpr (WRITE) {
      // the largest magnitude as bits: a NaN's are above infinity's, which are above every finite value's
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        top = max(top, __float_as_uint(f[e]) & 0x7FFFFFFFu);
        top = max(top, __float_as_uint(g[e]) & 0x7FFFFFFFu);
      }
#pragma unroll
      for (int s = 1; s < D / 16; s *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, s, 64));
      if (now.on && now.kind != 0) {
        const int64_t slot = load_index(a.slots, t0 + now.t, a.slot64);
        if (slot >= 0 && slot < a.slot_count) {  // others (a padded batch's) are skipped
          const bool bad = top >= 0x7F800000u;
          const float scale = fmaxf(__uint_as_float(top), kAmaxFloor) * kInv448;
          const float inv = 1.0f / scale;
          const uint32_t page = (uint32_t)slot / (uint32_t)a.page, off = (uint32_t)slot % (uint32_t)a.page;
          const bool v = now.kind == 2;
          uint8_t* codes = (v ? a.vc.codes : a.kc.codes) + page * (v ? a.vc.code_page : a.kc.code_page);
          float* scales = (v ? a.vc.scales : a.kc.scales) + page * (v ? a.vc.scale_page : a.kc.scale_page);
          const int64_t token = (int64_t)now.head * a.page + off;
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f[e] = fminf(fmaxf(f[e] * inv, -448.0f), 448.0f);
            g[e] = fminf(fmaxf(g[e] * inv, -448.0f), 448.0f);
          }
          o[0] = pack4_e4m3(f[0], f[1], f[2], f[3]);
          o[1] = pack4_e4m3(f[4], f[5], f[6], f[7]);
          o[2] = pack4_e4m3(g[0], g[1], g[2], g[3]);
          o[3] = pack4_e4m3(g[4], g[5], g[6], g[7]);
          if (bad) o[0] = o[1] = o[2] = o[3] = 0;
          *reinterpret_cast<u32x2*>(codes + token * D + now.at0) = u32x2{o[0], o[1]};
          *reinterpret_cast<u32x2*>(codes + token * D + now.at1) = u32x2{o[2], o[3]};
          if (now.u == 0) scales[token] = bad ? __uint_as_float(0x7FC00000u) : scale;
        }
      }
    }
  }
}

// How many tokens a workgroup takes and how many workgroups share them: one item a lane, which is all that a write alone
// needs (8191 tokens of 8 heads of 256: 22.9 us, 4.4 TB/s of reads and writes; a large copy reaches 5.2). With a rotation,
// where that makes many workgroups, one takes all heads of a token, so that its angles are worked out once: 8192 tokens of
// 32 + 8 heads of 128 rotated and written in 43.9 us instead of 49.9 (two tokens a workgroup 43.0, four 43.9), 5003 rotated
// in 18.5 instead of 19.7 (two 19.7, four 21.7).
template <typename T, int D, bool ROT, bool WRITE>
int launch_vec(VecArgs& a, int head_dim, hipStream_t stream) {
  const int64_t row = (int64_t)((ROT ? a.q.heads : 0) + a.k.heads + (WRITE ? a.v.heads : 0)) * (head_dim / 16);
  const int64_t tokens = a.tokens;
  if (row == 0 || tokens == 0) return AKLR_OK;
  a.per_wg = (int)(row >= kThreads ? 1 : kThreads / row);
  if (ROT && a.per_wg > 2048 / a.rot) a.per_wg = 2048 / a.rot;  // angles a workgroup keeps: 8 KiB
  int64_t gy = (row * a.per_wg + kThreads - 1) / kThreads;
  if (ROT && (tokens + a.per_wg - 1) / a.per_wg * gy > kManyGroups) gy = 1;
  if (gy > 65535) return AKLR_ERR_INVALID_ARGUMENT;
  const size_t lds = ROT ? (size_t)a.per_wg * (a.rot / 2) * sizeof(float2) : 0;
  const int64_t most = kMostGroups * a.per_wg;
  for (int64_t first = 0; first < tokens; first += most) {
    a.first = (int)first;
    a.tokens = (int)(first + most < tokens ? first + most : tokens);
    hipLaunchKernelGGL((vec_kernel<T, D, ROT, WRITE>), dim3((unsigned)((a.tokens - first + a.per_wg - 1) / a.per_wg), (unsigned)gy),
                       dim3(kThreads), lds, stream, a, head_dim);
    AKLR_LAUNCH_CHECK();
  }
  return AKLR_OK;
}

// ---------------------------------------------------------------------------------------------------------------
// A packed prefix out of the pages: workgroup x takes `rows` consecutive rows, y keys or values. Rows' places are looked
// up once a row (a binary search of the sequence, then the block table), then a lane turns 16 codes into 16 values, two
// of them where there are many: 188 k rows of 8 heads of 128 in 224 us (5.1 TB/s of codes and values, as a large copy)
// instead of 240 with one or four items a lane and 266 with eight, 3 x 700 rows of 2 heads of 64 in 3.6 with one.
struct ReadSide {
  const uint8_t* codes;
  const float* scales;
  int64_t code_page, scale_page;
  void* out;
};

constexpr int kReadRows = 128;

template <int D, bool F16>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadSide k, ReadSide v, const int32_t* table, int64_t table_row,
                                                        int64_t table_cols, const int32_t* starts, int batch,
                                                        int64_t total, int heads, int page, int64_t pages, int rows) {
  constexpr int U = D / 16;
  __shared__ int64_t place[kReadRows];  // page, or -1: no such page, or -2: no such row
  __shared__ int offset[kReadRows];
  const int64_t r0 = (int64_t)blockIdx.x * rows;
  const ReadSide& s = blockIdx.y ? v : k;
  if ((int)threadIdx.x < rows) {
    const int64_t r = r0 + threadIdx.x;
    int lo = 0, hi = batch;  // the first sequence that ends behind r
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if ((int64_t)starts[mid + 1] > r)
        hi = mid;
      else
        lo = mid + 1;
    }
    int64_t at = -2;
    int off = 0;
    if (r < total && lo < batch && starts[lo] <= r) {
      const int64_t pos = r - starts[lo], p = pos / page;
      off = (int)(pos - p * page);
      at = p < table_cols ? (int64_t)table[lo * table_row + p] : -1;
      if (at < 0 || at >= pages) at = -1;
    }
    place[threadIdx.x] = at;
    offset[threadIdx.x] = off;
  }
  __syncthreads();
  const int row = heads * U;
  for (int i = threadIdx.x; i < rows * row; i += kThreads) {
    const int r = i / row, rest = i - r * row, h = rest / U, u = rest % U;
    const int64_t at = place[r];
    if (at == -2) continue;
    uint32_t o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (at >= 0) {
      const int64_t token = (int64_t)h * page + offset[r];
      const u32x4 c = ld16(s.codes + at * s.code_page + token * D + u * 16);
      const float scale = s.scales[at * s.scale_page + token];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[e], false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[e], true);
        o[2 * e] = pack_out2(lo[0] * scale, lo[1] * scale, F16 ? AKLR_OUT_F16 : AKLR_OUT_BF16);
        o[2 * e + 1] = pack_out2(hi[0] * scale, hi[1] * scale, F16 ? AKLR_OUT_F16 : AKLR_OUT_BF16);
      }
    }
    u32x4* p = reinterpret_cast<u32x4*>(static_cast<uint16_t*>(s.out) + ((r0 + r) * heads + h) * D + u * 16);
    __builtin_nontemporal_store(u32x4{o[0], o[1], o[2], o[3]}, p);
    __builtin_nontemporal_store(u32x4{o[4], o[5], o[6], o[7]}, p + 1);
  }
}

}  // namespace aklr

using namespace aklr;

namespace {

bool strides_ok(const void* p, int64_t token, int64_t head, int size) {
  return aklr_aligned16(p) && (token * size) % 16 == 0 && (head * size) % 16 == 0;
}

int element_size(int dtype) { return dtype == AKLR_F32 ? 4 : 2; }

bool cache_ok(const void* codes, const void* scales, int64_t code_page, int64_t scale_page, int64_t kv_heads,
              int64_t head_dim, int64_t page) {
  return codes && scales && aklr_aligned16(codes) && aklr_aligned16(scales) && code_page >= kv_heads * page * head_dim &&
         scale_page >= kv_heads * page && code_page % 16 == 0 && scale_page % 4 == 0;
}

bool cache_shape_ok(int64_t pages, int64_t page, int64_t kv_heads, int64_t head_dim) {
  return (head_dim == 64 || head_dim == 128 || head_dim == 256) && page >= 16 && page <= 1024 && page % 16 == 0 &&
         kv_heads >= 1 && kv_heads <= 1024 && pages >= 1 && pages * page <= 0x7FFFFFFF;
}

bool rotary_ok(const void* positions, const void* freq, int64_t rot, int64_t head_dim) {
  return positions && freq && rot >= 16 && rot % 16 == 0 && rot <= head_dim;
}

template <int D, bool ROT, bool WRITE>
int by_type(VecArgs& a, int64_t head_dim, int dtype, hipStream_t stream) {
  if (dtype == AKLR_OUT_BF16) return launch_vec<__bf16, D, ROT, WRITE>(a, (int)head_dim, stream);
  if (dtype == AKLR_OUT_F16) return launch_vec<_Float16, D, ROT, WRITE>(a, (int)head_dim, stream);
  return launch_vec<float, D, ROT, WRITE>(a, (int)head_dim, stream);
}

}  // namespace

extern "C" int aklr_rotary_embedding(const void* q, int64_t q_token, int64_t q_head, void* q_out, int64_t q_out_token,
                                     int64_t q_out_head, int64_t q_heads, const void* k, int64_t k_token,
                                     int64_t k_head, void* k_out, int64_t k_out_token, int64_t k_out_head,
                                     int64_t k_heads, const void* positions, int positions_64, const double* frequencies,
                                     int64_t tokens, int64_t head_dim, int64_t rotary_dim, int interleaved,
                                     float magnitude, int dtype, hipStream_t stream) {
  if (dtype < AKLR_OUT_BF16 || dtype > AKLR_F32) return AKLR_ERR_UNSUPPORTED;
  const int size = element_size(dtype);
  if (tokens < 0 || tokens > 0x7FFFFFFF || q_heads < 1 || k_heads < 0 || q_heads + k_heads > 65536 || head_dim < 16 ||
      head_dim > 1024 || head_dim % 16 != 0 || !rotary_ok(positions, frequencies, rotary_dim, head_dim))
    return AKLR_ERR_INVALID_ARGUMENT;
  if (!q || !q_out || !strides_ok(q, q_token, q_head, size) || !strides_ok(q_out, q_out_token, q_out_head, size))
    return AKLR_ERR_INVALID_ARGUMENT;
  if (k_heads && (!k || !k_out || !strides_ok(k, k_token, k_head, size) || !strides_ok(k_out, k_out_token, k_out_head, size)))
    return AKLR_ERR_INVALID_ARGUMENT;
  VecArgs a{};
  a.q = {q, q_out, q_token, q_head, q_out_token, q_out_head, (int)q_heads};
  a.k = {k, k_out, k_token, k_head, k_out_token, k_out_head, (int)k_heads};
  a.positions = positions;
  a.freq = frequencies;
  a.magnitude = magnitude;
  a.tokens = (int)tokens;
  a.rot = (int)rotary_dim;
  a.interleaved = interleaved;
  a.pos64 = positions_64;
  return by_type<0, true, false>(a, head_dim, dtype, stream);
}

extern "C" int aklr_kv_cache_write_fp8(const void* q, int64_t q_token, int64_t q_head, void* q_out, int64_t q_out_token,
                                       int64_t q_out_head, int64_t q_heads, const void* k, int64_t k_token,
                                       int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                                       const void* positions, int positions_64, const double* frequencies,
                                       int64_t rotary_dim, int interleaved, float magnitude, const void* slots,
                                       int slots_64, void* k_codes, void* v_codes, float* k_scales, float* v_scales,
                                       int64_t k_page, int64_t v_page, int64_t ks_page, int64_t vs_page,
                                       int64_t tokens, int64_t kv_heads, int64_t head_dim, int64_t pages,
                                       int64_t page_size, int dtype, hipStream_t stream) {
  if (dtype < AKLR_OUT_BF16 || dtype > AKLR_F32) return AKLR_ERR_UNSUPPORTED;
  const int size = element_size(dtype);
  if (!cache_shape_ok(pages, page_size, kv_heads, head_dim) || tokens < 0 || tokens > 0x7FFFFFFF || q_heads < 0 ||
      q_heads > 65536 || !slots)
    return AKLR_ERR_INVALID_ARGUMENT;
  if (!cache_ok(k_codes, k_scales, k_page, ks_page, kv_heads, head_dim, page_size) ||
      !cache_ok(v_codes, v_scales, v_page, vs_page, kv_heads, head_dim, page_size))
    return AKLR_ERR_INVALID_ARGUMENT;
  if (!k || !v || !strides_ok(k, k_token, k_head, size) || !strides_ok(v, v_token, v_head, size))
    return AKLR_ERR_INVALID_ARGUMENT;
  const bool rotate = rotary_dim != 0;
  if (rotate && !rotary_ok(positions, frequencies, rotary_dim, head_dim)) return AKLR_ERR_INVALID_ARGUMENT;
  if (q_heads && (!rotate || !q || !q_out || !strides_ok(q, q_token, q_head, size) ||
                  !strides_ok(q_out, q_out_token, q_out_head, size)))
    return AKLR_ERR_INVALID_ARGUMENT;
  VecArgs a{};
  a.q = {q, q_out, q_token, q_head, q_out_token, q_out_head, (int)q_heads};
  a.k = {k, nullptr, k_token, k_head, 0, 0, (int)kv_heads};
  a.v = {v, nullptr, v_token, v_head, 0, 0, (int)kv_heads};
  a.kc = {static_cast<uint8_t*>(k_codes), k_scales, k_page, ks_page};
  a.vc = {static_cast<uint8_t*>(v_codes), v_scales, v_page, vs_page};
  a.positions = positions;
  a.freq = frequencies;
  a.slots = slots;
  a.magnitude = magnitude;
  a.tokens = (int)tokens;
  a.rot = (int)rotary_dim;
  a.interleaved = interleaved;
  a.pos64 = positions_64;
  a.slot64 = slots_64;
  a.page = (int)page_size;
  a.slot_count = pages * page_size;
  const auto go = [&](auto d) {
    constexpr int D = decltype(d)::value;
    return rotate ? by_type<D, true, true>(a, D, dtype, stream) : by_type<D, false, true>(a, D, dtype, stream);
  };
  return head_dim == 64 ? go(IC<64>{}) : head_dim == 128 ? go(IC<128>{}) : go(IC<256>{});
}

extern "C" int aklr_kv_cache_read_fp8(const void* k_codes, const void* v_codes, const float* k_scales,
                                      const float* v_scales, int64_t k_page, int64_t v_page, int64_t ks_page,
                                      int64_t vs_page, const int32_t* block_table, int64_t table_stride,
                                      int64_t table_cols, const int32_t* starts, int64_t batch, int64_t total,
                                      void* k_out, void* v_out, int64_t kv_heads, int64_t head_dim, int64_t pages,
                                      int64_t page_size, int out_dtype, hipStream_t stream) {
  if (out_dtype != AKLR_OUT_BF16 && out_dtype != AKLR_OUT_F16) return AKLR_ERR_UNSUPPORTED;
  if (!cache_shape_ok(pages, page_size, kv_heads, head_dim) || batch < 0 || batch > 0x7FFFFFFF || total < 0 ||
      total > 0x7FFFFFFF || table_cols < 0 || table_stride < table_cols)
    return AKLR_ERR_INVALID_ARGUMENT;
  if (!cache_ok(k_codes, k_scales, k_page, ks_page, kv_heads, head_dim, page_size) ||
      !cache_ok(v_codes, v_scales, v_page, vs_page, kv_heads, head_dim, page_size))
    return AKLR_ERR_INVALID_ARGUMENT;
  if (batch == 0 || total == 0) return AKLR_OK;
  if (!block_table || !starts || !k_out || !v_out || !aklr_aligned16(k_out) || !aklr_aligned16(v_out))
    return AKLR_ERR_INVALID_ARGUMENT;
  const ReadSide k = {static_cast<const uint8_t*>(k_codes), k_scales, k_page, ks_page, k_out};
  const ReadSide v = {static_cast<const uint8_t*>(v_codes), v_scales, v_page, vs_page, v_out};
  const int64_t row = kv_heads * head_dim / 16;
  const int64_t fit = (kThreads * (total * row > kManyItems ? 2 : 1) + row - 1) / row;
  const int64_t rows = fit < kReadRows ? fit : kReadRows;
  if ((total + rows - 1) / rows > 0xFFFFFF) return AKLR_ERR_INVALID_ARGUMENT;  // a launch has fewer than 2^32 threads
  const dim3 grid((unsigned)((total + rows - 1) / rows), 2);
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, k, v, block_table, table_stride, table_cols, starts,
                       (int)batch, total, (int)kv_heads, (int)page_size, pages, (int)rows);
  };
  const bool f16 = out_dtype == AKLR_OUT_F16;
  if (head_dim == 64)
    f16 ? go(read_kernel<64, true>) : go(read_kernel<64, false>);
  else if (head_dim == 128)
    f16 ? go(read_kernel<128, true>) : go(read_kernel<128, false>);
  else
    f16 ? go(read_kernel<256, true>) : go(read_kernel<256, false>);
  AKLR_LAUNCH_CHECK();
  return AKLR_OK;
}

AKLR_SCALAR_FP32_END
