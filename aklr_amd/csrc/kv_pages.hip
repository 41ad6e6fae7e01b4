// Pages of the FP8 key/value cache: copied, compacted, and handed from sequence to sequence. gfx950 only.
//
// The cache is kv_cache.hip's: e4m3fn codes [pages, kv heads, page, head_dim] and fp32 scales [pages, kv heads, page] for
// keys and for values. Nothing here computes with what it holds; the operators move bytes and count holders.
#include "common.h"
#include "scan.h"

AKLR_SCALAR_FP32_BEGIN

namespace aklr {

constexpr int kThreads = 256;
constexpr int64_t kMostGroups = 1 << 23;  // of one launch: it has fewer than 2^32 threads

__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int is64) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

struct Side {  // keys or values
  uint8_t* codes;
  float* scales;
  int64_t code_page, scale_page;  // elements from one page to the next
};

// ---------------------------------------------------------------------------------------------------------------
// Page src[i] onto page dst[i], all four tensors in one launch. A page is 2 * (heads * page * (D + 4)) bytes in pieces of
// 16; a workgroup takes kCopyUnits of them, all its loads before its stores. Bound by memory: 1024 pages of 135 KB, 277 MB read
// and written, in 55 us, 5.0 TB/s; a call of a few pages is its launch and two dependent loads, 4.1 us.
constexpr int kCopyUnits = 4 * kThreads;

__global__ __launch_bounds__(kThreads) void copy_kernel(const Side k, const Side v, const void* src, const void* dst,
                                                        const int is64, const int64_t pages, const int code_units,
                                                        const int scale_units, const int chunks, const int64_t first) {
  const int64_t wg = first + blockIdx.x, i = wg / chunks;
  const int chunk = (int)(wg - i * chunks);
  const int64_t from = load_index(src, i, is64), to = load_index(dst, i, is64);
  if (from < 0 || from >= pages || to < 0 || to >= pages || from == to) return;
  const int units = 2 * (code_units + scale_units);
  u32x4 held[4];
  u32x4* place[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    int u = chunk * kCopyUnits + j * kThreads + (int)threadIdx.x;
    place[j] = nullptr;
    if (u >= units) continue;
    uint8_t* base;
    int64_t step;
    if (u < 2 * code_units) {
      const bool second = u >= code_units;
      base = second ? v.codes : k.codes;
      step = second ? v.code_page : k.code_page;
      u -= second ? code_units : 0;
    } else {
      u -= 2 * code_units;
      const bool second = u >= scale_units;
      base = reinterpret_cast<uint8_t*>(second ? v.scales : k.scales);
      step = 4 * (second ? v.scale_page : k.scale_page);
      u -= second ? scale_units : 0;
    }
    held[j] = ld16_nt(base + from * step + (int64_t)u * 16);
    place[j] = reinterpret_cast<u32x4*>(base + to * step + (int64_t)u * 16);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (place[j]) __builtin_nontemporal_store(held[j], place[j]);
}

// ---------------------------------------------------------------------------------------------------------------
// Compaction: position first + path[b, i] onto first + i, first = seq_lens[b] - T, T = starts[b + 1] - starts[b], for
// i < counts[b]. Entries outside [0, T) are passed over wherever they stand; the others, the items, ascend. Without such
// entries each item moves down (i < path[i]) or stays; behind some it may move up. A place of an item that moves down may be
// the source of an earlier one that does, never of a later one; of one that moves up, of a later one, never of an earlier
// one. And no place of one kind is a source of the other: of items i < j one has path[i] < path[j], so i < path[i] gives
// i < path[j], and j > path[j] gives j > path[i].
struct CompactArgs {
  Side k, v;
  const int32_t *table, *lens, *starts, *path, *counts;
  int64_t table_row, path_row;
  int table_cols, heads, page, most;
  int64_t pages;
  int b0, batch;      // the launch's sequences
  int w0, w1;         // its items
  uint8_t* saved;     // [2][sequences of the launch][w1 - w0][heads][D] codes, then the scales
  float* saved_scales;
  int32_t* up;        // with several windows: whether there are items that move up, which these leave alone
};

struct Place {  // of a position: its page, -1 where the cache has none, and the token's place in it
  int page, off;
};

__device__ __forceinline__ Place place_of(const CompactArgs& a, int b, int64_t pos) {
  if (pos < 0 || pos >= (int64_t)a.table_cols * a.page) return {-1, 0};
  const int col = (int)pos / a.page;  // a table reaches 2^28 positions
  const int32_t p = a.table[(int64_t)b * a.table_row + col];
  return {p < 0 || p >= a.pages ? -1 : p, (int)pos - col * a.page};
}

// Source and place of item i: no page in `from` where there is nothing to do (not an item, kept where it is, no such page).
__device__ __forceinline__ void item_of(const CompactArgs& a, int b, int i, Place& from, Place& to, int& source) {
  const int64_t t = (int64_t)a.starts[b + 1] - a.starts[b];
  const int64_t first = (int64_t)a.lens[b] - t;
  from = to = {-1, 0};
  source = -1;
  if (i >= a.counts[b] || i >= a.most) return;
  const int32_t x = a.path[(int64_t)b * a.path_row + i];
  if (x < 0 || x >= t || x == i) return;
  to = place_of(a, b, first + i);
  if (to.page >= 0) from = place_of(a, b, first + x);
  source = x;
}

// Items in an order in which nothing is read that has been written: those that move down from the first, those that move up
// from the last. A lane owns 16 bytes of one head (or its scale) for every item of a sequence, kHeld at a time: it reads what
// it will move before it writes. A workgroup takes a sequence's units kThreads at a time; the items' places are worked out
// once, a lane an item, kShort in a round.
// Short paths, the accepted ones of drafted tokens, are one round. Bound by its chain of loads (lengths and path, table, rows):
// 64 sequences of 5 kept tokens, 8 heads of 128, 4.4 us; two launches of the long form's kind would take 9. UP: of paths in
// several windows, the items that move up, rounds from the last, one after the other: 90000 of them, 8 heads of 128, 15 ms.
// Where there are none, as in every path without entries that are passed over, it ends at once.
constexpr int kShort = 64;

template <int D, bool UP>
__global__ __launch_bounds__(kThreads) void compact_short_kernel(const CompactArgs a) {
  constexpr int U = D / 16, kHeld = UP ? 32 : 8;
  __shared__ Place from[kShort], to[kShort];
  __shared__ int moved;
  if (UP && !*a.up) return;
  const int b = a.b0 + blockIdx.x, units = a.heads * U;
  const int last = UP ? max(min(a.counts[b], a.most) - 1, 0) / kShort * kShort : 0;
  for (int first = last; first >= 0; first -= kShort) {
    if (UP) __syncthreads();  // the last round's reads are done
    if (threadIdx.x < 64) {
      Place f = {-1, 0}, t = {-1, 0};
      int source = -1;
      const int i = first + (int)threadIdx.x;
      if (i < a.most) item_of(a, b, i, f, t, source);
      const bool on = f.page >= 0, rises = source < i;
      const uint64_t down = __ballot(on && !rises), up = __ballot(on && rises), below = (1ull << threadIdx.x) - 1;
      if (on && (rises || !UP)) {
        const int at = rises ? (UP ? 0 : __popcll(down)) + __popcll(up & ~below) - 1 : __popcll(down & below);
        from[at] = f;
        to[at] = t;
      }
      if (threadIdx.x == 0) moved = __popcll(UP ? up : up | down);
    }
    __syncthreads();
    const int n = moved;
    for (int id = blockIdx.y * kThreads + threadIdx.x; id < 2 * (units + a.heads); id += gridDim.y * kThreads) {
      const bool scale = id >= 2 * units;
      const int r = scale ? id - 2 * units : id;
      const bool second = r >= (scale ? a.heads : units);
      const int x = r - (second ? (scale ? a.heads : units) : 0);
      const Side& s = second ? a.v : a.k;
      const int head = scale ? x : x / U, u = scale ? 0 : x % U;
      const auto locate = [&](const Place& p) -> int64_t {
        const int64_t token = (int64_t)head * a.page + p.off;
        return scale ? p.page * s.scale_page + token : p.page * s.code_page + token * D + u * 16;
      };
      for (int i0 = 0; i0 < n; i0 += kHeld) {
        u32x4 held[kHeld];
        if (scale) {
#pragma unroll
          for (int j = 0; j < kHeld; ++j)
            if (i0 + j < n) held[j][0] = __float_as_uint(s.scales[locate(from[i0 + j])]);
#pragma unroll
          for (int j = 0; j < kHeld; ++j)
            if (i0 + j < n) s.scales[locate(to[i0 + j])] = __uint_as_float(held[j][0]);
        } else {
#pragma unroll
          for (int j = 0; j < kHeld; ++j)
            if (i0 + j < n) held[j] = ld16(s.codes + locate(from[i0 + j]));
#pragma unroll
          for (int j = 0; j < kHeld; ++j)
            if (i0 + j < n) *reinterpret_cast<u32x4*>(s.codes + locate(to[i0 + j])) = held[j];
        }
      }
    }
  }
}

// Long paths (contexts cut to the positions worth keeping) in windows of items, each in two launches: SAVE copies the items
// whose source is a place of the window (path[i] < w1) aside, then every item of the window moves, those from the copy. With
// several windows an item that moves up may have its source in one before: those are left to compact_short_kernel. All items
// of a launch are independent, so it fills the chip whatever the path; what lies past the window's places, as after a cut that
// drops more than it keeps, is read once. A workgroup takes kRows items of a sequence, for keys or values.
// Bound by memory: 8 contexts cut from 16384 to 4095 positions, 8 heads of 128, 85 MB moved, 25.0 us with 4.6 us of SAVE;
// the move is 4.1 TB/s, of rows of 128 bytes at a head's distance from each other. Eight loads a lane in flight instead of four
// take 29 to 31, non-temporal stores the same. Where most is copied aside its bytes move twice: as many positions of the same
// contexts, scattered, 51; all but 7 early ones 64, all but 1000 early ones 59.
constexpr int kRows = 32;
constexpr int kSavers = 16;  // workgroups of a sequence that look for what to copy aside

// Whether anything of a tile may be copied aside, by its first entry alone, for both launches: path ascends, so not if that is
// a position behind the window. An entry that is no position says nothing of those behind it.
__device__ __forceinline__ bool looked_at(const CompactArgs& a, int b, int i0) {
  const int32_t x = a.path[(int64_t)b * a.path_row + i0];
  return x < a.w1 || x >= (int64_t)a.starts[b + 1] - a.starts[b];
}

template <int D, bool SAVE>
__global__ __launch_bounds__(kThreads) void compact_long_kernel(const CompactArgs a) {
  constexpr int U = D / 16;
  __shared__ Place from[kRows], to[kRows];
  __shared__ int aside[kRows], any;
  __shared__ uint64_t ahead[kThreads / 64];
  const int tiles = (a.w1 - a.w0 + kRows - 1) / kRows, groups = SAVE ? min(tiles, kSavers) : tiles;
  const int seq = blockIdx.x / groups, b = a.b0 + seq, items = min(a.counts[b], a.w1);
  const auto move = [&](int i0, bool looked) {  // the tile that begins with item i0
    __syncthreads();
    if (threadIdx.x < 64) {
      Place f = {-1, 0}, t = {-1, 0};
      int source = -1;
      const int i = i0 + threadIdx.x;
      if (threadIdx.x < kRows && i < a.w1) item_of(a, b, i, f, t, source);
      if (a.up) {
        if (!SAVE && __ballot(f.page >= 0 && source < i) && threadIdx.x == 0)
          __hip_atomic_store(a.up, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (source < i) f.page = -1;
      }
      const bool kept = f.page >= 0 && looked && source < a.w1;
      if (SAVE && !kept) f.page = -1;
      const uint64_t on = __ballot(f.page >= 0);
      if (threadIdx.x < kRows) {
        from[threadIdx.x] = f;
        to[threadIdx.x] = t;
        aside[threadIdx.x] = kept;
      }
      if (threadIdx.x == 0) any = on != 0;
    }
    __syncthreads();
    if (!any) return;
    const Side& s = blockIdx.y ? a.v : a.k;
    // the copies' rows: [keys or values][sequence][item of the window][head]
    const int64_t row0 = ((int64_t)blockIdx.y * a.batch + seq) * (a.w1 - a.w0) + (i0 - a.w0);
    const int total = kRows * a.heads * U;
    const auto in_cache = [&](const Place& p, int head, int u) {
      return s.codes + p.page * s.code_page + ((int64_t)head * a.page + p.off) * D + u * 16;
    };
    const auto in_copy = [&](int r, int head, int u) { return a.saved + ((row0 + r) * a.heads + head) * D + u * 16; };
    const auto unit = [&](int id, int& r, int& head, int& u) {  // items of one head side by side
      u = id % U;
      r = id / U % kRows;
      head = id / (U * kRows);
    };
    for (int base = threadIdx.x; base < total; base += 4 * kThreads) {
      u32x4 held[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int r, head, u;
        unit(base + j * kThreads, r, head, u);
        if (base + j * kThreads >= total || from[r].page < 0) continue;
        held[j] = ld16_nt(!SAVE && aside[r] ? in_copy(r, head, u) : in_cache(from[r], head, u));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int r, head, u;
        unit(base + j * kThreads, r, head, u);
        if (base + j * kThreads >= total || from[r].page < 0) continue;
        *reinterpret_cast<u32x4*>(SAVE ? in_copy(r, head, u) : in_cache(to[r], head, u)) = held[j];
      }
    }
    for (int id = threadIdx.x; id < kRows * a.heads; id += kThreads) {
      const int r = id % kRows, head = id / kRows;
      if (from[r].page < 0) continue;
      float* const copy = a.saved_scales + (row0 + r) * a.heads + head;
      float* const old = s.scales + from[r].page * s.scale_page + (int64_t)head * a.page + from[r].off;
      float* const now = s.scales + to[r].page * s.scale_page + (int64_t)head * a.page + to[r].off;
      if (SAVE)
        *copy = *old;
      else
        *now = aside[r] ? *copy : *old;
    }
  };
  const int first = blockIdx.x - seq * groups;
  if (SAVE && a.up && a.w0 == 0 && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.up = 0;
  if constexpr (!SAVE) {
    const int i0 = a.w0 + first * kRows;
    if (i0 < items) move(i0, looked_at(a, b, i0));
  } else {  // a lane a tile looks which there are, then those one after the other
    for (int tile0 = first; tile0 < tiles; tile0 += groups * kThreads) {
      const int tile = tile0 + (int)threadIdx.x * groups, i0 = a.w0 + tile * kRows;
      const uint64_t on = __ballot(tile < tiles && i0 < items && looked_at(a, b, i0));
      __syncthreads();  // the last round's reads are done
      if ((threadIdx.x & 63) == 0) ahead[threadIdx.x >> 6] = on;
      __syncthreads();
#pragma unroll 1
      for (int w = 0; w < kThreads / 64; ++w)
#pragma unroll 1
        for (uint64_t left = ahead[w]; left; left &= left - 1)
          move(a.w0 + (tile0 + (w * 64 + __ffsll((unsigned long long)left) - 1) * groups) * kRows, true);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Which pages each sequence holds. refs[p] counts the block-table entries (and whoever else) that hold page p; 0 is free.
struct UpdateArgs {
  int32_t* refs;
  const int32_t *table, *lens, *want, *parents;
  int32_t *out, *granted, *src, *dst;
  int64_t table_row, pages;
  int batch, cols, page;
  int32_t *before, *begin;  // [batch] each: new pages asked for by the sequences before, and the first column of one's own
};

struct Row {
  int parent, kept, full, want;  // positions kept of the parent's, whole pages among them, positions asked for
  bool part;                     // a page of which a part is kept
};

__device__ __forceinline__ int clamp_len(const UpdateArgs& a, int32_t n) {
  const int64_t room = (int64_t)a.cols * a.page;
  return (int)(n < 0 ? 0 : n > room ? room : n);
}

__device__ __forceinline__ Row row_of(const UpdateArgs& a, int b) {
  Row r;
  r.parent = a.parents ? a.parents[b] : b;
  if (r.parent < 0 || r.parent >= a.batch) r.parent = -1;
  r.want = clamp_len(a, a.want[b]);
  r.kept = r.parent < 0 ? 0 : min(r.want, clamp_len(a, a.lens[r.parent]));
  r.full = r.kept / a.page;
  r.part = r.kept != r.full * a.page;
  return r;
}

__device__ __forceinline__ int page_at(const UpdateArgs& a, int b, int col) {  // -1: the cache has no such page
  const int32_t p = a.table[(int64_t)b * a.table_row + col];
  return p < 0 || p >= a.pages ? -1 : p;
}

__device__ __forceinline__ int32_t ref_load(const int32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A sequence a workgroup: it lets go of the pages it held, takes hold of the whole pages it keeps, and writes them into
// the new table. The page that it keeps a part of is let go of here; who may go on writing into it is decided once all have
// let go. Bound by its chain of loads and the atomics: 3.6 us for 64 sequences that keep what they have, 9 for 512 forks.
__global__ __launch_bounds__(kThreads) void update_hold_kernel(const UpdateArgs a) {
  const int b = blockIdx.x;
  const Row r = row_of(a, b);
  const int held = (clamp_len(a, a.lens[b]) + a.page - 1) / a.page;
  for (int c = threadIdx.x; c < a.cols; c += kThreads) {
    const int kept = c < r.full ? page_at(a, r.parent, c) : -1, own = c < held ? page_at(a, b, c) : -1;
    if (kept != own) {  // a page that it held and keeps, as forks of one prompt do, stays as it is
      if (kept >= 0) atomicAdd(a.refs + kept, 1);
      if (own >= 0) atomicSub(a.refs + own, 1);
    }
    a.out[(int64_t)b * a.cols + c] = kept;
  }
}

constexpr int kJoin = 1024;

constexpr int kLdsRows = 2048;  // sequences whose sums are searched in LDS; of more, in memory
constexpr int kScan = 8;        // pages a lane looks at in one round
constexpr int kRound = kJoin * kScan;
constexpr int32_t kClaim = INT32_MIN;

// Every atomic before it has been performed, for all lanes of the workgroup.
__device__ __forceinline__ void settle() {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
}

// One workgroup for what hangs on an order. A partly kept page that nobody holds any more goes to the lowest of the
// sequences that keep a part of it (each claims it, by an atomic minimum where another has); the others, and all that keep
// a part of a page somebody still holds, copy it to a new one. New pages are then asked for in the order of sequences and
// columns, and the k-th asked for is the k-th lowest free page: rounds of 8192 pages are counted into a list of the free
// ones, and a lane takes one that is asked for and searches whose it is in the sums of what the sequences ask for. Bound by
// its chain of loads and atomics, 7 to 9 us: a lane keeps what it knows of its first sequence, so that up to 1024 are read
// once, and the first round's counts come beside that: all that changes among them is what this kernel claims, which LDS
// remembers. Spread over workgroups it would wait for each of three steps by words in memory, about as long.
// That is with free pages among the first 8192. The search begins at page 0 and ends with the last page asked for, or with the
// pool: 2.8 us a round, so a pool whose low pages are all held costs its length: of 2^18 pages 93 us, of 2^20 358.
__global__ __launch_bounds__(kJoin) void update_grow_kernel(const UpdateArgs a) {
  __shared__ int sums[kJoin / 64];
  __shared__ int32_t lds_before[kLdsRows], lds_begin[kLdsRows], list[kRound];
  __shared__ uint8_t claimed[kRound];
  const bool fits = a.batch <= kLdsRows;
  const auto load_refs = [&](int64_t p0, i32x4 (&x)[2]) {  // past the last page: not 0
    const int64_t p = p0 + (int)threadIdx.x * kScan;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (p + 4 * h + 4 <= a.pages) {
        __builtin_memcpy(&x[h], a.refs + p + 4 * h, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[h][e] = p + 4 * h + e < a.pages ? a.refs[p + 4 * h + e] : 1;
      }
    }
  };
  i32x4 counts[2];
  load_refs(0, counts);
  *reinterpret_cast<uint64_t*>(claimed + threadIdx.x * kScan) = 0;
  struct Part {
    Row r;
    int page;  // of which a part is kept; -1: none, or one that the cache does not have
  };
  const auto read = [&](int b) {
    Part p;
    p.r = row_of(a, b);
    p.page = p.r.part ? page_at(a, p.r.parent, p.r.full) : -1;
    return p;
  };
  Part own{};
  if ((int)threadIdx.x < a.batch) own = read(threadIdx.x);
  const auto part = [&](int b) { return b < kJoin ? own : read(b); };
#pragma unroll 1
  for (int b = threadIdx.x; b < a.batch; b += kJoin) {
    const Part p = part(b);
    if (p.page < 0) continue;
    const int32_t n = atomicCAS(a.refs + p.page, 0, kClaim + b);
    if (n < 0 && n < kClaim + a.batch) atomicMin(a.refs + p.page, kClaim + b);
  }
  settle();
  int asked = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < a.batch; b0 += kJoin) {
    const int b = b0 + threadIdx.x;
    int need = 0, begin = 0;
    bool copies = false;
    if (b < a.batch) {
      const Part p = part(b);
      const bool takes = p.page >= 0 && ref_load(a.refs + p.page) == kClaim + b;
      if (takes) {
        a.out[(int64_t)b * a.cols + p.r.full] = p.page;
        if (p.page < kRound) claimed[p.page] = 1;
      }
      copies = p.page >= 0 && !takes;
      begin = p.r.full + (p.r.part && !copies ? 1 : 0);  // a part of no page stays one of none
      need = max((p.r.want + a.page - 1) / a.page - begin, 0);
    }
    int total;
    const int off = asked + block_before<kJoin>(need, sums, total);
    asked += total;
    if (b < a.batch) {
      a.begin[b] = begin;
      a.before[b] = off;
      if (fits) lds_begin[b] = begin, lds_before[b] = off;
      a.src[b] = copies ? -2 : -1;  // until it is known whether there is a page
    }
  }
  settle();
#pragma unroll 1
  for (int b = threadIdx.x; b < a.batch; b += kJoin) {  // claims become holders, now that all have read them
    const Part p = part(b);
    if (p.page >= 0 && a.src[b] != -2) __hip_atomic_store(a.refs + p.page, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (a.pages > kRound) settle();
  const int32_t* const before = fits ? lds_before : a.before;
  const int32_t* const begin = fits ? lds_begin : a.begin;
  int found = 0;
#pragma unroll 1
  for (int64_t p0 = 0; p0 < a.pages && found < asked; p0 += kRound) {
    if (p0 > 0) {
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");  // the claims among them
      load_refs(p0, counts);
    }
    const int at = threadIdx.x * kScan;
    uint32_t free = 0;
#pragma unroll
    for (int j = 0; j < kScan; ++j)
      if (counts[j / 4][j % 4] == 0 && (p0 > 0 || !claimed[at + j])) free |= 1u << j;
    int total;
    int k = block_before<kJoin>(__popc(free), sums, total);
#pragma unroll 1
    for (; free; ++k, free &= free - 1) list[k] = at + __ffs(free) - 1;
    __syncthreads();
    const int taken = min(total, asked - found);
#pragma unroll 1
    for (int i = threadIdx.x; i < taken; i += kJoin) {
      const int64_t page = p0 + list[i];
      int lo = 0, hi = a.batch;  // the last sequence whose first new page is this one or before
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= found + i)
          lo = mid;
        else
          hi = mid;
      }
      a.out[(int64_t)lo * a.cols + begin[lo] + found + i - before[lo]] = (int)page;
      __hip_atomic_store(a.refs + page, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    found += total;
  }
  settle();
#pragma unroll 1
  for (int b = threadIdx.x; b < a.batch; b += kJoin) {
    const Part p = part(b);
    const int first = begin[b], got = found - before[b];
    const int need = max((p.r.want + a.page - 1) / a.page - first, 0);
    a.granted[b] = got >= need ? p.r.want : min(p.r.want, (first + max(got, 0)) * a.page);
    const bool copies = a.src[b] == -2 && got > 0;  // its first new page is the copy
    a.src[b] = copies ? p.page : -1;
    a.dst[b] = copies ? a.out[(int64_t)b * a.cols + first] : -1;
  }
}

}  // namespace aklr

using namespace aklr;

namespace {

bool side_ok(const void* codes, const void* scales, int64_t code_page, int64_t scale_page, int64_t kv_heads,
             int64_t head_dim, int64_t page) {
  return codes && scales && aklr_aligned16(codes) && aklr_aligned16(scales) && code_page >= kv_heads * page * head_dim &&
         scale_page >= kv_heads * page && code_page % 16 == 0 && scale_page % 4 == 0;
}

bool shape_ok(int64_t pages, int64_t page, int64_t kv_heads, int64_t head_dim) {
  return (head_dim == 64 || head_dim == 128 || head_dim == 256) && page >= 16 && page <= 1024 && page % 16 == 0 &&
         kv_heads >= 1 && kv_heads <= 1024 && pages >= 1 && pages * page <= 0x7FFFFFFF;
}

// How a compaction goes: items of a window and sequences of a launch.
struct Windows {
  int64_t items, sequences, bytes;
};
constexpr int64_t kSaveBytes = 128 << 20;

Windows windows_of(int64_t batch, int64_t most, int64_t kv_heads, int64_t head_dim) {
  if (most <= kShort || batch < 1) return {most, batch, 0};
  const int64_t item = 2 * kv_heads * (head_dim + 4);  // at most 520 KiB
  const int64_t fit = kSaveBytes / item;               // at least 252
  if (most > fit) {  // several windows, and behind their copies whether items move up
    const int64_t items = (fit - 1) / kRows * kRows;
    return {items, 1, (items + 1) * item};
  }
  const int64_t items = most;
  int64_t sequences = fit / items;
  const int64_t tiles = (items + kRows - 1) / kRows;
  if (sequences > kMostGroups / 2 / tiles) sequences = kMostGroups / 2 / tiles;
  if (sequences > batch) sequences = batch;
  return {items, sequences, sequences * items * item};
}

template <int D>
int compact(CompactArgs a, int64_t batch, uint8_t* ws, hipStream_t stream) {
  const Windows w = windows_of(batch, a.most, a.heads, D);
  const unsigned in_order = (unsigned)((2ll * a.heads * (D / 16 + 1) + kThreads - 1) / kThreads);
  if (a.most <= kShort) {
    a.b0 = 0;
    a.batch = (int)batch;
    hipLaunchKernelGGL((compact_short_kernel<D, false>), dim3((unsigned)batch, in_order), dim3(kThreads), 0, stream, a);
    AKLR_LAUNCH_CHECK();
    return AKLR_OK;
  }
  if (w.items < a.most) a.up = reinterpret_cast<int32_t*>(ws + w.items * 2 * a.heads * (D + 4));
  for (int64_t b0 = 0; b0 < batch; b0 += w.sequences) {
    a.b0 = (int)b0;
    a.batch = (int)(batch - b0 < w.sequences ? batch - b0 : w.sequences);
    for (int64_t w0 = 0; w0 < a.most; w0 += w.items) {
      a.w0 = (int)w0;
      a.w1 = (int)(a.most - w0 < w.items ? a.most : w0 + w.items);
      a.saved = ws;
      a.saved_scales = reinterpret_cast<float*>(ws + 2ll * a.batch * (a.w1 - a.w0) * a.heads * D);
      const int tiles = (a.w1 - a.w0 + kRows - 1) / kRows, savers = tiles < kSavers ? tiles : kSavers;
      hipLaunchKernelGGL((compact_long_kernel<D, true>), dim3((unsigned)(a.batch * savers), 2), dim3(kThreads), 0, stream, a);
      AKLR_LAUNCH_CHECK();
      hipLaunchKernelGGL((compact_long_kernel<D, false>), dim3((unsigned)(a.batch * tiles), 2), dim3(kThreads), 0, stream, a);
      AKLR_LAUNCH_CHECK();
    }
    if (a.up) {
      hipLaunchKernelGGL((compact_short_kernel<D, true>), dim3((unsigned)a.batch, in_order), dim3(kThreads), 0, stream, a);
      AKLR_LAUNCH_CHECK();
    }
  }
  return AKLR_OK;
}

}  // namespace

extern "C" int aklr_kv_cache_copy_pages_fp8(void* k_codes, void* v_codes, float* k_scales, float* v_scales, int64_t k_page,
                                            int64_t v_page, int64_t ks_page, int64_t vs_page, const void* src,
                                            const void* dst, int indices_64, int64_t count, int64_t kv_heads,
                                            int64_t head_dim, int64_t pages, int64_t page_size, hipStream_t stream) {
  if (!shape_ok(pages, page_size, kv_heads, head_dim) || count < 0 || count > 0x7FFFFFFF) return AKLR_ERR_INVALID_ARGUMENT;
  if (!side_ok(k_codes, k_scales, k_page, ks_page, kv_heads, head_dim, page_size) ||
      !side_ok(v_codes, v_scales, v_page, vs_page, kv_heads, head_dim, page_size))
    return AKLR_ERR_INVALID_ARGUMENT;
  if (count == 0) return AKLR_OK;
  if (!src || !dst) return AKLR_ERR_INVALID_ARGUMENT;
  const Side k = {static_cast<uint8_t*>(k_codes), k_scales, k_page, ks_page};
  const Side v = {static_cast<uint8_t*>(v_codes), v_scales, v_page, vs_page};
  const int64_t code_units = kv_heads * page_size * head_dim / 16, scale_units = kv_heads * page_size / 4;
  const int64_t chunks = (2 * (code_units + scale_units) + kCopyUnits - 1) / kCopyUnits;
  for (int64_t first = 0; first < count * chunks; first += kMostGroups) {
    const int64_t groups = count * chunks - first < kMostGroups ? count * chunks - first : kMostGroups;
    hipLaunchKernelGGL(copy_kernel, dim3((unsigned)groups), dim3(kThreads), 0, stream, k, v, src, dst, indices_64, pages,
                       (int)code_units, (int)scale_units, (int)chunks, first);
    AKLR_LAUNCH_CHECK();
  }
  return AKLR_OK;
}

extern "C" size_t aklr_kv_cache_compact_fp8_workspace_bytes(int64_t batch, int64_t most, int64_t kv_heads, int64_t head_dim) {
  if (batch < 1 || most < 1 || kv_heads < 1 || kv_heads > 1024 || head_dim < 1 || head_dim > 256) return 0;
  return (size_t)windows_of(batch, most, kv_heads, head_dim).bytes;
}

extern "C" int aklr_kv_cache_compact_fp8(void* k_codes, void* v_codes, float* k_scales, float* v_scales, int64_t k_page,
                                         int64_t v_page, int64_t ks_page, int64_t vs_page, const int32_t* block_table,
                                         int64_t table_stride, int64_t table_cols, const int32_t* seq_lens,
                                         const int32_t* starts, const int32_t* path, int64_t path_stride, int64_t most,
                                         const int32_t* counts, int64_t batch, int64_t kv_heads, int64_t head_dim,
                                         int64_t pages, int64_t page_size, void* workspace, size_t workspace_bytes,
                                         hipStream_t stream) {
  if (!shape_ok(pages, page_size, kv_heads, head_dim) || batch < 0 || batch > 65536 || most < 0 || most > (1 << 28) ||
      table_cols < 0 || table_cols * page_size > (1 << 28) || table_stride < table_cols || path_stride < most)
    return AKLR_ERR_INVALID_ARGUMENT;
  if (!side_ok(k_codes, k_scales, k_page, ks_page, kv_heads, head_dim, page_size) ||
      !side_ok(v_codes, v_scales, v_page, vs_page, kv_heads, head_dim, page_size))
    return AKLR_ERR_INVALID_ARGUMENT;
  if (batch == 0 || most == 0 || table_cols == 0) return AKLR_OK;
  if (!block_table || !seq_lens || !starts || !path || !counts) return AKLR_ERR_INVALID_ARGUMENT;
  const size_t bytes = aklr_kv_cache_compact_fp8_workspace_bytes(batch, most, kv_heads, head_dim);
  if (bytes && (!workspace || !aklr_aligned16(workspace) || workspace_bytes < bytes)) return AKLR_ERR_WORKSPACE;
  CompactArgs a{};
  a.k = {static_cast<uint8_t*>(k_codes), k_scales, k_page, ks_page};
  a.v = {static_cast<uint8_t*>(v_codes), v_scales, v_page, vs_page};
  a.table = block_table;
  a.lens = seq_lens;
  a.starts = starts;
  a.path = path;
  a.counts = counts;
  a.table_row = table_stride;
  a.path_row = path_stride;
  a.table_cols = (int)table_cols;
  a.heads = (int)kv_heads;
  a.page = (int)page_size;
  a.most = (int)most;
  a.pages = pages;
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  return head_dim == 64    ? compact<64>(a, batch, ws, stream)
         : head_dim == 128 ? compact<128>(a, batch, ws, stream)
                           : compact<256>(a, batch, ws, stream);
}

extern "C" size_t aklr_kv_cache_update_pages_workspace_bytes(int64_t batch) {
  return batch < 1 ? 0 : (size_t)(8 * ((batch + 3) / 4 * 4));
}

extern "C" int aklr_kv_cache_update_pages(int32_t* page_refs, int64_t pages, const int32_t* block_table, int64_t table_stride,
                                          int64_t table_cols, const int32_t* lens, const int32_t* new_lens,
                                          const int32_t* parents, int64_t batch, int64_t page_size, int32_t* new_table,
                                          int32_t* granted, int32_t* src, int32_t* dst, void* workspace,
                                          size_t workspace_bytes, hipStream_t stream) {
  if (batch < 0 || batch > 65536 || pages < 1 || page_size < 1 || pages * page_size > 0x7FFFFFFF || table_cols < 0 ||
      table_cols * page_size > (1 << 28) || table_stride < table_cols || batch * table_cols > 0x7FFFFFFF)
    return AKLR_ERR_INVALID_ARGUMENT;
  if (batch == 0) return AKLR_OK;
  if (!page_refs || !lens || !new_lens || !granted || !src || !dst || (table_cols && (!block_table || !new_table)))
    return AKLR_ERR_INVALID_ARGUMENT;
  const size_t bytes = aklr_kv_cache_update_pages_workspace_bytes(batch);
  if (!workspace || !aklr_aligned16(workspace) || workspace_bytes < bytes) return AKLR_ERR_WORKSPACE;
  UpdateArgs a{};
  a.refs = page_refs;
  a.table = block_table;
  a.lens = lens;
  a.want = new_lens;
  a.parents = parents;
  a.out = new_table;
  a.granted = granted;
  a.src = src;
  a.dst = dst;
  a.table_row = table_stride;
  a.pages = pages;
  a.batch = (int)batch;
  a.cols = (int)table_cols;
  a.page = (int)page_size;
  a.before = static_cast<int32_t*>(workspace);
  a.begin = a.before + (batch + 3) / 4 * 4;
  hipLaunchKernelGGL(update_hold_kernel, dim3((unsigned)batch), dim3(kThreads), 0, stream, a);
  AKLR_LAUNCH_CHECK();
  hipLaunchKernelGGL(update_grow_kernel, dim3(1), dim3(kJoin), 0, stream, a);
  AKLR_LAUNCH_CHECK();
  return AKLR_OK;
}

AKLR_SCALAR_FP32_END
