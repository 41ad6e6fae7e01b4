// Which drafted tokens stand against the target's probabilities, and the token that follows them. gfx950 only.
//
// A sequence's query tokens are a tree: the first is its last token that stands, the others are drafts, each after its
// parent. At a node with target row p and draft row q the children are tried in their order, from W = p, S = 1, A = 0:
//   child x stands if u * S * q(x) < W(x), and the search goes on at it;
//   else A += S, W = max(p - A q, 0), S = sum(W)           (max(max(p - a q, 0) - s q, 0) = max(p - (a + s) q, 0))
// and without draft rows (drafts that were certain) if u * S < W(x), else S -= W(x), W(x) = 0. Where no child stands, the
// next token is the least v with W(0) + ... + W(v) > u' * sum(W). If the drafts were drawn from q, the tokens that come out
// are distributed as the target's own.
//
// Bound by memory and, for few sequences, by its chain of loads: the whole rows p and q of one node a sequence, and once
// more for each rejection that another child follows. Everything is in 64 bits: which token is drawn hangs on a running sum
// over the vocabulary, and 32 bits would move some of its borders with the order of the additions; in 64 they move by some
// 2^-50 of the row's sum. The order is set by the sizes, not by who arrives when. The sums are bound by the loads all the same
// (figures at plan_verify).
#include "common.h"
#include "scan.h"

AKLR_SCALAR_FP32_BEGIN

namespace aklr {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kMost = 1024;  // query tokens of a sequence
constexpr int kUnit = 512;   // values of a row that one wave adds up to a partial sum: 8 a lane
constexpr int kGroup = 2;    // units whose loads a wave has in flight
constexpr int kNone = 0x7FFFFFFF;

enum Status : int { kRefused, kEnd, kWholeRow, kDone };

struct State {  // of a sequence's search, from one launch to the next
  int node, count, next, status;
  double a, s;  // A; S before the last rejection is in A
};

struct VerifyArgs {
  const void *target, *draft;
  int64_t target_row, draft_row;
  const void* tokens;
  const int32_t *parents, *starts;
  const float *accept, *sample;
  void* out;
  int32_t *path, *counts;
  uint64_t* words;
  State* states;
  double* partial;  // [batch][units]
  int64_t total;    // tokens in all
  int vocab, units, most, batch, token64, splits, per_wave;
};

template <typename T>
__device__ __forceinline__ float widen(T x);
template <>
__device__ __forceinline__ float widen<float>(float x) { return x; }
template <>
__device__ __forceinline__ float widen<uint16_t>(uint16_t x) { return bf16_lo(x); }
template <>
__device__ __forceinline__ float widen<_Float16>(_Float16 x) { return (float)x; }

// Entries that are no probabilities (negative, NaN, infinite) count as zero.
__device__ __forceinline__ float proper(float x) {
  constexpr int kPositiveFinite = 0x180;  // subnormal, normal
  return __builtin_amdgcn_classf(x, kPositiveFinite) ? x : 0.0f;
}

__device__ __forceinline__ double unit_number(float u) {
  return u > 0.0f ? (double)fminf(u, 0x1.fffffep-1f) : 0.0;
}

__device__ __forceinline__ double weight(float p, float q, double a) {  // no contraction: the product of a = 1 is exact
  return fmax(__dsub_rn((double)p, __dmul_rn(a, (double)q)), 0.0);
}

// Eight values of a row. Rows start at any multiple of their element: the loads are 16 bytes wide whatever the alignment.
template <typename T>
struct Eight {
  u32x4 x[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(x, p, sizeof(x)); }
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (sizeof(T) == 4) {
      return proper(__uint_as_float(x[e / 4][e % 4]));
    } else {
      const uint16_t h = (uint16_t)(x[0][e / 2] >> (e % 2 * 16));
      return proper(widen<T>(__builtin_bit_cast(T, h)));
    }
  }
};

struct Drafts {  // a sequence's tokens, in LDS
  int parent[kMost], token[kMost];
  float u[kMost], p[kMost], q[kMost];
  int gone[kMost];  // tokens refused at the node, where drafts are certain
};

template <typename T, bool CHAIN, bool SURE>
__global__ __launch_bounds__(kThreads, 4) void verify_kernel(const VerifyArgs a, const int round, const int rounds) {
  __shared__ Drafts d;
  __shared__ State st;
  __shared__ int gones;
  __shared__ double wave_total[kWaves];
  __shared__ unsigned slot;
  __shared__ int again, first_unit[kWaves], last_unit[kWaves];
  __shared__ double unit_before[kWaves];
  const int seq = (int)(blockIdx.x / (unsigned)a.splits), split = (int)(blockIdx.x % (unsigned)a.splits);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t seen = 0;
  if (a.splits > 1 && threadIdx.x == 0) seen = splitk_peek(a.words + seq);

  const int64_t lo = a.starts[seq], hi = a.starts[seq + 1] < a.total ? a.starts[seq + 1] : a.total;
  const int n = lo < 0 || hi <= lo ? 0 : (int)(hi - lo < a.most ? hi - lo : a.most);
  if (n == 0) {  // no such sequence: nothing stands, nothing follows
    if (round == 0 && split == 0) {
#pragma unroll 1
      for (int i = threadIdx.x; i < a.most; i += kThreads) {
        a.path[(int64_t)seq * a.most + i] = -1;
        if (a.token64)
          static_cast<int64_t*>(a.out)[(int64_t)seq * a.most + i] = -1;
        else
          static_cast<int32_t*>(a.out)[(int64_t)seq * a.most + i] = -1;
      }
      if (threadIdx.x == 0) a.counts[seq] = 0;
    }
    return;
  }
  const auto target = [&](int node) { return static_cast<const T*>(a.target) + (lo + node) * a.target_row; };
  const auto draft = [&](int node) { return static_cast<const T*>(a.draft) + (lo + node) * a.draft_row; };
  const auto token_at = [&](int i) {
    return a.token64 ? static_cast<const int64_t*>(a.tokens)[lo + i] : (int64_t) static_cast<const int32_t*>(a.tokens)[lo + i];
  };
  const auto put_token = [&](int i, int64_t x) {
    if (a.token64)
      static_cast<int64_t*>(a.out)[(int64_t)seq * a.most + i] = x;
    else
      static_cast<int32_t*>(a.out)[(int64_t)seq * a.most + i] = (int32_t)x;
  };

  // The sequence's drafts into LDS, with what the two rows of their parents hold for them.
  const auto gather = [&]() {
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int64_t x = token_at(i);
      int parent = CHAIN ? i - 1 : a.parents[lo + i];
      if (i == 0 || x < 0 || x >= a.vocab || parent < 0 || parent >= i) parent = -1;  // never tried
      d.parent[i] = parent;
      d.token[i] = (int)x;
      d.u[i] = a.accept[lo + i];
      d.p[i] = parent < 0 ? 0.0f : proper(widen<T>(target(parent)[x]));
      if (!SURE) d.q[i] = parent < 0 ? 0.0f : proper(widen<T>(draft(parent)[x]));
    }
  };
  // The first draft from `i` on that follows `node`, or n. One wave.
  const auto child = [&](int node, int i) {
#pragma unroll 1
    for (int base = i & ~63; base < n; base += 64) {
      const int j = base + lane;
      const uint64_t on = __ballot(j >= i && j < n && d.parent[j] == node);
      if (on) return base + __ffsll((unsigned long long)on) - 1;
    }
    return n;
  };

  const float chance = a.sample[seq];
  bool searches = round == 0, writes = split == 0, alone = false;
  if (searches) gather();
  if (threadIdx.x == 0) {
    st = round == 0 ? State{0, 1, 1, kEnd, 0.0, 1.0} : a.states[seq];
    gones = 0;
    if (searches && writes) a.path[(int64_t)seq * a.most] = 0;
  }
  __syncthreads();
  if (st.status == kDone) return;
  double* const partial = a.partial + (int64_t)seq * a.units;
  int from = (split * kWaves + wave) * a.per_wave, step = 1, to = min(from + a.per_wave, a.units);
  double total = 0.0, before = 0.0, mine = 0.0;  // of the row's sums; of the units before this lane's; of this lane's
  const int per = (a.units + kThreads - 1) / kThreads, u0 = threadIdx.x * per, u1 = min(u0 + per, a.units);

  // The eight values of lane `l` of a unit, and how many of them belong to the lane before: the row's last ones are read from
  // eight before its end.
  const auto place = [&](int unit, int& skip) {
    const int v = unit * kUnit + lane * 8, v0 = min(v, a.vocab - 8);
    skip = v - v0;
    return v0;
  };
  const auto fetch = [&](int v, Eight<T>& p, Eight<T>& q) {
    p.load(target(st.node) + v);
    if (!SURE && st.a != 0.0) q.load(draft(st.node) + v);
  };
  const auto weigh = [&](int v, int skip, const Eight<T>& p, const Eight<T>& q, double (&w)[8]) {
    const double by = st.a;
    if (!SURE && by != 0.0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = weight(p[e], q[e], by);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = p[e];
    }
    if (skip > 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < skip) w[e] = 0.0;
    }
    if (SURE && st.status != kWholeRow)
#pragma unroll 1
      for (int g = 0; g < gones; ++g) {
        const int at = d.gone[g] - v;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (at == e) w[e] = 0.0;
      }
  };

  for (;;) {
    bool sums = true;  // whether the row has to be added up
    if (searches) {
      if (CHAIN && wave == 0) {  // every draft is its node's only one: all are tried at once, up to the first that falls
        int last = n - 1;  // the node at which the chain ends, and whether a draft after it was refused
        bool falls = false;
#pragma unroll 1
        for (int base = 0; base < n; base += 64) {
          const int j = base + lane;
          const bool on = j > 0 && j < n, tried = on && d.parent[j] >= 0;
          const double u = on ? unit_number(d.u[j]) : 0.0, p = on ? d.p[j] : 0.0, q = SURE || !on ? 1.0 : d.q[j];
          const bool stands = tried && __dmul_rn(u, q) < p;
          const uint64_t ends = __ballot(on && !stands), refused = __ballot(tried);
          const int end = ends ? base + __ffsll((unsigned long long)ends) - 1 : n;
          if (writes && on && j < end) {
            a.path[(int64_t)seq * a.most + j] = j;
            put_token(j - 1, d.token[j]);
          }
          if (ends) {
            last = end - 1;
            falls = refused >> (end - base) & 1;
            break;
          }
        }
        if (lane == 0) {
          st.node = last;
          st.count = last + 1;
          st.a = !SURE && falls ? 1.0 : 0.0;
          if (SURE && falls) {
            d.gone[0] = d.token[last + 1];
            gones = 1;
          }
          again = true;
        }
      }
      if (!CHAIN && wave == 0) {  // goes on until a row has to be added up, for a rejection or for the token that follows
        State s = st;
        int refused = gones;
        bool moved = round == 0 && !alone;
        for (;;) {
          const int j = child(s.node, s.next);
          if (j >= n) {
            s.status = kEnd;
            break;
          }
          moved = true;
          s.next = j + 1;
          const double u = __dmul_rn(unit_number(d.u[j]), s.s);
          double w;
          if (SURE) {
            bool twice = false;
#pragma unroll 1
            for (int g = lane; g < refused; g += 64) twice |= d.gone[g] == d.token[j];
            w = __ballot(twice) ? 0.0 : (double)d.p[j];
          } else {
            w = weight(d.p[j], d.q[j], s.a);
          }
          if ((SURE ? u : __dmul_rn(u, (double)d.q[j])) < w) {
            if (writes && lane == 0) {
              a.path[(int64_t)seq * a.most + s.count] = j;
              put_token(s.count - 1, d.token[j]);
            }
            s.node = j;
            s.count += 1;
            s.a = 0.0;
            s.s = 1.0;
            refused = 0;
          } else if (SURE) {
            s.s -= w;
            if (lane == 0) d.gone[refused] = d.token[j];
            refused += 1;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          } else {
            s.a += s.s;
            s.status = kRefused;
            break;
          }
        }
        if (lane == 0) {
          st = s;
          gones = refused;
          again = moved;
        }
      }
      __syncthreads();
      sums = again;  // not if there was no other draft to try: the row's sums are there
      if (sums && alone && round + 1 < rounds) {  // the next launch adds it up
        if (threadIdx.x == 0) a.states[seq] = st;
        return;
      }
    }
    if (sums) {
      // Units kGroup at a time: all their loads, then their sums, which the lanes add up together: a half of them the one,
      // the other half the other.
      bool first = true;
#pragma unroll 1
      for (int u = from; u < to || first; u += kGroup * step) {
        Eight<T> p[kGroup], q[kGroup];
        int skip[kGroup], v[kGroup];
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
          v[j] = place(min(u + j * step, a.units - 1), skip[j]);
          fetch(v[j], p[j], q[j]);
        }
        if (first && round != 0 && !alone) gather();  // beside the loads; the workgroup that goes on with the search needs it
        first = false;
        double sum[kGroup];
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
          double w[8];
          weigh(v[j], skip[j], p[j], q[j], w);
          sum[j] = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
        }
        static_assert(kGroup == 2, "the exchange below");
        const bool upper = lane >= 32;
        const double all = sum_upto<false>((upper ? sum[1] : sum[0]) + __shfl_xor(upper ? sum[0] : sum[1], 32, 64));
        const int at = u + (lane >> 5) * step;
        if ((lane & 31) == 31 && at < to) __hip_atomic_store(partial + at, all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      if (!alone && a.splits > 1 && !splitk_arrive(a.words + seq, seen, a.splits, &slot)) return;
      // the last workgroup of the sequence: the sums of the units in their order
      alone = writes = true;
      from = wave, step = kWaves, to = a.units;
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      mine = 0.0;
#pragma unroll 1
      for (int u = u0; u < u1; ++u) mine += __hip_atomic_load(partial + u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const double upto = sum_upto<true>(mine);
      if (lane == 63) wave_total[wave] = upto;
      __syncthreads();
      total = 0.0;
      before = upto - mine;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        if (w == wave) before += total;
        total += wave_total[w];
      }
    }
    searches = !CHAIN && !SURE && st.status == kRefused;
    const bool nothing = !(total > 0.0) && st.status == kEnd;
    __syncthreads();
    if (!searches && !nothing) break;
    if (threadIdx.x == 0) {
      if (searches) {
        st.s = total;  // what the rejection leaves, for the node's next draft
      } else {  // nothing is left of the row: the target's own
        st.status = kWholeRow;
        st.a = 0.0;
      }
    }
    __syncthreads();
  }

  // the unit in which the running sum passes the number, then the value; the last that weighs if rounding takes the last step
  const double level = unit_number(chance) * total;
  const int count = st.count;
  if (total > 0.0) {
    int found = kNone, end = -1;
    double run = before, found_before = 0.0;
#pragma unroll 1
    for (int u = u0; u < u1; ++u) {
      const double x = per == 1 ? mine : __hip_atomic_load(partial + u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (x > 0.0) {
        end = u;
        if (found == kNone && run + x > level) {
          found = u;
          found_before = run;
        }
      }
      run += x;
    }
    const uint64_t on = __ballot(found != kNone), any = __ballot(end >= 0);
    if (on ? lane == __ffsll((unsigned long long)on) - 1 : any && lane == 63 - __clzll((long long)any)) {
      first_unit[wave] = found;
      last_unit[wave] = end;
      unit_before[wave] = found_before;
    } else if (!any && lane == 0) {
      first_unit[wave] = kNone;
      last_unit[wave] = -1;
    }
    __syncthreads();
    int unit = -1;
    double sum = -__builtin_inf();
#pragma unroll
    for (int w = kWaves - 1; w >= 0; --w) {
      if (unit < 0) unit = last_unit[w];
    }
#pragma unroll
    for (int w = kWaves - 1; w >= 0; --w) {
      if (first_unit[w] != kNone) {
        unit = first_unit[w];
        sum = unit_before[w];
      }
    }
    if (wave == 0) {
      double w[8];
      Eight<T> p, q;
      int skip;
      const int v = place(unit, skip);
      fetch(v, p, q);
      weigh(v, skip, p, q, w);
      const double own = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      sum += sum_upto<true>(own) - own;
      int pick = kNone, final = -1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum += w[e];
        if (w[e] > 0.0) {
          final = v + e;
          if (pick == kNone && sum > level) pick = v + e;
        }
      }
      const uint64_t passed = __ballot(pick != kNone), weighs = __ballot(final >= 0);
      pick = passed ? __shfl(pick, __ffsll((unsigned long long)passed) - 1, 64)
                    : __shfl(final, 63 - __clzll((long long)weighs), 64);
      if (lane == 0) put_token(count - 1, pick);
    }
  } else if (threadIdx.x == 0) {
    put_token(count - 1, -1);
  }
#pragma unroll 1
  for (int i = count + threadIdx.x; i < a.most; i += kThreads) {
    a.path[(int64_t)seq * a.most + i] = -1;
    put_token(i, -1);
  }
  if (threadIdx.x == 0) {
    a.counts[seq] = count;
    if (rounds > 1) a.states[seq].status = kDone;
  }
}

}  // namespace aklr

using namespace aklr;

namespace {

constexpr int64_t kAtOnce = 512, kMostSplits = 16;
constexpr int kRounds = 4;

struct Plan {
  int units, splits, per_wave, rounds;
};

// How many workgroups share a row: one unit a wave while that makes no more workgroups than run at once (two of 512 lanes a
// CU), and at most 16: they arrive by atomics on one word, which wait for each other. Only trees whose drafts have rows need
// more than one sum of a row a sequence; they get up to four launches for it, and what is left after those the last workgroup
// does alone, at the rate of one CU (15 us for two rows of 128003 floats). Measured, fp32, us (both sides of each choice):
// - 16 trees of 33 tokens, vocabulary 128003: 33 with 16 workgroups a row; 44 with 4, 38 with 8, 76 with 32. 64 chains of
//   8, vocabulary 131072: 18.2 with any of them, 67 MB of rows at 3.7 TB/s. 4 chains of 5, vocabulary 32000: 8.1.
// - the same trees in 3 launches 42, 4: 30 to 33, 5: 36, 8: 36. A sequence adds up 1.6 rows at the mean, 3 or 4 at the most; a
//   launch that finds its sequences done takes 1.3. Chosen for trees like these; where many siblings fall one after the other,
//   each past the fourth takes 15 to 20: 16 roots of 4 siblings 33 to 37, of 8 (all fall in some) 82 to 119, of 20 142 to 375.
// - drafts without rows take one launch whatever falls: the same trees 12, 64 chains of 8 15.8, 4 chains of 5 8.4.
// - four units' loads in flight a wave instead of two no longer fit the registers.
// What bounds a call of few sequences is its chain of dependent loads, starts, then parents and tokens, then what the rows hold
// for them, then the rows, at 0.8 to 2 us each, and the 64-bit tail: a lone wave issues a vector instruction every five cycles.
Plan plan_verify(int64_t batch, int64_t vocab, bool chain, bool sure, int64_t most) {
  Plan p;
  p.units = (int)((vocab + kUnit - 1) / kUnit);
  int64_t splits = (p.units + kWaves - 1) / kWaves;
  const int64_t room = batch < kAtOnce ? kAtOnce / batch : 1;
  if (splits > room) splits = room;
  if (splits > kMostSplits) splits = kMostSplits;
  p.per_wave = (int)((p.units + splits * kWaves - 1) / (splits * kWaves));
  p.splits = (int)((p.units + p.per_wave * kWaves - 1) / (p.per_wave * kWaves));
  p.rounds = chain || sure || most <= 2 ? 1 : most <= kRounds ? (int)most - 1 : kRounds;
  return p;
}

struct Layout {
  size_t states, partial, bytes;
};
Layout layout_of(int64_t batch, int64_t units) {
  Layout l;
  l.states = (size_t)(8 * ((batch + 1) / 2 * 2));
  l.partial = l.states + sizeof(State) * (size_t)batch;
  l.bytes = l.partial + 8 * (size_t)(batch * units);
  return l;
}

bool sizes_ok(int64_t batch, int64_t vocab, int64_t most) {
  return batch >= 1 && batch <= 65536 && vocab >= 8 && vocab <= (1 << 24) && most >= 1 && most <= kMost;
}

}  // namespace

extern "C" size_t aklr_verify_drafts_workspace_bytes(int64_t batch, int64_t vocab, int64_t most) {
  return sizes_ok(batch, vocab, most) ? layout_of(batch, (vocab + kUnit - 1) / kUnit).bytes : 0;
}

extern "C" int aklr_verify_drafts(const void* target_probs, int64_t target_stride, const void* draft_probs,
                                  int64_t draft_stride, int64_t tokens, int64_t vocab, const void* draft_tokens,
                                  int tokens_64, const int32_t* parents, const int32_t* starts,
                                  const float* accept_uniforms, const float* sample_uniforms, int64_t batch, int64_t most,
                                  void* out_tokens, int32_t* path, int32_t* counts, int dtype, void* workspace,
                                  size_t workspace_bytes, hipStream_t stream) {
  if (dtype < AKLR_OUT_BF16 || dtype > AKLR_F32) return AKLR_ERR_UNSUPPORTED;
  if (batch == 0) return AKLR_OK;
  if (!sizes_ok(batch, vocab, most) || tokens < 0 || tokens > 0x7FFFFFFF || target_stride < vocab ||
      (draft_probs && draft_stride < vocab))
    return AKLR_ERR_INVALID_ARGUMENT;
  if (!starts || !sample_uniforms || !out_tokens || !path || !counts ||
      (tokens && (!target_probs || !draft_tokens || !accept_uniforms)))
    return AKLR_ERR_INVALID_ARGUMENT;
  const bool chain = !parents, sure = !draft_probs;
  const Plan p = plan_verify(batch, vocab, chain, sure, most);
  const Layout l = layout_of(batch, p.units);
  if (!workspace || !aklr_aligned16(workspace) || workspace_bytes < l.bytes) return AKLR_ERR_WORKSPACE;
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  VerifyArgs a{};
  a.target = target_probs;
  a.draft = draft_probs;
  a.target_row = target_stride;
  a.draft_row = draft_stride;
  a.tokens = draft_tokens;
  a.parents = parents;
  a.starts = starts;
  a.accept = accept_uniforms;
  a.sample = sample_uniforms;
  a.out = out_tokens;
  a.path = path;
  a.counts = counts;
  a.words = reinterpret_cast<uint64_t*>(ws);
  a.states = reinterpret_cast<State*>(ws + l.states);
  a.partial = reinterpret_cast<double*>(ws + l.partial);
  a.total = tokens;
  a.vocab = (int)vocab;
  a.units = p.units;
  a.most = (int)most;
  a.batch = (int)batch;
  a.token64 = tokens_64;
  a.splits = p.splits;
  a.per_wave = p.per_wave;
  const auto go = [&](auto kernel) -> int {
    for (int round = 0; round < p.rounds; ++round) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)(batch * p.splits)), dim3(kThreads), 0, stream, a, round, p.rounds);
      AKLR_LAUNCH_CHECK();
    }
    return AKLR_OK;
  };
  const auto form = [&](auto t) -> int {
    using T = decltype(t);
    if (chain) return sure ? go(verify_kernel<T, true, true>) : go(verify_kernel<T, true, false>);
    return sure ? go(verify_kernel<T, false, true>) : go(verify_kernel<T, false, false>);
  };
  return dtype == AKLR_OUT_BF16 ? form(uint16_t{}) : dtype == AKLR_OUT_F16 ? form(_Float16{}) : form(float{});
}

AKLR_SCALAR_FP32_END
