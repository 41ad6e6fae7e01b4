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
// over the vocabulary, and 32 bits would move some of its borders with the order of the additions. The sums are bound by the
// loads all the same (figures at plan_verify).
#include "common.h"

AKLR_SCALAR_FP32_BEGIN

namespace aklr {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kMost = 1024;  // query tokens of a sequence
constexpr int kUnit = 512;   // values of a row that one wave adds up to a partial sum: 8 a lane

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
__device__ __forceinline__ float proper(float x) { return x > 0.0f && x < __builtin_inff() ? x : 0.0f; }

__device__ __forceinline__ double unit_number(float u) {
  return u > 0.0f ? (double)fminf(u, 0x1.fffffep-1f) : 0.0;
}

__device__ __forceinline__ double weight(float p, float q, double a) {  // no contraction: the product of a = 1 is exact
  return fmax(__dsub_rn((double)p, __dmul_rn(a, (double)q)), 0.0);
}

// Eight values of a row from v on, past its end zeros. Rows start at any multiple of their element: the loads are 16 bytes
// wide whatever the alignment.
template <typename T>
__device__ __forceinline__ void eight(const T* row, int v, int vocab, float (&f)[8]) {
  T x[8];
  if (v + 8 <= vocab) {
    __builtin_memcpy(x, row + v, sizeof(x));
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = widen<T>(x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = v + e < vocab ? widen<T>(row[v + e]) : 0.0f;
  }
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, 64);
  return x;
}

struct Drafts {  // a sequence's tokens, in LDS
  int parent[kMost], token[kMost];
  float u[kMost], p[kMost], q[kMost];
  int gone[kMost];  // tokens refused at the node, where drafts are certain
};

template <typename T, bool CHAIN, bool SURE>
__global__ __launch_bounds__(kThreads) void verify_kernel(const VerifyArgs a, const int round, const int rounds) {
  __shared__ Drafts d;
  __shared__ State st;
  __shared__ int gones;
  __shared__ double wave_total[kWaves];
  __shared__ unsigned slot;
  __shared__ int chosen, chosen_last, chosen_unit;
  __shared__ double chosen_before;
  const int seq = (int)(blockIdx.x / (unsigned)a.splits), split = (int)(blockIdx.x % (unsigned)a.splits);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t seen = 0;
  if (a.splits > 1 && threadIdx.x == 0) seen = splitk_peek(a.words + seq);

  const int64_t lo = a.starts[seq], hi = a.starts[seq + 1] < a.total ? a.starts[seq + 1] : a.total;
  const int n = lo < 0 || hi <= lo ? 0 : (int)(hi - lo < a.most ? hi - lo : a.most);
  if (n == 0) {  // no such sequence: nothing stands, nothing follows
    if (round == 0 && split == 0) {
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
    if (CHAIN) return node + 1 < n && i <= node + 1 && d.parent[node + 1] == node ? node + 1 : n;
    for (int base = i & ~63; base < n; base += 64) {
      const int j = base + lane;
      const uint64_t on = __ballot(j >= i && j < n && d.parent[j] == node);
      if (on) return base + __ffsll((unsigned long long)on) - 1;
    }
    return n;
  };
  // One wave: goes on from `st` until a row has to be added up, for a rejection or for the token that follows.
  const auto search = [&](State& s, int& refused, bool writes) {
    for (;;) {
      const int j = child(s.node, s.next);
      if (j >= n) {
        s.status = kEnd;
        return;
      }
      s.next = j + 1;
      const float q = SURE ? 1.0f : d.q[j];
      double w;
      if (SURE) {
        bool twice = false;
        for (int g = lane; g < refused; g += 64) twice |= d.gone[g] == d.token[j];
        w = __ballot(twice) ? 0.0 : (double)d.p[j];
      } else {
        w = weight(d.p[j], q, s.a);
      }
      if (__dmul_rn(__dmul_rn(unit_number(d.u[j]), s.s), (double)q) < w) {
        if (writes && lane == 0) {
          a.path[(int64_t)seq * a.most + s.count] = j;
          put_token(s.count - 1, token_at(j));
        }
        s.node = j;
        s.count += 1;
        s.a = 0.0;
        s.s = 1.0;
        refused = 0;
        continue;
      }
      if (SURE) {
        s.s -= w;
        if (lane == 0) d.gone[refused] = d.token[j];
        refused += 1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        continue;
      }
      s.a += s.s;
      s.status = kRefused;
      return;
    }
  };
  const auto search_all = [&](bool writes) {  // by the first wave; the state is everybody's afterwards
    __syncthreads();
    if (wave == 0) {
      State s = st;
      int refused = gones;
      search(s, refused, writes);
      if (lane == 0) {
        st = s;
        gones = refused;
      }
    }
    __syncthreads();
  };

  if (round == 0) {
    gather();
    if (threadIdx.x == 0) {
      st = {0, 1, 1, kEnd, 0.0, 1.0};
      gones = 0;
      if (split == 0) a.path[(int64_t)seq * a.most] = 0;
    }
    search_all(split == 0);
  } else {
    if (threadIdx.x == 0) {
      st = a.states[seq];
      gones = 0;
    }
    __syncthreads();
    if (st.status == kDone) return;
  }

  // What eight values from v on weigh.
  const auto weights = [&](const State& s, int v, double (&w)[8]) {
    float p[8], q[8];
    eight(target(s.node), v, a.vocab, p);
    const bool less = !SURE && s.a != 0.0;
    if (less) eight(draft(s.node), v, a.vocab, q);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = less ? weight(proper(p[e]), proper(q[e]), s.a) : (double)proper(p[e]);
    if (SURE && s.status != kWholeRow)
      for (int g = 0; g < gones; ++g) {
        const int at = d.gone[g] - v;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (at == e) w[e] = 0.0;
      }
  };
  double* const partial = a.partial + (int64_t)seq * a.units;
  const auto add_up = [&](int from, int to, int step) {  // the units from, from + step, ... of this wave
    const State s = st;
    for (int u = from; u < to; u += step) {
      double w[8];
      weights(s, u * kUnit + lane * 8, w);
      const double sum = wave_sum(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
      if (lane == 0) __hip_atomic_store(partial + u, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  };
  const int w0 = (split * kWaves + wave) * a.per_wave;
  add_up(w0, min(w0 + a.per_wave, a.units), 1);
  if (a.splits > 1) {
    if (!splitk_arrive(a.words + seq, seen, a.splits, &slot)) return;
  }
  if (round != 0) gather();

  // The last workgroup of the sequence: the sums of the units, in their order.
  for (;;) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    const int per = (a.units + kThreads - 1) / kThreads;
    const int u0 = threadIdx.x * per, u1 = min(u0 + per, a.units);
    double mine = 0.0;
    for (int u = u0; u < u1; ++u) mine += __hip_atomic_load(partial + u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    double upto = mine;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
      const double y = __shfl_up(upto, s, 64);
      if (lane >= s) upto += y;
    }
    if (lane == 63) wave_total[wave] = upto;
    __syncthreads();
    double total = 0.0, before = upto - mine;
    for (int w = 0; w < kWaves; ++w) {
      if (w == wave) before += total;
      total += wave_total[w];
    }
    if (st.status == kRefused) {
      __syncthreads();
      if (wave == 0) {  // another child of the node: it is tried against what the rejection leaves
        const bool more = child(st.node, st.next) < n;
        if (lane == 0) {
          st.s = total;
          if (!more) st.status = kEnd;
        }
      }
      __syncthreads();
      if (st.status == kRefused) {
        search_all(true);
        if (round + 1 < rounds) {  // the next launch's
          if (threadIdx.x == 0) a.states[seq] = st;
          return;
        }
        add_up(wave, a.units, kWaves);
        continue;
      }
    }
    if (!(total > 0.0) && st.status != kWholeRow) {  // nothing is left of the row: the target's own
      __syncthreads();
      if (threadIdx.x == 0) {
        st.status = kWholeRow;
        st.a = 0.0;
      }
      __syncthreads();
      add_up(wave, a.units, kWaves);
      continue;
    }
    // the unit in which the running sum passes the number, then the value
    const double level = unit_number(a.sample[seq]) * total;
    if (threadIdx.x == 0) {
      chosen = chosen_unit = 0x7FFFFFFF;
      chosen_last = -1;
    }
    __syncthreads();
    if (total > 0.0) {
      double run = before;
      int found = 0x7FFFFFFF, last = -1;
      double found_before = 0.0;
      for (int u = u0; u < u1; ++u) {
        const double x = __hip_atomic_load(partial + u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (x > 0.0) {
          last = u;
          if (found == 0x7FFFFFFF && run + x > level) {
            found = u;
            found_before = run;
          }
        }
        run += x;
      }
      if (found != 0x7FFFFFFF) atomicMin(&chosen_unit, found);
      if (last >= 0) atomicMax(&chosen_last, last);
      __syncthreads();
      if (chosen_unit == found && found != 0x7FFFFFFF) chosen_before = found_before;
      if (threadIdx.x == 0 && chosen_unit == 0x7FFFFFFF) {  // rounding took the last step: the last value that weighs
        chosen_unit = chosen_last;
        chosen_before = __builtin_inf();
      }
      __syncthreads();
      if (wave == 0) {
        const State s = st;
        double w[8];
        const int v = chosen_unit * kUnit + lane * 8;
        weights(s, v, w);
        double own = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) own += w[e];
        double to = own;
#pragma unroll
        for (int step = 1; step < 64; step *= 2) {
          const double y = __shfl_up(to, step, 64);
          if (lane >= step) to += y;
        }
        double sum = chosen_before + (to - own);
        int first = 0x7FFFFFFF, last_one = -1;
        if (chosen_before == __builtin_inf()) sum = -__builtin_inf();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sum += w[e];
          if (w[e] > 0.0) {
            last_one = v + e;
            if (first == 0x7FFFFFFF && sum > level) first = v + e;
          }
        }
        const uint64_t on = __ballot(first != 0x7FFFFFFF), any = __ballot(last_one >= 0);
        const int pick = on ? __shfl(first, __ffsll((unsigned long long)on) - 1, 64)
                            : __shfl(last_one, 63 - __clzll((long long)any), 64);
        if (lane == 0) chosen = pick;
      }
      __syncthreads();
    }
    const int count = st.count;
    for (int i = count + threadIdx.x; i < a.most; i += kThreads) {
      a.path[(int64_t)seq * a.most + i] = -1;
      put_token(i, -1);
    }
    if (threadIdx.x == 0) {
      put_token(count - 1, total > 0.0 ? chosen : -1);
      a.counts[seq] = count;
      if (rounds > 1) a.states[seq].status = kDone;
    }
    return;
  }
}

}  // namespace aklr

using namespace aklr;

namespace {

struct Plan {
  int units, splits, per_wave, rounds;
};

// How many workgroups share a row: one unit a wave until they fill the chip twice over (four of 512 lanes a CU), and at
// most 255, what an arrival word counts. Only trees whose drafts have rows need more than one sum of a row a sequence;
// they get `rounds` launches for it, and what is left after those the last workgroup does alone.
Plan plan_verify(int64_t batch, int64_t vocab, bool chain, bool sure, int64_t most) {
  Plan p;
  p.units = (int)((vocab + kUnit - 1) / kUnit);
  int64_t splits = (p.units + kWaves - 1) / kWaves;
  const int64_t room = batch < 2048 ? 2048 / batch : 1;
  if (splits > room) splits = room;
  if (splits > 255) splits = 255;
  p.per_wave = (int)((p.units + splits * kWaves - 1) / (splits * kWaves));
  p.splits = (int)((p.units + p.per_wave * kWaves - 1) / (p.per_wave * kWaves));
  p.rounds = chain || sure || most <= 2 ? 1 : most < 6 ? (int)most - 1 : 5;
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
  return batch >= 1 && batch <= 65536 && vocab >= 1 && vocab <= (1 << 24) && most >= 1 && most <= kMost;
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
