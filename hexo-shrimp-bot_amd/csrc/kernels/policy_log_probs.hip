// Log probabilities of the moves played, entropy and best alternatives of a
// ragged policy (the legal rows of each position, CSR offsets) for gfx950, and
// the gradient of all of them.  With x the logits of one run, m their maximum
// and l = sum exp(x - m):
//   lse = m + log l,  log_prob(i) = (x_i - m) - log l,
//   entropy = log l - sum exp(x - m) (x - m) / l,
//   the best `top` entries by (x descending, index ascending), x > -inf
//   dx_i = p_i (g_lse - sum_g G_g - sum_k K_k - g_H (log p_i + H))
//          + sum of the G_g with move g = i + sum of the K_k with top k = i
// A run without a finite weight (empty, or -inf everywhere) has lse -inf,
// entropy 0, log probabilities -inf, no alternatives and zero gradients; a run
// with a NaN or +inf is NaN, without alternatives.
//
// Forward: one pass over the logits, each lane with its own running maximum,
// sum and weighted sum in fp32, joined by shuffles and through LDS in a fixed
// order.  The best entries of a wavefront are a list of 64-bit keys (value,
// then index) sorted across its lanes, joined by VALU lane moves: entries that
// beat the last one are inserted one by one where they are few, and sorted and
// merged as 64 where they are many (a run's first), so the pass costs a
// comparison per 16 bytes and about top * ln(n / top) insertions.  One workgroup
// per run; long runs are cut into slices over several workgroups whose partial
// results a second launch joins.
//
// Measured: one run of 271 with 16 alternatives 6.4 us, the latency of one
// workgroup (a load, the sort of 64, the join); 512 runs of 180-1,200 fp32 with 8
// alternatives 10.5 us, the lists' sorting, and 7.1 backward; 64 runs of 131,072 bf16
// with 4 alternatives 13.7 + 6.2 us (16.8 MB: 3.5 at the rate of a large copy; the
// exponentials and the list's upkeep bound it), backward 12.4 (33.6 MB: 7.0).
#include "common.hpp"

namespace mantis {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTop = 64;
constexpr int kMaxMoves = 1024;
constexpr int kMaxSlices = 256;
constexpr int64_t kMinSlice = 4096;  // entries of a slice: one pass of its loads in flight
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Bf16 {
  uint16_t bits;
};
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(_Float16 x) { return float(x); }
__device__ __forceinline__ float widen(Bf16 x) { return bf2f(x.bits); }
__device__ __forceinline__ void narrow(float& d, float x) { d = x; }
__device__ __forceinline__ void narrow(_Float16& d, float x) { d = _Float16(x); }
__device__ __forceinline__ void narrow(Bf16& d, float x) { d.bits = uint16_t(pack_bf16x2(x, x)); }

// exp(x) for x <= 0 and NaN
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// The running softmax state of a set of logits.
struct State {
  float m, l, t;  // maximum, sum exp(x - m), sum exp(x - m) (x - m)
};
__device__ __forceinline__ State empty_state() { return State{-INFINITY, 0.f, 0.f}; }

// a state seen from the maximum m >= s.m
__device__ __forceinline__ void lift(State& s, float m) {
  if (m > s.m) {
    const float d = fmaxf(s.m - m, -200.f);  // (exp is 0 long before; keeps 0 * -inf out)
    const float a = exp_neg(d);
    s.t = a * fmaf(s.l, d, s.t);
    s.l = s.m == -INFINITY ? s.l : a * s.l;
    s.m = m;
  }
}
__device__ __forceinline__ void add(State& s, float x) {
  const float d = x - (s.m == -INFINITY ? 0.f : s.m);
  const float e = exp_neg(d);
  s.l += e;
  s.t = fmaf(e, fmaxf(d, -200.f), s.t);  // (e is 0 long before; keeps 0 * -inf out)
}
__device__ __forceinline__ void join(State& s, State o) {
  const float m = fmaxf(s.m, o.m);
  lift(s, m);
  lift(o, m);
  s.l += o.l;
  s.t += o.t;
}
__device__ __forceinline__ State wave_join(State s) {
  float m = s.m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  lift(s, m);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    s.l += __shfl_xor(s.l, o);
    s.t += __shfl_xor(s.t, o);
  }
  return s;
}

// The value of lane ^ X: VALU lane moves, no LDS round trip.
template <int X>
__device__ __forceinline__ uint32_t from_lane_xor(uint32_t x) {
  constexpr int kDpp = X == 1 ? 0xB1 : X == 2 ? 0x4E : X == 3 ? 0x1B : X == 7 ? 0x141 : X == 15 ? 0x140 : 0;
  if constexpr (kDpp != 0) {  // quad permutations, mirrored half rows and rows of 16
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(x), kDpp, 0xF, 0xF, false));
  } else if constexpr (X == 4) {
    return from_lane_xor<3>(from_lane_xor<7>(x));
  } else if constexpr (X == 8) {
    return from_lane_xor<7>(from_lane_xor<15>(x));
  } else if constexpr (X == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  } else if constexpr (X == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
  } else {
    static_assert(X == 31 || X == 63, "a butterfly or mirror distance");
    return from_lane_xor<(X + 1) / 2>(from_lane_xor<X / 2>(x));
  }
}

// An entry as one number: greater comes first (the value, then the lower
// index); 0 is no entry.  NaN and -inf are none.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t at) {
  const uint32_t u = __float_as_uint(x + 0.f);  // (-0 and 0 are one value)
  const uint32_t up = u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
  return x > -INFINITY ? uint64_t(up) << 32 | (0xFFFFFFFFu - at) : 0u;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t up = uint32_t(key >> 32);
  return key ? __uint_as_float(up ^ (up >> 31 ? 0x80000000u : 0xFFFFFFFFu)) : -INFINITY;
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xFFFFFFFFu - uint32_t(key); }

__device__ __forceinline__ uint64_t key_in_lane(uint64_t key, int lane) {
  return uint64_t(__builtin_amdgcn_readlane(uint32_t(key >> 32), lane)) << 32 |
         uint32_t(__builtin_amdgcn_readlane(uint32_t(key), lane));
}

// lane and lane ^ X: the greater key to the lower lane
template <int X>
__device__ __forceinline__ void exchange(uint64_t& key) {
  const uint64_t other = uint64_t(from_lane_xor<X>(uint32_t(key >> 32))) << 32 | from_lane_xor<X>(uint32_t(key));
  constexpr int kTop = X >= 32 ? 32 : X >= 16 ? 16 : X >= 8 ? 8 : X >= 4 ? 4 : X >= 2 ? 2 : 1;
  if ((other > key) != bool(threadIdx.x & kTop)) key = other;
}
template <int X>
__device__ __forceinline__ void exchanges_from(uint64_t& key) {  // X, X / 2, .. 1
  exchange<X>(key);
  if constexpr (X > 1) exchanges_from<X / 2>(key);
}
// 64 keys into descending lanes: bitonic, every merge opened by a mirrored exchange
__device__ __forceinline__ void sort_keys(uint64_t& key) {
  exchange<1>(key);
  exchange<3>(key), exchanges_from<1>(key);
  exchange<7>(key), exchanges_from<2>(key);
  exchange<15>(key), exchanges_from<4>(key);
  exchange<31>(key), exchanges_from<8>(key);
  exchange<63>(key), exchanges_from<16>(key);
}

// The best entries of a wavefront, descending over its lanes; the first `top` count.
struct Best {
  uint64_t key, worst;  // worst: the top-th, in every lane
  float worst_v;
  __device__ __forceinline__ void clear() {
    key = worst = 0;
    worst_v = -INFINITY;
  }
  __device__ __forceinline__ void settle(int top) {
    worst = key_in_lane(key, top - 1);
    worst_v = value_of(worst);
  }
  // one sorted list more: `reversed` holds its 63 - lane-th
  __device__ __forceinline__ void merge(uint64_t reversed, int top) {
    key = reversed > key ? reversed : key;  // the best 64 of both, as a bitonic sequence
    exchanges_from<32>(key);
    settle(top);
  }
  // a candidate per lane (0: none), wavefront-uniform.  A few are inserted one
  // by one (a ballot and a one-lane shift each, about a sixth of a sort and merge)
  __device__ __forceinline__ void take(uint64_t candidate, int top) {
    uint64_t left = __builtin_amdgcn_ballot_w64(candidate > worst);
    if (__builtin_popcountll(left) > 6) {
      sort_keys(candidate);
      const uint64_t reversed = uint64_t(from_lane_xor<63>(uint32_t(candidate >> 32))) << 32 |
                                from_lane_xor<63>(uint32_t(candidate));
      merge(reversed, top);
      return;
    }
    const int lane = threadIdx.x % 64;
    while (left) {
      const uint64_t c = key_in_lane(candidate, __builtin_ctzll(left));
      left &= left - 1;
      if (c <= worst) continue;  // (uniform)
      const int pos = __builtin_popcountll(__builtin_amdgcn_ballot_w64(key > c));
      // lane - 1's key (wave_shr:1)
      const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(key >> 32), 0x138, 0xF, 0xF, false));
      const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(key), 0x138, 0xF, 0xF, false));
      key = lane > pos ? uint64_t(hi) << 32 | lo : lane == pos ? c : key;
      settle(top);
    }
  }
};

struct Out {
  float* log_probs;
  float* entropy;
  float* lse;
  float* top_log_probs;
  int64_t* top_moves;
  float* norm;  // (P, 2): m and log l
};

// entries [a, b) of run p, clamped into [0, n); false (and the flag) for a run that is not one
__device__ __forceinline__ bool run_of(const int64_t* offsets, int64_t p, int64_t n, int64_t& a, int64_t& b,
                                       int32_t* flag) {
  a = offsets[p], b = offsets[p + 1];
  if (a >= 0 && b >= a && b <= n && b - a <= 0x7FFFFFFFLL) return true;
  if (threadIdx.x == 0) raise_flag(flag, MANTIS_FLAG_ORDER);
  a = b = 0;
  return false;
}

// A chosen move's logit, in lane g: read before the run so that its two
// dependent loads do not follow the pass.
struct Chosen {
  int64_t move;
  float x;
};
template <typename T>
__device__ __forceinline__ Chosen chosen(const T* logits, int64_t stride, int64_t a, int64_t b, int64_t p,
                                         const int64_t* moves, int64_t n_moves, int64_t g) {
  Chosen c{-1, 0.f};
  if (g < n_moves) c.move = moves[p * n_moves + g];
  if (c.move >= 0 && c.move < b - a) c.x = widen(logits[(a + c.move) * stride]);
  return c;
}

// What a position answers, from its joined state and list (in wavefront 0's lanes).
template <typename T>
__device__ __forceinline__ void write_run(const T* logits, int64_t stride, int64_t a, int64_t b, int64_t p, State s,
                                          const Best& best, Chosen c, const int64_t* moves, int64_t n_moves, int top,
                                          const Out& out, int32_t* flag) {
  const int lane = threadIdx.x;
  const bool none = s.m == -INFINITY && s.l == 0.f, bad = s.l != s.l;
  const float m = none ? 0.f : s.m;
  const float log_l = none ? -INFINITY : logf(s.l);
  if (lane == 0) {
    out.entropy[p] = none ? 0.f : log_l - s.t / s.l;
    out.lse[p] = m + log_l;
    out.norm[2 * p] = m;
    out.norm[2 * p + 1] = log_l;
  }
  for (int64_t g = lane; g < n_moves; g += 64) {
    if (g >= 64) c = chosen(logits, stride, a, b, p, moves, n_moves, g);
    float lp = 0.f;
    if (c.move >= 0 && c.move < b - a) lp = none ? -INFINITY : (c.x - m) - log_l;
    else if (c.move != -1) raise_flag(flag, MANTIS_FLAG_INDEX);
    out.log_probs[p * n_moves + g] = lp;
  }
  if (lane < top) {
    const bool there = best.key && !bad;
    out.top_moves[p * top + lane] = there ? int64_t(index_of(best.key)) : -1;
    out.top_log_probs[p * top + lane] = bad ? NAN : there ? (value_of(best.key) - m) - log_l : -INFINITY;
  }
}

// The workgroup's join: every wavefront's state and list; the result in wavefront 0.
__device__ __forceinline__ void block_join(State& s, Best& best, int top) {
  __shared__ State states[kWaves];
  __shared__ uint64_t keys[kWaves][64];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  s = wave_join(s);
  if (lane == 0) states[wave] = s;
  if (wave > 0) keys[wave][63 - lane] = best.key;
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    join(s, states[w]);
    if (top > 0) best.merge(keys[w][lane], top);
  }
}

// kN entries of each lane, x[e] at index at + step(e) >= at (past the end: -inf)
template <int kN, typename Step>
__device__ __forceinline__ void absorb(const float (&x)[kN], uint32_t at, Step step, int top, State& s, Best& best) {
  float m = x[0];
#pragma unroll
  for (int e = 1; e < kN; ++e) m = fmaxf(m, x[e]);
  lift(s, m);
#pragma unroll
  for (int e = 0; e < kN; ++e) add(s, x[e]);
  if (top > 0 && __builtin_amdgcn_ballot_w64(m > best.worst_v || (m == best.worst_v && best.worst && at < index_of(best.worst)))) {
    // What can still be among the best: entries up to the last one's value, or, before there is
    // one, up to the top-th of the lanes' maxima (top lanes hold at least one that great)
    float cut = best.worst_v;
    if (kN > 1 && !best.worst) {
      uint64_t maxima = key_of(m, 0);
      sort_keys(maxima);
      cut = value_of(key_in_lane(maxima, top - 1));
    }
#pragma unroll
    for (int e = 0; e < kN; ++e)
      if (__builtin_amdgcn_ballot_w64(x[e] >= cut && x[e] > -INFINITY))
        best.take(x[e] >= cut ? key_of(x[e], at + step(e)) : 0u, top);
  }
}

// The workgroup's entries [from, to) of the run at `a` into each lane's state and
// each wavefront's list: 16-byte loads where the entries are dense, those before
// and after the aligned blocks and strided ones one by one; four loads of a lane in flight.
template <typename T>
__device__ __forceinline__ void stream(const T* logits, int64_t stride, int64_t a, int64_t from, int64_t to, int top,
                                       State& s, Best& best) {
  constexpr int kV = 16 / sizeof(T), kLoads = 4;
  const T* run = logits + a * stride;
  if (stride == 1 && to - from >= kThreads * kV / 2) {
    const int head = int((kV - reinterpret_cast<uintptr_t>(run + from) / sizeof(T) % kV) % kV);
    const int64_t blocks = (to - from - head) / kV, body = from + head, tail = body + blocks * kV;
    for (int64_t base = 0; base < blocks; base += kThreads * kLoads) {
      uint4 raw[kLoads];
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        const int64_t b = base + u * kThreads + threadIdx.x;
        raw[u] = *reinterpret_cast<const uint4*>(run + body + (b < blocks ? b : 0) * kV);
      }
      float x[kLoads * kV];
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        T v[kV];
        __builtin_memcpy(v, &raw[u], 16);
#pragma unroll
        for (int e = 0; e < kV; ++e)
          x[u * kV + e] = base + u * kThreads + threadIdx.x < blocks ? widen(v[e]) : -INFINITY;
      }
      absorb(x, uint32_t(body + (base + threadIdx.x) * kV), [](int i) { return uint32_t(i / kV * kThreads * kV + i % kV); },
             top, s, best);
    }
    if (threadIdx.x < 64) {  // up to kV - 1 entries on each side
      const int lane = threadIdx.x;
      const int64_t i = lane < head ? from + lane : tail + lane - head;
      const float x[1] = {i < to && lane < 2 * kV ? widen(run[i]) : -INFINITY};
      absorb(x, uint32_t(i), [](int) { return 0u; }, top, s, best);
    }
    return;
  }
  for (int64_t base = from; base < to; base += kThreads * kLoads) {
    float x[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int64_t i = base + u * kThreads + threadIdx.x;
      x[u] = i < to ? widen(run[i * stride]) : -INFINITY;
    }
    absorb(x, uint32_t(base + threadIdx.x), [](int i) { return uint32_t(i * kThreads); }, top, s, best);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
policy_run_kernel(const T* __restrict__ logits, int64_t stride, const int64_t* __restrict__ offsets, int64_t n,
                  const int64_t* __restrict__ moves, int64_t n_moves, int top, Out out, int32_t* flag) {
  const int64_t p = blockIdx.x;
  int64_t a, b;
  run_of(offsets, p, n, a, b, flag);
  const Chosen c = chosen(logits, stride, a, b, p, moves, n_moves, threadIdx.x < 64 ? threadIdx.x : n_moves);
  State s = empty_state();
  Best best;
  best.clear();
  stream(logits, stride, a, 0, b - a, top, s, best);
  block_join(s, best, top);
  if (threadIdx.x < 64) write_run(logits, stride, a, b, p, s, best, c, moves, n_moves, top, out, flag);
}

// Workspace of a sliced call: the list, then the state of each (position, slice).
struct Parts {
  uint64_t* key;  // (P, S, top), each slice's descending
  float* state;   // (P, S, 3)
};

template <typename T>
__global__ void __launch_bounds__(kThreads)
policy_slice_kernel(const T* __restrict__ logits, int64_t stride, const int64_t* __restrict__ offsets, int64_t n,
                    int top, int slices, Parts parts, int32_t* flag) {
  const int64_t p = blockIdx.x / slices, sl = blockIdx.x % slices;
  int64_t a, b;
  run_of(offsets, p, n, a, b, flag);
  const int64_t len = b - a, from = len * sl / slices, to = len * (sl + 1) / slices;
  State s = empty_state();
  Best best;
  best.clear();
  stream(logits, stride, a, from, to, top, s, best);
  block_join(s, best, top);
  if (threadIdx.x >= 64) return;
  const int64_t at = p * slices + sl;
  if (threadIdx.x == 0) {
    parts.state[3 * at] = s.m;
    parts.state[3 * at + 1] = s.l;
    parts.state[3 * at + 2] = s.t;
  }
  if (int(threadIdx.x) < top) parts.key[at * top + threadIdx.x] = best.key;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
policy_join_kernel(const T* __restrict__ logits, int64_t stride, const int64_t* __restrict__ offsets, int64_t n,
                   const int64_t* __restrict__ moves, int64_t n_moves, int top, int slices, Parts parts, Out out,
                   int32_t* flag) {
  const int64_t p = blockIdx.x;
  int64_t a, b;
  run_of(offsets, p, n, a, b, flag);
  const Chosen c = chosen(logits, stride, a, b, p, moves, n_moves, threadIdx.x < 64 ? threadIdx.x : n_moves);
  State s = empty_state();
  Best best;
  best.clear();
  for (int sl = threadIdx.x; sl < slices; sl += kThreads) {
    const int64_t at = p * slices + sl;
    join(s, State{parts.state[3 * at], parts.state[3 * at + 1], parts.state[3 * at + 2]});
  }
  const int64_t entries = int64_t(slices) * top;
  for (int64_t e = 0; e < entries; e += kThreads) {
    const int64_t j = p * entries + e + threadIdx.x;
    best.take(e + int(threadIdx.x) < entries ? parts.key[j] : 0u, top);
  }
  block_join(s, best, top);
  if (threadIdx.x < 64) write_run(logits, stride, a, b, p, s, best, c, moves, n_moves, top, out, flag);
}

// The gradient of a slice of a run: every entry's share of the sums, then the
// entries that a move or an alternative names once more with what they add.
template <typename T>
__global__ void __launch_bounds__(kThreads)
policy_backward_kernel(const T* __restrict__ logits, int64_t stride, const int64_t* __restrict__ offsets,
                       int64_t n_pos, int64_t n, const int64_t* __restrict__ moves, int64_t n_moves, int top,
                       const int64_t* __restrict__ top_moves, const float* __restrict__ entropy,
                       const float* __restrict__ norm, const float* __restrict__ g_log,
                       const float* __restrict__ g_ent, const float* __restrict__ g_lse,
                       const float* __restrict__ g_top, int slices, T* __restrict__ dx, int32_t* flag) {
  extern __shared__ __attribute__((aligned(16))) char shared[];
  const int entries = int(n_moves) + top;
  int64_t* at = reinterpret_cast<int64_t*>(shared);     // (entries): the index named, or -1
  float* add = reinterpret_cast<float*>(at + entries);  // (entries): its gradient
  __shared__ float sums[kWaves];
  const int64_t p = blockIdx.x / slices, sl = blockIdx.x % slices;
  auto clear = [&](int64_t lo, int64_t hi) {  // this slice's share of [lo, hi)
    for (int64_t i = lo + sl * kThreads + threadIdx.x; i < hi; i += int64_t(slices) * kThreads) narrow(dx[i], 0.f);
  };
  auto bound = [&](int64_t i) { return i < 0 ? 0 : i > n ? n : i; };
  int64_t a, b;
  // what no run holds has no gradient: entries between offsets that are no run, before the first and after the last
  if (!run_of(offsets, p, n, a, b, flag)) clear(bound(offsets[p]), bound(offsets[p + 1]));
  if (p == 0) clear(0, bound(offsets[0]));
  if (p == n_pos - 1) clear(bound(offsets[n_pos]), n);
  const int64_t len = b - a, from = len * sl / slices, to = len * (sl + 1) / slices;
  const float m = norm[2 * p], log_l = norm[2 * p + 1], h = entropy[p];
  const bool none = log_l == -INFINITY;
  float part = 0.f;
  for (int e = threadIdx.x; e < entries; e += kThreads) {
    const bool is_move = e < n_moves;
    const int64_t i = is_move ? moves[p * n_moves + e] : top_moves[p * top + e - n_moves];
    const float* src = is_move ? g_log : g_top;
    const bool there = i >= 0 && i < len && src;
    const float g = there ? src[is_move ? p * n_moves + e : p * top + e - n_moves] : 0.f;
    at[e] = there ? i : -1;
    add[e] = g;
    part += g;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) part += __shfl_xor(part, o);
  if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = part;
  __syncthreads();
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) total += sums[w];
  const float common = (g_lse ? g_lse[p] : 0.f) - total, ge = g_ent ? g_ent[p] : 0.f;
  auto base_of = [&](float x) {
    const float lp = (x - m) - log_l;
    const float pr = exp_neg(lp);
    return pr * (common - ge * (fmaxf(lp, -200.f) + h));  // (pr is 0 long before; keeps 0 * inf out)
  };
  auto base = [&](int64_t i) { return base_of(widen(logits[(a + i) * stride])); };
  constexpr int kV = 16 / sizeof(T);
  int64_t body = from, tail = from;  // the entries in blocks of 16 bytes, where both sides share their alignment
  if (stride == 1 && (reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(dx)) % 16 == 0) {
    const int64_t head = int64_t((kV - reinterpret_cast<uintptr_t>(dx + a + from) / sizeof(T) % kV) % kV);
    if (head < to - from) {
      body = from + head;
      tail = body + (to - body) / kV * kV;
    }
  }
  for (int64_t i = body + kV * threadIdx.x; i < tail; i += kV * kThreads) {
    const uint4 raw = *reinterpret_cast<const uint4*>(logits + a + i);
    T v[kV];
    __builtin_memcpy(v, &raw, 16);
#pragma unroll
    for (int e = 0; e < kV; ++e) narrow(v[e], none ? 0.f : base_of(widen(v[e])));
    uint4 res;
    __builtin_memcpy(&res, v, 16);
    *reinterpret_cast<uint4*>(dx + a + i) = res;
  }
  for (int64_t i = from + threadIdx.x; i < body; i += kThreads) narrow(dx[a + i], none ? 0.f : base(i));
  for (int64_t i = tail + threadIdx.x; i < to; i += kThreads) narrow(dx[a + i], none ? 0.f : base(i));
  if (none) return;
  __syncthreads();  // (orders the writes above before those of the same entries below)
  for (int e = threadIdx.x; e < entries; e += kThreads) {
    const int64_t i = at[e];
    if (i < from || i >= to) continue;
    bool first = true;
    for (int f = 0; f < e; ++f) first = first && at[f] != i;
    if (!first) continue;
    float g = 0.f;
    for (int f = e; f < entries; ++f) g += at[f] == i ? add[f] : 0.f;
    narrow(dx[a + i], base(i) + g);
  }
}

// Workgroups of a run, from the mean length (the offsets stay on the device): up
// to `groups` in all, of `least` entries or more.
int slices_of(int64_t n_pos, int64_t n, int64_t least, int64_t groups) {
  const int64_t mean = n / n_pos, most = mean / least, want = (groups + n_pos - 1) / n_pos;
  const int64_t s = most < want ? most : want;
  return int(s < 1 ? 1 : s > kMaxSlices ? kMaxSlices : s);
}

int forward_slices(int64_t n_pos, int64_t n) { return slices_of(n_pos, n, kMinSlice, 1024); }

template <typename T>
int32_t forward(const void* logits, int64_t stride, const int64_t* offsets, int64_t n_pos, int64_t n,
                const int64_t* moves, int64_t n_moves, int top, const Out& out, void* workspace, int32_t* flag,
                hipStream_t st) {
  const T* x = static_cast<const T*>(logits);
  const int slices = forward_slices(n_pos, n);
  if (slices == 1) {
    policy_run_kernel<T><<<unsigned(n_pos), kThreads, 0, st>>>(x, stride, offsets, n, moves, n_moves, top, out, flag);
    return launched();
  }
  Parts parts;
  parts.key = static_cast<uint64_t*>(workspace);
  parts.state = reinterpret_cast<float*>(parts.key + n_pos * slices * top);
  policy_slice_kernel<T><<<unsigned(n_pos * slices), kThreads, 0, st>>>(x, stride, offsets, n, top, slices, parts, flag);
  policy_join_kernel<T><<<unsigned(n_pos), kThreads, 0, st>>>(x, stride, offsets, n, moves, n_moves, top, slices, parts,
                                                             out, flag);
  return launched();
}

bool good_run_args(const void* logits, int32_t dtype, int64_t stride, const int64_t* offsets, int64_t n_pos, int64_t n,
                   const int64_t* moves, int64_t n_moves, int32_t top) {
  if (!offsets || n_pos < 0 || n < 0 || (n > 0 && !logits) || stride < 1) return false;
  if (n_moves < 0 || n_moves > kMaxMoves || (n_moves > 0 && !moves) || top < 0 || top > kMaxTop) return false;
  if (dtype != MANTIS_F32 && dtype != MANTIS_F16 && dtype != MANTIS_BF16) return false;
  return n_pos <= 2147483647LL / kMaxSlices && reinterpret_cast<uintptr_t>(logits) % (dtype == MANTIS_F32 ? 4 : 2) == 0;
}

}  // namespace
}  // namespace mantis

using namespace mantis;

extern "C" int64_t mantis_policy_log_probs_workspace(int64_t n_pos, int64_t n, int32_t top) {
  if (n_pos <= 0 || n < 0 || top < 0) return 0;
  const int64_t slices = forward_slices(n_pos, n);
  return slices == 1 ? 0 : n_pos * slices * (12 + 8 * int64_t(top));
}

extern "C" int32_t mantis_policy_log_probs(const void* logits, int32_t dtype, int64_t stride, const int64_t* offsets,
                                           int64_t n_pos, int64_t n, const int64_t* moves, int64_t n_moves, int32_t top,
                                           float* log_probs, float* entropy, float* lse, float* top_log_probs,
                                           int64_t* top_moves, float* norm, void* workspace, int64_t workspace_bytes,
                                           int32_t* err_flag, void* stream) {
  if (n_pos == 0) return MANTIS_OK;
  if (!good_run_args(logits, dtype, stride, offsets, n_pos, n, moves, n_moves, top)) return MANTIS_E_ARG;
  if (!entropy || !lse || !norm || (n_moves > 0 && !log_probs) || (top > 0 && (!top_log_probs || !top_moves)))
    return MANTIS_E_ARG;
  const int64_t need = mantis_policy_log_probs_workspace(n_pos, n, top);
  if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 8)) return MANTIS_E_ARG;
  const Out out{log_probs, entropy, lse, top_log_probs, top_moves, norm};
  auto go = dtype == MANTIS_F32 ? forward<float> : dtype == MANTIS_F16 ? forward<_Float16> : forward<Bf16>;
  return go(logits, stride, offsets, n_pos, n, moves, n_moves, top, out, workspace, err_flag, as_stream(stream));
}

extern "C" int32_t mantis_policy_log_probs_backward(const void* logits, int32_t dtype, int64_t stride,
                                                    const int64_t* offsets, int64_t n_pos, int64_t n,
                                                    const int64_t* moves, int64_t n_moves, int32_t top,
                                                    const int64_t* top_moves, const float* entropy, const float* norm,
                                                    const float* grad_log_probs, const float* grad_entropy,
                                                    const float* grad_lse, const float* grad_top, void* grad_logits,
                                                    int32_t* err_flag, void* stream) {
  if (n_pos == 0 || n == 0) return MANTIS_OK;
  if (!good_run_args(logits, dtype, stride, offsets, n_pos, n, moves, n_moves, top)) return MANTIS_E_ARG;
  if (!entropy || !norm || !grad_logits || (top > 0 && !top_moves)) return MANTIS_E_ARG;
  const int slices = slices_of(n_pos, n, kThreads * 4, 4096);
  const size_t lds = size_t(n_moves + top) * 12;
  hipStream_t st = as_stream(stream);
#define MANTIS_POLICY_BWD(T)                                                                                       \
  policy_backward_kernel<T><<<unsigned(n_pos * slices), kThreads, lds, st>>>(                                      \
      static_cast<const T*>(logits), stride, offsets, n_pos, n, moves, n_moves, top, top_moves, entropy, norm,     \
      grad_log_probs, grad_entropy, grad_lse, grad_top, slices, static_cast<T*>(grad_logits), err_flag)
  if (dtype == MANTIS_F32) MANTIS_POLICY_BWD(float);
  else if (dtype == MANTIS_F16) MANTIS_POLICY_BWD(_Float16);
  else MANTIS_POLICY_BWD(Bf16);
#undef MANTIS_POLICY_BWD
  return launched();
}
