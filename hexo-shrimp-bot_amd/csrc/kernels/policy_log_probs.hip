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
// order.  The best entries of a wavefront are a sorted list across its lanes:
// an entry that beats the last one is inserted by a ballot and a one-lane shift,
// so the pass costs two comparisons per entry and about top * ln(n / top)
// insertions.  One workgroup per run; long runs are cut into slices over
// several workgroups whose partial results a second launch joins.
#include "common.hpp"

namespace mantis {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTop = 64;
constexpr int kMaxMoves = 1024;
constexpr int kMaxSlices = 256;
constexpr int64_t kMinSlice = 4096;  // entries of a slice
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

// The best `top` entries of a wavefront: lane r holds the r-th.
struct Best {
  float v;
  uint32_t i;
  float worst_v;  // the last one's, in every lane
  uint32_t worst_i;
  __device__ __forceinline__ void clear() {
    v = worst_v = -INFINITY;
    i = worst_i = 0u;
  }
  // whether (x, at) comes before the last one (-inf and NaN never do)
  __device__ __forceinline__ bool wants(float x, uint32_t at) const {
    return x > worst_v || (x == worst_v && at < worst_i);
  }
  // one candidate per lane; in lanes without one `want` is false
  __device__ __forceinline__ void insert(float x, uint32_t at, bool want, int top) {
    uint64_t left = __builtin_amdgcn_ballot_w64(want);
    const int lane = threadIdx.x % 64;
    while (left) {
      const int src = __builtin_ctzll(left);
      left &= left - 1;
      const float cx = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), src));
      const uint32_t ci = __builtin_amdgcn_readlane(at, src);
      if (!wants(cx, ci)) continue;  // (uniform)
      const bool before = lane < top && (v > cx || (v == cx && i < ci));
      const int pos = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before));
      const float pv = __shfl_up(v, 1);
      const uint32_t pi = __shfl_up(i, 1);
      if (lane == pos) {
        v = cx;
        i = ci;
      } else if (lane > pos) {
        v = pv;
        i = pi;
      }
      worst_v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), top - 1));
      worst_i = __builtin_amdgcn_readlane(i, top - 1);
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

// What a position answers, from its joined state and list (in wavefront 0's lanes).
template <typename T>
__device__ __forceinline__ void write_run(const T* logits, int64_t stride, int64_t a, int64_t b, int64_t p, State s,
                                          const Best& best, const int64_t* moves, int64_t n_moves, int top,
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
    const int64_t mv = moves[p * n_moves + g];
    float lp = 0.f;
    if (mv >= 0 && mv < b - a) lp = none ? -INFINITY : (widen(logits[(a + mv) * stride]) - m) - log_l;
    else if (mv != -1) raise_flag(flag, MANTIS_FLAG_INDEX);
    out.log_probs[p * n_moves + g] = lp;
  }
  if (lane < top) {
    const bool there = best.v > -INFINITY && !bad;
    out.top_moves[p * top + lane] = there ? int64_t(best.i) : -1;
    out.top_log_probs[p * top + lane] = bad ? NAN : there ? (best.v - m) - log_l : -INFINITY;
  }
}

// The workgroup's join: every wavefront's state and list; the result in wavefront 0.
__device__ __forceinline__ void block_join(State& s, Best& best, int top) {
  __shared__ State states[kWaves];
  __shared__ float lv[kWaves][kMaxTop];
  __shared__ uint32_t li[kWaves][kMaxTop];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  s = wave_join(s);
  if (lane == 0) states[wave] = s;
  if (wave > 0 && lane < top) {
    lv[wave][lane] = best.v;
    li[wave][lane] = best.i;
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    join(s, states[w]);
    if (top > 0) {
      const float x = lane < top ? lv[w][lane] : -INFINITY;
      const uint32_t at = lane < top ? li[w][lane] : 0u;
      best.insert(x, at, best.wants(x, at), top);
    }
  }
}

constexpr int kBatch = 4;  // entries of a lane in flight

// The workgroup's entries [a + from, a + to) of a run into each lane's state and each wavefront's list.
template <typename T>
__device__ __forceinline__ void stream(const T* logits, int64_t stride, int64_t a, int64_t from, int64_t to, int top,
                                       State& s, Best& best) {
  for (int64_t base = from; base < to; base += kThreads * kBatch) {
    float x[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int64_t i = base + u * kThreads + threadIdx.x;
      x[u] = i < to ? widen(logits[(a + i) * stride]) : -INFINITY;
    }
    float m = x[0];
#pragma unroll
    for (int u = 1; u < kBatch; ++u) m = fmaxf(m, x[u]);
    lift(s, m);
    bool any = false;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      add(s, x[u]);
      any = any || best.wants(x[u], uint32_t(base + u * kThreads + threadIdx.x));
    }
    if (top > 0 && __builtin_amdgcn_ballot_w64(any)) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const uint32_t at = uint32_t(base + u * kThreads + threadIdx.x);
        best.insert(x[u], at, best.wants(x[u], at), top);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
policy_run_kernel(const T* __restrict__ logits, int64_t stride, const int64_t* __restrict__ offsets, int64_t n,
                  const int64_t* __restrict__ moves, int64_t n_moves, int top, Out out, int32_t* flag) {
  const int64_t p = blockIdx.x;
  int64_t a, b;
  run_of(offsets, p, n, a, b, flag);
  State s = empty_state();
  Best best;
  best.clear();
  stream(logits, stride, a, 0, b - a, top, s, best);
  block_join(s, best, top);
  if (threadIdx.x < 64) write_run(logits, stride, a, b, p, s, best, moves, n_moves, top, out, flag);
}

// Workspace of a sliced call: state, then values, then indices of each (position, slice).
struct Parts {
  float* state;  // (P, S, 3)
  float* v;      // (P, S, top)
  uint32_t* i;   // (P, S, top)
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
  if (int(threadIdx.x) < top) {
    parts.v[at * top + threadIdx.x] = best.v;
    parts.i[at * top + threadIdx.x] = best.i;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
policy_join_kernel(const T* __restrict__ logits, int64_t stride, const int64_t* __restrict__ offsets, int64_t n,
                   const int64_t* __restrict__ moves, int64_t n_moves, int top, int slices, Parts parts, Out out,
                   int32_t* flag) {
  const int64_t p = blockIdx.x;
  int64_t a, b;
  run_of(offsets, p, n, a, b, flag);
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
    const bool in = e + int(threadIdx.x) < entries;
    const float x = in ? parts.v[j] : -INFINITY;
    const uint32_t at = in ? parts.i[j] : 0u;
    best.insert(x, at, best.wants(x, at), top);
  }
  block_join(s, best, top);
  if (threadIdx.x < 64) write_run(logits, stride, a, b, p, s, best, moves, n_moves, top, out, flag);
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
  int64_t a, b;
  run_of(offsets, p, n, a, b, flag);
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
  auto base = [&](int64_t i) {
    const float lp = (widen(logits[(a + i) * stride]) - m) - log_l;
    const float pr = exp_neg(lp);
    return pr * (common - ge * (fmaxf(lp, -200.f) + h));  // (pr is 0 long before; keeps 0 * inf out)
  };
  for (int64_t i = from + threadIdx.x; i < to; i += kThreads) narrow(dx[a + i], none ? 0.f : base(i));
  // what no run holds has no gradient
  const int64_t stop = p == 0 ? (offsets[0] < 0 ? 0 : offsets[0] > n ? n : offsets[0]) : 0;
  for (int64_t i = sl * kThreads + threadIdx.x; i < stop; i += int64_t(slices) * kThreads) narrow(dx[i], 0.f);
  if (p == n_pos - 1)
    for (int64_t i = (offsets[n_pos] < 0 ? 0 : offsets[n_pos]) + sl * kThreads + threadIdx.x; i < n;
         i += int64_t(slices) * kThreads)
      narrow(dx[i], 0.f);
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
  parts.state = static_cast<float*>(workspace);
  parts.v = parts.state + 3 * n_pos * slices;
  parts.i = reinterpret_cast<uint32_t*>(parts.v + n_pos * slices * top);
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
  if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 4)) return MANTIS_E_ARG;
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
