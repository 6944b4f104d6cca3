// Dropout of a residual branch for gfx950, its mask drawn where it is used
// and never stored (the trunk blocks' x + drop(f(x)), model.py:263-380):
//   out = residual + (keep ? x / (1 - p) : 0),  keep = word >= round(p 2^32)
// The same kernel without a residual is the operator's backward, dx of the
// incoming gradient.
//
// The words are Philox4x32 with ten rounds (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011): element i of the
// row-major order takes word i % 4 of the counter (i / 4 low, i / 4 high, step,
// salt) under the 64-bit key `seed`, with (seed, step) read on the device, so a
// captured graph draws another mask when the caller advances step.
// Sums and products are fp32 (one fma), the output rounds once.
#include <cmath>

#include "common.hpp"

namespace mantis {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint4 philox(uint64_t group, uint32_t step, uint32_t salt, uint32_t k0, uint32_t k1) {
  uint32_t a = uint32_t(group), b = uint32_t(group >> 32), c = step, d = salt;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p = uint64_t(0xD2511F53u) * a, q = uint64_t(0xCD9E8D57u) * c;
    a = uint32_t(q >> 32) ^ b ^ k0;
    b = uint32_t(q);
    c = uint32_t(p >> 32) ^ d ^ k1;
    d = uint32_t(p);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(a, b, c, d);
}

struct Bf16 {
  uint16_t bits;
};
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(_Float16 x) { return float(x); }
__device__ __forceinline__ float widen(Bf16 x) { return bf2f(x.bits); }
// (round to nearest even; an fp16 overflow is an infinity and NaN stays NaN)
__device__ __forceinline__ void narrow(float& d, float x) { d = x; }
__device__ __forceinline__ void narrow(_Float16& d, float x) { d = _Float16(x); }
__device__ __forceinline__ void narrow(Bf16& d, float x) { d.bits = uint16_t(pack_bf16x2(x, x)); }

template <typename T>
struct alignas(4 * sizeof(T)) Four {
  T v[4];
};

// A thread takes one group of four elements, one generator call: 16 of its
// bytes in flight, and enough threads to hide the ten rounds.  kVec: the bases
// are aligned to a group (the last group's elements one by one).
//
// Bound by memory: 63,488 x 128 elements, bf16 onto fp32, 14.4 us (81 MB, 5.6 TB/s),
// its backward 10.5 us (49 MB, 4.6 TB/s); 131,071 x 255 in bf16, 26.5 us each way
// (134 MB, 5.0 TB/s; a large copy 4.8).  Small calls are launches: 4 us.
template <typename TX, typename TO, bool kResidual, bool kVec>
__global__ void __launch_bounds__(kThreads)
residual_dropout_kernel(const TX* __restrict__ x, const TO* __restrict__ residual, const int64_t* __restrict__ rng,
                        int64_t n, uint32_t threshold, bool none, float scale, uint32_t salt,
                        TO* __restrict__ out) {
  const uint64_t seed = uint64_t(rng[0]);
  const uint32_t step = uint32_t(rng[1]);
  const int64_t g = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t i = 4 * g;
  if (i >= n) return;
  const uint4 w = philox(uint64_t(g), step, salt, uint32_t(seed), uint32_t(seed >> 32));
  const bool keep[4] = {w.x >= threshold && !none, w.y >= threshold && !none, w.z >= threshold && !none,
                        w.w >= threshold && !none};
  auto one = [&](int t, TX xv, TO rv) {
    TO o;
    const float base = kResidual ? widen(rv) : 0.f;
    narrow(o, keep[t] ? fmaf(widen(xv), scale, base) : base);
    return o;
  };
  if (kVec && i + 4 <= n) {
    const Four<TX> xv = *reinterpret_cast<const Four<TX>*>(x + i);
    Four<TO> rv{}, o;
    if (kResidual) rv = *reinterpret_cast<const Four<TO>*>(residual + i);
#pragma unroll
    for (int t = 0; t < 4; ++t) o.v[t] = one(t, xv.v[t], rv.v[t]);
    *reinterpret_cast<Four<TO>*>(out + i) = o;
  } else {
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (i + t < n) out[i + t] = one(t, x[i + t], kResidual ? residual[i + t] : TO{});
  }
}

template <typename TX, typename TO>
int32_t launch(const void* x, const void* residual, const int64_t* rng, int64_t n, uint32_t threshold, bool none,
               float scale, uint32_t salt, void* out, hipStream_t st) {
  const int64_t grid = ((n + 3) / 4 + kThreads - 1) / kThreads;
  if (grid > 2147483647LL) return MANTIS_E_ARG;
  auto on = [](const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
  const bool vec = on(x, 4 * sizeof(TX)) && on(out, 4 * sizeof(TO)) && on(residual, 4 * sizeof(TO));
  auto kernel = residual ? (vec ? residual_dropout_kernel<TX, TO, true, true> : residual_dropout_kernel<TX, TO, true, false>)
                         : (vec ? residual_dropout_kernel<TX, TO, false, true> : residual_dropout_kernel<TX, TO, false, false>);
  kernel<<<unsigned(grid), kThreads, 0, st>>>(static_cast<const TX*>(x), static_cast<const TO*>(residual), rng, n,
                                              threshold, none, scale, salt, static_cast<TO*>(out));
  return launched();
}

template <typename TX>
int32_t launch_out(int32_t out_dtype, const void* x, const void* residual, const int64_t* rng, int64_t n,
                   uint32_t threshold, bool none, float scale, uint32_t salt, void* out, hipStream_t st) {
  if (out_dtype == MANTIS_F32) return launch<TX, float>(x, residual, rng, n, threshold, none, scale, salt, out, st);
  if (out_dtype == MANTIS_F16) return launch<TX, _Float16>(x, residual, rng, n, threshold, none, scale, salt, out, st);
  if (out_dtype == MANTIS_BF16) return launch<TX, Bf16>(x, residual, rng, n, threshold, none, scale, salt, out, st);
  return MANTIS_E_ARG;
}

}  // namespace
}  // namespace mantis

using namespace mantis;

extern "C" int32_t mantis_residual_dropout(const void* x, int32_t x_dtype, const void* residual, const int64_t* rng,
                                           int64_t n, double p, int64_t salt, void* out, int32_t out_dtype,
                                           void* stream) {
  if (n == 0) return MANTIS_OK;
  if (!x || !rng || !out || n < 0) return MANTIS_E_ARG;
  if (!(p >= 0.0 && p <= 1.0) || salt < 0 || salt > 0xFFFFFFFFLL) return MANTIS_E_ARG;
  auto width = [](int32_t d) { return d == MANTIS_F32 ? 4u : 2u; };
  if (reinterpret_cast<uintptr_t>(x) % width(x_dtype) || reinterpret_cast<uintptr_t>(out) % width(out_dtype) ||
      reinterpret_cast<uintptr_t>(residual) % width(out_dtype) || reinterpret_cast<uintptr_t>(rng) % 8)
    return MANTIS_E_ARG;
  // p within 2^-33 of 1 drops every element, as p = 1 does
  const double border = std::nearbyint(p * 4294967296.0);
  const bool none = border >= 4294967296.0;
  const uint32_t threshold = none ? 0xFFFFFFFFu : uint32_t(border);
  const float scale = none ? 0.f : float(1.0 / (1.0 - p));
  hipStream_t st = as_stream(stream);
  const uint32_t s = uint32_t(salt);
  if (x_dtype == MANTIS_F32) return launch_out<float>(out_dtype, x, residual, rng, n, threshold, none, scale, s, out, st);
  if (x_dtype == MANTIS_F16) return launch_out<_Float16>(out_dtype, x, residual, rng, n, threshold, none, scale, s, out, st);
  if (x_dtype == MANTIS_BF16) return launch_out<Bf16>(out_dtype, x, residual, rng, n, threshold, none, scale, s, out, st);
  return MANTIS_E_ARG;
}
