// The learned bias of a (query, key) pair by its relative position, shared by
// the forward and backward of the relative attention.
//
// A pair's bucket is looked up by the displacement c_key - c_query of the two
// rows' integer coordinates, clamped to the bucket table's half extents
// (hq, hr); the latent rows (index < n_latents) have no coordinates: a latent
// key's pairs take bucket B - 2, the other pairs of a latent query B - 1.  A
// workgroup serves one head and holds its bias per displacement in LDS, in
// raw-score units (bias * sqrt(hd)), where it is the C operand of the score
// product.  Coordinates are packed as two int16 halves, so an entry's address
// is a saturating subtraction, two clamps and one two-way dot product:
// four instructions and one LDS read per pair.
#pragma once

#include "common.hpp"

namespace mantis {
namespace {

constexpr int kMaxDisplacements = 4096;  // entries of a bucket table
constexpr int kMaxBuckets = 384;

struct Relative {
  const int32_t* coords;   // (P, T, 2)
  const int32_t* buckets;  // (nq, nr)
  const float* bias;       // (heads, n_buckets)
  int nq, nr, n_buckets;
  int64_t n_latents;
  int32_t* flag;
};

typedef short s16x2_t __attribute__((ext_vector_type(2)));

// c in int16 as the low half, r as the high one; outside of int16 the flag and the nearest
__device__ __forceinline__ uint32_t pack_coords(int32_t c, int32_t r, int32_t* flag) {
  const int32_t cc = c < -32768 ? -32768 : c > 32767 ? 32767 : c, rr = r < -32768 ? -32768 : r > 32767 ? 32767 : r;
  if (cc != c || rr != r) raise_flag(flag, MANTIS_FLAG_INDEX);
  return uint32_t(uint16_t(cc)) | uint32_t(uint16_t(rr)) << 16;
}

// row t of position p: its packed coordinates, zeros at or past L
__device__ __forceinline__ uint32_t coords_of(const Relative& rel, int64_t p, int64_t T, int64_t t, int64_t L) {
  if (t >= L) return 0u;
  const int2 c = *reinterpret_cast<const int2*>(rel.coords + 2 * (p * T + t));
  return t < rel.n_latents ? 0u : pack_coords(c.x, c.y, rel.flag);
}

// a bias in raw-score units; a finite one stays finite (a mask of the type's lowest value is no -inf)
constexpr float kLargest = 3.402823466e38f;
__device__ __forceinline__ float raw_bias(float b, float root_hd) {
  const float x = b * root_hd;
  return fabsf(b) <= kLargest ? fminf(fmaxf(x, -kLargest), kLargest) : b;
}

// Entry displacement d of a head's table: entries nq nr and nq nr + 1 are the latents'.
__device__ __forceinline__ int bucket_of(const Relative& rel, int i) {
  const int n = rel.nq * rel.nr;
  int b = i < n ? rel.buckets[i] : rel.n_buckets - (i == n ? 2 : 1);
  if (b < 0 || b >= rel.n_buckets) {
    if (i < n) raise_flag(rel.flag, MANTIS_FLAG_INDEX);
    b = rel.n_buckets;  // (no bias, no gradient)
  }
  return b;
}

// the head's table, staged by the workgroup: table[i], i < nq nr + 2
__device__ __forceinline__ void stage_bias(const Relative& rel, int64_t head, float root_hd, float* table) {
  for (int i = threadIdx.x; i < rel.nq * rel.nr + 2; i += blockDim.x) {
    const int b = bucket_of(rel, i);
    table[i] = b < rel.n_buckets ? raw_bias(rel.bias[head * rel.n_buckets + b], root_hd) : 0.f;
  }
}

// This lane's side of its pairs: the byte offset of the entry of a pair with
// the other side's packed coordinates (kQuery: this lane holds the query).
template <bool kQuery>
struct Side {
  s16x2_t own, lo, hi, mult;
  int base, latent_other;
  __device__ __forceinline__ Side(const Relative& rel, uint32_t packed, bool latent) {
    const short hq = short((rel.nq - 1) / 2), hr = short((rel.nr - 1) / 2);
    const int n = rel.nq * rel.nr;
    own = __builtin_bit_cast(s16x2_t, packed);
    lo = s16x2_t{short(-hq), short(-hr)};
    hi = s16x2_t{hq, hr};
    // a latent row's pairs all have one entry, whatever the displacement
    mult = latent ? s16x2_t{0, 0} : s16x2_t{short(4 * rel.nr), 4};
    base = latent ? 4 * (kQuery ? n + 1 : n) : 4 * (hq * rel.nr + hr);
    // the entry of a pair whose other side is a latent row
    latent_other = kQuery || latent ? 4 * n : 4 * (n + 1);
  }
  __device__ __forceinline__ int at(uint32_t other) const {
    const s16x2_t o = __builtin_bit_cast(s16x2_t, other);
    s16x2_t d = kQuery ? __builtin_elementwise_sub_sat(o, own) : __builtin_elementwise_sub_sat(own, o);
    d = __builtin_elementwise_max(__builtin_elementwise_min(d, hi), lo);
    return __builtin_amdgcn_sdot2(d, mult, base, false);
  }
};
__device__ __forceinline__ float entry(const float* table, int byte_offset) {
  return *reinterpret_cast<const float*>(reinterpret_cast<const char*>(table) + byte_offset);
}

inline bool good_relative(const Relative& rel, int64_t t) {
  if (!rel.coords || !rel.buckets || !rel.bias || reinterpret_cast<uintptr_t>(rel.coords) % 8) return false;
  if (rel.nq < 1 || rel.nr < 1 || rel.nq % 2 == 0 || rel.nr % 2 == 0) return false;
  if (rel.nq > kMaxDisplacements || rel.nr > kMaxDisplacements || rel.nq * rel.nr > kMaxDisplacements) return false;
  if (rel.n_buckets < 1 || rel.n_buckets > kMaxBuckets) return false;
  return rel.n_latents >= 0 && rel.n_latents <= t && (rel.n_latents == 0 || rel.n_buckets >= 2);
}

}  // namespace
}  // namespace mantis
