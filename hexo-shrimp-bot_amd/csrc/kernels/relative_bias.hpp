// The learned bias of a (query, key) pair by its relative position, shared by
// the forward and backward of the relative attention.
//
// A pair's bucket is looked up by the displacement c_key - c_query of the two
// rows' integer coordinates, clamped to the bucket table's half extents
// (hq, hr); the latent rows (index < n_latents) have no coordinates: a latent
// key's pairs take bucket B - 2, the other pairs of a latent query B - 1.  A
// workgroup serves one head and holds its bias per displacement in LDS, in
// raw-score units (bias * sqrt(hd)), where it is the C operand of the score
// product.  Coordinates are packed as two int16 halves and one side carries
// the half extents, so an entry's address is a saturating subtraction, two
// clamps and two 16-bit multiply-adds: five instructions and one LDS read per
// pair.  (A two-way dot product for the last two needs wait states after it.)
#pragma once

#include "common.hpp"

namespace mantis {
namespace {

constexpr int kXcds = 8;
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

constexpr int kMaxCoord = 30000;  // with a half extent of at most 2,047 a sum stays in int16

// c as the low half, r as the high one; past kMaxCoord the flag and the nearest
__device__ __forceinline__ uint32_t pack_coords(int32_t c, int32_t r, int32_t* flag) {
  const int32_t cc = c < -kMaxCoord ? -kMaxCoord : c > kMaxCoord ? kMaxCoord : c;
  const int32_t rr = r < -kMaxCoord ? -kMaxCoord : r > kMaxCoord ? kMaxCoord : r;
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

// The head's table, staged by the workgroup: store(i, bias, bucket) for entry
// i < nq nr + 2 (entries nq nr and nq nr + 1 are the latents'; a bucket that is
// none has bias 0 and the number n_buckets).  A bias is a load that depends on
// another one: the first kMany buckets of a thread are requested as a kernel
// begins, their biases once its rows are on their way.
struct TableStage {
  static constexpr int kMany = 4;
  int b[kMany];
  float x[kMany];
  __device__ __forceinline__ void request(const Relative& rel, int base = 0) {
    const int n = rel.nq * rel.nr;
#pragma unroll
    for (int u = 0; u < kMany; ++u) {
      const int i = base + 256 * u + int(threadIdx.x);
      b[u] = rel.buckets[i < n ? i : 0];
    }
  }
  __device__ __forceinline__ void biases(const Relative& rel, int64_t head, int base = 0) {
    const int n = rel.nq * rel.nr;
    const float* bias = rel.bias + head * rel.n_buckets;
#pragma unroll
    for (int u = 0; u < kMany; ++u) {
      const int i = base + 256 * u + int(threadIdx.x);
      if (i >= n) b[u] = rel.n_buckets - (i == n ? 2 : 1);
      const bool good = b[u] >= 0 && b[u] < rel.n_buckets;
      if (!good && i < n) raise_flag(rel.flag, MANTIS_FLAG_INDEX);
      b[u] = good ? b[u] : rel.n_buckets;
      x[u] = bias[good ? b[u] : 0];
    }
  }
  template <typename Store>
  __device__ __forceinline__ void store(const Relative& rel, float root_hd, Store put, int base = 0) const {
    const int n = rel.nq * rel.nr;
#pragma unroll
    for (int u = 0; u < kMany; ++u) {
      const int i = base + 256 * u + int(threadIdx.x);
      if (i < n + 2) put(i, b[u] < rel.n_buckets ? raw_bias(x[u], root_hd) : 0.f, b[u]);
    }
  }
  // after request and biases: the whole table
  template <typename Store>
  __device__ __forceinline__ void finish(const Relative& rel, int64_t head, float root_hd, Store put) {
    store(rel, root_hd, put);
    for (int base = 256 * kMany; base < rel.nq * rel.nr + 2; base += 256 * kMany) {
      request(rel, base);
      biases(rel, head, base);
      store(rel, root_hd, put, base);
    }
  }
};

// This lane's side of its pairs: the byte offset of the table entry (kEntry
// bytes each) of a pair with the other side's packed coordinates (kQuery: this
// lane holds the query).  A latent row's pairs all have one entry, which its
// clamps hold, whatever the displacement.
template <bool kQuery, int kEntry>
struct Side {
  s16x2_t own, lo, hi;
  uint32_t row_bytes;  // of the table
  int latent_other;    // the entry of a pair whose other side is a latent row
  __device__ __forceinline__ Side(const Relative& rel, uint32_t packed, bool latent) {
    const short hq = short((rel.nq - 1) / 2), hr = short((rel.nr - 1) / 2);
    const s16x2_t half{hq, hr}, c = __builtin_bit_cast(s16x2_t, packed);
    own = kQuery ? c - half : c + half;
    lo = latent ? s16x2_t{short(rel.nq), short(kQuery ? 1 : 0)} : s16x2_t{0, 0};
    hi = latent ? lo : s16x2_t{short(2 * hq), short(2 * hr)};
    row_bytes = uint32_t(kEntry * rel.nr);
    latent_other = kEntry * (rel.nq * rel.nr + (kQuery || latent ? 0 : 1));
  }
  // Four pairs side by side: saturating difference, clamps, column * entry bytes + row * row_bytes.
  // (Such instructions wait a cycle for the one before; left to itself the compiler puts a
  // pair's five in a row where registers are few, with an empty cycle after each: the passes of
  // two lines of 2,049-4,096 rows, 64 dims, 254 + 339 against 245 + 333 us.)
  __device__ __forceinline__ void at(uint4 other, int (&at)[4]) const {
    const uint32_t l = __builtin_bit_cast(uint32_t, lo), h = __builtin_bit_cast(uint32_t, hi);
    uint32_t o[4] = {other.x, other.y, other.z, other.w};
#define MANTIS_FOUR(op, a, b, c, d) op a "\n" op b "\n" op c "\n" op d "\n"
#define MANTIS_REST                                                                                              \
  MANTIS_FOUR("v_pk_min_i16 ", "%4, %4, %10", "%5, %5, %10", "%6, %6, %10", "%7, %7, %10")                       \
  MANTIS_FOUR("v_pk_max_i16 ", "%4, %4, %9", "%5, %5, %9", "%6, %6, %9", "%7, %7, %9")                           \
  MANTIS_FOUR("v_mad_i32_i16 ", "%0, %4, %12, 0 op_sel:[1,0,0,0]", "%1, %5, %12, 0 op_sel:[1,0,0,0]",            \
              "%2, %6, %12, 0 op_sel:[1,0,0,0]", "%3, %7, %12, 0 op_sel:[1,0,0,0]")                              \
  MANTIS_FOUR("v_mad_i32_i16 ", "%0, %4, %11, %0", "%1, %5, %11, %1", "%2, %6, %11, %2", "%3, %7, %11, %3")
#define MANTIS_OPERANDS                                                                                          \
  : "=&v"(at[0]), "=&v"(at[1]), "=&v"(at[2]), "=&v"(at[3]), "+v"(o[0]), "+v"(o[1]), "+v"(o[2]), "+v"(o[3])      \
  : "v"(own), "v"(l), "v"(h), "s"(row_bytes), "n"(kEntry)
    if constexpr (kQuery)
      asm(MANTIS_FOUR("v_pk_sub_i16 ", "%4, %4, %8 clamp", "%5, %5, %8 clamp", "%6, %6, %8 clamp", "%7, %7, %8 clamp")
              MANTIS_REST MANTIS_OPERANDS);
    else
      asm(MANTIS_FOUR("v_pk_sub_i16 ", "%4, %8, %4 clamp", "%5, %8, %5 clamp", "%6, %8, %6 clamp", "%7, %8, %7 clamp")
              MANTIS_REST MANTIS_OPERANDS);
#undef MANTIS_FOUR
#undef MANTIS_REST
#undef MANTIS_OPERANDS
  }
};

// table offsets of this lane's pairs with 64 rows of the other side, row 16 tt + 4 g + t
// from `first` on, their packed coordinates in LDS
template <bool kQuery, int kEntry>
__device__ __forceinline__ void pair_offsets(const Side<kQuery, kEntry>& side, int n_latents, const uint32_t* sc,
                                             int first, int g, int (&at)[4][4]) {
#pragma unroll
  for (int tt = 0; tt < 4; ++tt) side.at(*reinterpret_cast<const uint4*>(&sc[16 * tt + 4 * g]), at[tt]);
  if (first < n_latents) {  // uniform
    asm volatile("");       // (a branch: most chunks hold no latent row)
    const int lat = n_latents - first - 4 * g;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int t = 0; t < 4; ++t) at[tt][t] = 16 * tt + t < lat ? side.latent_other : at[tt][t];
  }
}
__device__ __forceinline__ float entry(const void* table, int byte_offset) {
  return *reinterpret_cast<const float*>(static_cast<const char*>(table) + byte_offset);
}

// Work items (position and head, tile of rows) to workgroups, which the
// dispatcher deals round-robin over the XCDs.  The unit that an XCD takes
// whole is a position where there are many, so that the heads that share its
// rows' cache lines share an L2, and a (position, head) where there are few,
// so that a long position's work is spread.  (Two lines of 2,049-4,096 rows, 8
// heads, against consecutive items on one XCD: the forward 198 -> 165 us, the
// backward's passes 585 + 324 -> 508 + 285; 512 positions of 44-124 rows by
// position 33 us, by head 35.)
struct Item {
  int64_t pa, tile;
};
constexpr int64_t kManyPositions = 64;
__device__ __forceinline__ Item item_of(int64_t n_pa, int heads, int64_t n_tiles) {
  const bool whole = n_pa / heads >= kManyPositions;
  const uint32_t per = uint32_t(whole ? heads * n_tiles : n_tiles);  // (the grid fits 31 bits)
  const uint32_t x = blockIdx.x % kXcds, i = blockIdx.x / kXcds, r = i % per;
  const int64_t unit = int64_t(i / per) * kXcds + x;
  return Item{whole ? unit * heads + r / uint32_t(n_tiles) : unit, int64_t(r % uint32_t(n_tiles))};
}
inline int64_t item_grid(int64_t n_pos, int heads, int64_t n_tiles) {
  const bool whole = n_pos >= kManyPositions;
  const int64_t units = whole ? n_pos : n_pos * heads, per = whole ? heads * n_tiles : n_tiles;
  return (units + kXcds - 1) / kXcds * kXcds * per;
}

// Long rows (T > 128) whose 64-row tiles leave half the CUs or more without a
// workgroup: tiles of 16 rows, the other side's chunks dealt over a workgroup's
// wavefronts.  Each stages its own, so the LDS grows with the head's width and at
// 64 dims the few workgroups that fit a CU gain from this only when tiles are fewer
// still.  The three passes of one position, 16 rows to a workgroup against 64: 2,000
// rows of 4 heads, 32 dims (128 tiles of 64) 133 against 161 us, 16 dims 121 / 160;
// 1,024 rows, 32 dims 52 / 89; 4,096 rows, 32 dims (256 tiles) 427 / 402, 16 dims 398 / 388;
// 64 dims, 2 heads, 1,024 rows (32 tiles) 74 / 100, 2,048 rows (64 tiles) 217 / 183.
inline bool few_groups(int64_t n_pos, int64_t heads, int64_t t, int64_t hd) {
  return t > 128 && n_pos * heads * ((t + 63) / 64) <= (hd < 64 ? 128 : 32);
}

// orders a wavefront's own LDS accesses around a tile that no other one uses
__device__ __forceinline__ void wave_sync() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

inline bool good_relative(const Relative& rel, int64_t t) {
  if (!rel.coords || !rel.buckets || !rel.bias || reinterpret_cast<uintptr_t>(rel.coords) % 8) return false;
  if (rel.nq < 1 || rel.nr < 1 || rel.nq % 2 == 0 || rel.nr % 2 == 0) return false;
  if (rel.nq > kMaxDisplacements || rel.nr > kMaxDisplacements || rel.nq * rel.nr > kMaxDisplacements) return false;
  if (rel.n_buckets < 1 || rel.n_buckets > kMaxBuckets) return false;
  return rel.n_latents >= 0 && rel.n_latents <= t && (rel.n_latents == 0 || rel.n_buckets >= 2);
}

}  // namespace
}  // namespace mantis
