// Backward of the relative attention on 16-bit MFMA for gfx950.  With the
// forward's statistics (m, log2 l) per row, s_ij the raw scores with their bias
// (relative_bias.hpp) and c = log2(e) / sqrt(hd):
//   p_ij = exp2(c (s_ij - m_i) - log2 l_i),  dp_ij = go_i . v_j,
//   delta_i = sum_j p_ij dp_ij,  ds_ij = p_ij (dp_ij - delta_i),
//   dq_i = sum_j ds_ij k_j / sqrt(hd),  dk_j = sum_i ds_ij q_i / sqrt(hd),
//   dv_j = sum_i p_ij go_i,  dbias[a, b] = sum of ds_ij over the pairs of bucket b.
//
// Two passes, each a workgroup per (position, head, 64 rows), 16 rows per
// wavefront, the other side's rows in 64-row chunks through LDS, two buffers
// (where those are few workgroups, 16 rows each and the chunks dealt over the
// wavefronts, whose sums join at the end in their order):
//   query-major  S^T = K Q^T and dP^T = V dO^T, then dQ^T += K^T dS^T
//   key-major    S = Q K^T and dP = dO V^T, then dV^T += dO^T P, dK^T += Q^T dS
// Both keep a lane on one row of its own side, so a score fragment is the next
// product's B operand as it stands, and read the transposed A operand from the
// same row-major LDS rows (the transposing 64-bit LDS read of gfx950).
// delta needs every key of a row before the first ds (and the 16-bit output
// times its gradient is no substitute: its rounding would stay in every ds of
// the row and in the bias gradient's long sums).  Up to two chunks of keys (T <=
// 128) keep p and dp in registers until delta is known.  Longer rows are met
// once, with a reference r in delta's place, the mean of dp by the weights met so far:
//   dq = sum p (dp - r) k - (delta - r) sum p k,
// both sums brought to the new r after every chunk, and the buckets' sums move to the key
// pass, which knows delta.  (A second sweep over the keys instead: the two passes 511 + 285 us
// against 258 + 352 at two lines of 2,049-4,096 rows.  With r = 0 the passes take 3-5% less, but where
// one key holds a row or dp has a mean of many deviations the terms cancel after
// their cut to parts: a row with all but 5e-6 of its weight on one key lost 30% of dq.)
//
// Precision: scores and dp are exact products of 16-bit rows summed in fp32.
// The probabilities and ds enter their products as two 16-bit parts, hi + lo:
// bf16 beside bf16 rows (16 significant bits), beside fp16 rows fp16 parts of the
// value times a power of two that follows the largest of its column (22
// bits of that one).  What is cut is 2^-17 of a term p (dp - delta) k, or p (dp - r) k, which is
// of the same size: under the 2^-8 or 2^-11 that the outputs round unless terms of that size
// cancel again, over keys that share a large mean.  (fp32 MFMAs with widened rows instead: the passes
// 1,741 + 957 us where these parts took 619 + 337.)
// dk and dv keep the sums of both parts apart until the end, where an infinite one is
// the hi parts' alone (join_parts); any infinity that reaches dq is NaN by the formula.
// (That took the backward of one position of 1,024 rows, 2 heads of 64 dims, from 53.3 to
// 55.9 us, and left wider grids as they were.)
//
// The bias gradient: every lane adds its ds to its own column of the
// workgroup's LDS table (a row of 64 lanes per bucket and wavefront: no two
// lanes meet, no bank is asked twice), four entries read, added and written
// at a time; where that table does not fit, the four lane groups in turn to 16
// columns.  (LDS float atomics instead: 2.5 cycles per lane, half of the whole
// pass.)  The columns join in a fixed order into the workgroup's partial sums and
// those of a head by sum_bias.  Every sum is fp32 in a fixed order: two calls agree bitwise.
//
// Bound by the pairs' vector and LDS work, not by memory or the matrix units: a
// pair takes two products to recompute p and dp, exp2, the split into parts and,
// in the pass with the bucket sums, two LDS accesses more.  Measured, query pass
// + key pass: 192 positions of 44-124 rows, 4 heads, 32 dims, 25 + 20 us; 16 of
// 511-1,021 rows, 8 heads of 16 dims, 101 + 156; two lines of 2,049-4,096 rows, 8
// heads of 64 dims, 263 + 324 (their products alone at the rate of a large matrix product: 118).
#include <atomic>
#include <type_traits>

#include "attention_rows.hpp"
#include "relative_bias.hpp"

namespace mantis {
namespace {

constexpr int kBwdWaves = 4;
constexpr size_t kLdsBytes = 160 * 1024;

// Dynamic LDS: the table by displacement (the bias; in the pass with the bucket sums
// the bias and the byte offset of the bucket's row of columns), then that pass's columns.
__host__ __device__ constexpr size_t table_bytes(int n_disp, int entry) {
  return (size_t(n_disp + 2) * entry + 15) / 16 * 16;
}
__host__ __device__ constexpr size_t column_bytes(int n_buckets, int columns) {
  return size_t(kBwdWaves) * (n_buckets + 1) * columns * 4;  // (a row for the pairs of no bucket)
}

// 64 rows of one operand, staged by kThreads threads: kPer 16-byte pieces of each, in registers and
// then in LDS at kPitch; rows at or past the descriptor's count are zeros.
template <int HD, int kThreads>
struct RowTile {
  static constexpr int kPitch = HD + 8;           // 16-bit elements
  static constexpr int kPieces = kTile * HD / 8;  // 16-byte pieces
  static constexpr int kPer = kPieces < kThreads ? 1 : kPieces / kThreads;
  uint4 reg[kPer];
  __device__ __forceinline__ void fetch(i32x4_t rows, int32_t first) {
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const int i = int(threadIdx.x) % kThreads + kThreads * r;
      reg[r] = row_load16(rows, i < kPieces ? first + i / (HD / 8) : -1, 16 * (i % (HD / 8)));
    }
  }
  __device__ __forceinline__ void stage(uint16_t* s) const {
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const int i = int(threadIdx.x) % kThreads + kThreads * r;
      if (i < kPieces) *reinterpret_cast<uint4*>(s + (i / (HD / 8)) * kPitch + 8 * (i % (HD / 8))) = reg[r];
    }
  }
};

__device__ __forceinline__ i32x4_t rows_of(const Rows& r, int64_t pos, int64_t a, int64_t L) {
  return rows_rsrc(r.at(pos, a), uint32_t(r.st * 2), uint32_t(L));
}

// this lane's row as the B fragments of a product over dims (HD = 16: lanes g >= 2 hold zeros)
template <bool kHalf, int HD>
__device__ __forceinline__ void row_frags(i32x4_t rows, int64_t row, int g, uint4 (&u)[Geom<kHalf, HD>::kKs]) {
  using G = Geom<kHalf, HD>;
#pragma unroll
  for (int ks = 0; ks < G::kKs; ++ks) {
    u[ks] = row_load16(rows, int32_t(row), 2 * G::kdim(ks, g));
    if (HD < 32 && g >= 2) u[ks] = make_uint4(0u, 0u, 0u, 0u);
  }
}

// two fp32 values as their packed 16-bit parts: hi rounded, lo what is left
template <bool kHalf>
__device__ __forceinline__ void parts(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = Frag<kHalf>::pack_unit(a, b);
  if constexpr (kHalf) {
    const f16x2_t h = __builtin_bit_cast(f16x2_t, hi);
    lo = Frag<true>::pack_unit(a - float(h[0]), b - float(h[1]));
  } else {
    lo = Frag<false>::pack_unit(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
  }
}

// hi + lo (HD dims x this lane's row) += transposed rows . x for the staged rows
// below n, x the 16 fp32 values of this lane (rows 16 tt + 4 g + t; zeros from n on).
// Each part has its own sum where a row or a value may be infinite (join_parts);
// one serves as both where every such product is NaN anyhow.
template <bool kHalf, int HD>
__device__ __forceinline__ void accumulate_parts(const uint16_t* s, int n, int l16, int g, const f32x4_t (&x)[4],
                                                 f32x4_t (&acc_hi)[Geom<kHalf, HD>::kDt],
                                                 f32x4_t (&acc_lo)[Geom<kHalf, HD>::kDt]) {
  using FR = Frag<kHalf>;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (32 * h >= n) {  // uniform
      around_products();
      continue;
    }
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      parts<kHalf>(x[2 * h + i / 2][2 * (i % 2)], x[2 * h + i / 2][2 * (i % 2) + 1], hi[i], lo[i]);
    const typename FR::vec bh = FR::cast(make_uint4(hi[0], hi[1], hi[2], hi[3]));
    const typename FR::vec bl = FR::cast(make_uint4(lo[0], lo[1], lo[2], lo[3]));
#pragma unroll
    for (int dt = 0; dt < Geom<kHalf, HD>::kDt; ++dt) {
      const typename FR::vec a = FR::cast(transposed_frag<HD>(s, h, dt, l16, g));
      acc_hi[dt] = mfma16x16x32(a, bh, acc_hi[dt]);
      acc_lo[dt] = mfma16x16x32(a, bl, acc_lo[dt]);
    }
  }
}

// The sum of both parts; a sum that is not finite is the hi parts' alone.  An infinite row
// meets the lo parts too, which are zero or of either sign, and an infinite value
// has lo = inf - inf: added, they would make a NaN of an infinity.
template <int kDt>
__device__ __forceinline__ void join_parts(f32x4_t (&hi)[kDt], const f32x4_t (&lo)[kDt]) {
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
    for (int t = 0; t < 4; ++t) hi[dt][t] = __builtin_isfinite(hi[dt][t]) ? hi[dt][t] + lo[dt][t] : hi[dt][t];
}

// the same for two sums of one operand, whose fragments are read once
template <bool kHalf, int HD>
__device__ __forceinline__ void accumulate_two(const uint16_t* s, int n, int l16, int g, const f32x4_t (&x)[4],
                                               f32x4_t (&acc_x)[Geom<kHalf, HD>::kDt], const f32x4_t (&y)[4],
                                               f32x4_t (&acc_y)[Geom<kHalf, HD>::kDt]) {
  using FR = Frag<kHalf>;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (32 * h >= n) {  // uniform
      around_products();
      continue;
    }
    uint32_t xh[4], xl[4], yh[4], yl[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      parts<kHalf>(x[2 * h + i / 2][2 * (i % 2)], x[2 * h + i / 2][2 * (i % 2) + 1], xh[i], xl[i]);
      parts<kHalf>(y[2 * h + i / 2][2 * (i % 2)], y[2 * h + i / 2][2 * (i % 2) + 1], yh[i], yl[i]);
    }
#pragma unroll
    for (int dt = 0; dt < Geom<kHalf, HD>::kDt; ++dt) {
      const typename FR::vec a = FR::cast(transposed_frag<HD>(s, h, dt, l16, g));
      acc_x[dt] = mfma16x16x32(a, FR::cast(make_uint4(xh[0], xh[1], xh[2], xh[3])), acc_x[dt]);
      acc_x[dt] = mfma16x16x32(a, FR::cast(make_uint4(xl[0], xl[1], xl[2], xl[3])), acc_x[dt]);
      acc_y[dt] = mfma16x16x32(a, FR::cast(make_uint4(yh[0], yh[1], yh[2], yh[3])), acc_y[dt]);
      acc_y[dt] = mfma16x16x32(a, FR::cast(make_uint4(yl[0], yl[1], yl[2], yl[3])), acc_y[dt]);
    }
  }
}

// the scale of a probability's fp16 parts (it is at most 1)
template <bool kHalf>
constexpr float kPScale = kHalf ? 0x1p14f : 1.f;

// The power of two that a column's fp16 parts are scaled by: the largest value
// met so far lands in [2^13, 2^15].  bf16 parts need none.
template <bool kHalf>
struct ColumnScale {
  float s = kHalf ? 0x1p126f : 1.f;
  // scales x, and the sums when the scale moves; the four lanes of a column agree
  template <int kDt, typename... Acc>
  __device__ __forceinline__ void apply(f32x4_t (&x)[4], f32x4_t (&acc)[kDt], Acc&... more) {
    if constexpr (kHalf) {
      float m = 0.f;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int t = 0; t < 4; ++t) m = fmaxf(m, fabsf(x[tt][t]));
      m = max_xor32(max_xor16(m));
      const bool over = m * s > 32768.f;
      if (__builtin_amdgcn_ballot_w64(over)) {  // wavefront-uniform
        const int e = 267 - int(__float_as_uint(m) >> 23);  // 2^13 over m's power of two
        const float next = over ? __uint_as_float(uint32_t(e < 1 ? 1 : e > 253 ? 253 : e) << 23) : s;
        const float ratio = next / s;
        s = next;
#pragma unroll
        for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            acc[dt][t] *= ratio;
            ((more[dt][t] *= ratio), ...);
          }
      }
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int t = 0; t < 4; ++t) x[tt][t] *= s;
    }
  }
};

// A chunk's values in fp16 parts by themselves: x scaled so that the column's
// largest lands in [2^13, 2^14), and what undoes it.
__device__ __forceinline__ float chunk_scale(f32x4_t (&x)[4]) {
  float m = 0.f;
#pragma unroll
  for (int tt = 0; tt < 4; ++tt)
#pragma unroll
    for (int t = 0; t < 4; ++t) m = fmaxf(m, fabsf(x[tt][t]));
  m = max_xor32(max_xor16(m));
  const int e = 267 - int(__float_as_uint(m) >> 23), in = e > 253 ? 253 : e;  // (12 for an infinity)
  const float s = __uint_as_float(uint32_t(in) << 23);
#pragma unroll
  for (int tt = 0; tt < 4; ++tt)
#pragma unroll
    for (int t = 0; t < 4; ++t) x[tt][t] *= s;
  return __uint_as_float(uint32_t(254 - in) << 23);
}

// Four adds of a lane to its own LDS words, all read before the first is
// written: words named twice take the sum so far (merge4, before the reads'
// answer where it can be: one set of comparisons serves every turn).
__device__ __forceinline__ void merge4(const int (&at)[4], float (&x)[4]) {
  const float x1 = x[1] + (at[1] == at[0] ? x[0] : 0.f);
  const float x2 = x[2] + (at[2] == at[1] ? x1 : at[2] == at[0] ? x[0] : 0.f);
  x[3] += at[3] == at[2] ? x2 : at[3] == at[1] ? x1 : at[3] == at[0] ? x[0] : 0.f;
  x[1] = x1;
  x[2] = x2;
}
template <bool kMerged>
__device__ __forceinline__ void add4(char* base, const int (&at)[4], float (&x)[4]) {
  float old[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) old[t] = *reinterpret_cast<const float*>(base + at[t]);
  if (!kMerged) merge4(at, x);
#pragma unroll
  for (int t = 0; t < 4; ++t) *reinterpret_cast<float*>(base + at[t]) = old[t] + x[t];
}

// The workgroup's bucket sums: kColumns columns per wavefront of n_buckets + 1
// rows (the last for pairs of no bucket), behind the table of (bias, byte
// offset of the bucket's row) by displacement.
template <int kColumns>
struct BucketSums {
  const char* table;
  float* columns;
  char* own;  // this lane's column (a dead row's lanes spoil only their own, which no sum takes)
  int n_rows;
  __device__ __forceinline__ BucketSums(const Relative& rel, char* dynamic) {
    table = dynamic;
    columns = reinterpret_cast<float*>(dynamic + table_bytes(rel.nq * rel.nr, 8));
    n_rows = rel.n_buckets + 1;
    own = reinterpret_cast<char*>(columns + threadIdx.x / 64 * n_rows * kColumns + threadIdx.x % kColumns);
  }
  __device__ __forceinline__ void stage(TableStage& biases, const Relative& rel, int64_t head, float root_hd,
                                        char* dynamic) {
    uint2* entries = reinterpret_cast<uint2*>(dynamic);
    biases.finish(rel, head, root_hd, [&](int d, float x, int b) {
      entries[d] = make_uint2(__float_as_uint(x), uint32_t(b) * kColumns * 4);
    });
    for (int c = threadIdx.x; c < kBwdWaves * n_rows * kColumns / 4; c += 256)
      reinterpret_cast<float4*>(columns)[c] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // a pair's raw bias, by its table offset, for which it leaves the one of its bucket's columns
  __device__ __forceinline__ float entry(int& at) const {
    const uint2 e = *reinterpret_cast<const uint2*>(table + at);
    at = int(e.y);
    return __uint_as_float(e.x);
  }
  // four pairs of this lane, by what entry left
  __device__ __forceinline__ void add(const int (&to)[4], const f32x4_t& ds, bool live) {
    float x[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) x[t] = kColumns < 16 && !live ? 0.f : ds[t];  // (two rows share a column of eight)
    if constexpr (kColumns == 64) {
      add4<false>(own, to, x);
    } else {
      merge4(to, x);
#pragma unroll
      for (int turn = 0; turn < 64 / kColumns; ++turn) {
        if (int(threadIdx.x) % 64 / kColumns == turn) add4<true>(own, to, x);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the next group reads what this one wrote)
      }
    }
  }
  // every bucket's sum over the columns of the workgroup's first n_live rows
  // (`step` rows on from a wavefront to the next; 0: the same 16 in each):
  // eight threads to a bucket, starting apart so that a wavefront's reads meet other banks
  __device__ __forceinline__ void flush(int n_live, int step, float* sums) const {
    for (int b0 = 0; b0 < n_rows - 1; b0 += 32) {
      const int b = b0 + int(threadIdx.x) / 8, eighth = threadIdx.x % 8;
      float sum = 0.f;
      if (b < n_rows - 1)
        for (int w = 0; w < kBwdWaves; ++w)
#pragma unroll
          for (int c = 0; c < kColumns / 8; ++c) {
            const int col = (8 * c + eighth + 8 * (int(threadIdx.x) / 8)) % kColumns;
            const float x = columns[(w * n_rows + b) * kColumns + col];
            sum += step * w + col % 16 < n_live ? x : 0.f;
          }
      sum += __shfl_xor(sum, 1);
      sum += __shfl_xor(sum, 2);
      sum += __shfl_xor(sum, 4);
      if (b < n_rows - 1 && eighth == 0) sums[b] = sum;
    }
  }
};

// a kernel without bucket sums stages the biases alone
template <>
struct BucketSums<0> {
  const char* table;
  __device__ __forceinline__ BucketSums(const Relative&, char* dynamic) : table(dynamic) {}
  __device__ __forceinline__ float entry(int at) const { return mantis::entry(table, at); }
  __device__ __forceinline__ void stage(TableStage& biases, const Relative& rel, int64_t head, float root_hd,
                                        char* dynamic) {
    biases.finish(rel, head, root_hd, [&](int d, float x, int) { reinterpret_cast<float*>(dynamic)[d] = x; });
  }
  __device__ __forceinline__ void add(const int (&)[4], const f32x4_t&, bool) {}
  __device__ __forceinline__ void flush(int, int, float*) const {}
};

// The partial bucket sums of a workgroup: (head, position, tile, bucket).
__device__ __forceinline__ float* partial_of(float* partial, const Relative& rel, int64_t n_pa, int heads,
                                             int64_t n_tiles, int64_t pos, int64_t a, int64_t tile) {
  return partial + ((a * (n_pa / heads) + pos) * n_tiles + tile) * rel.n_buckets;
}

// What the four wavefronts of a split workgroup hold of one row's sums, added
// up in wavefront 0 in their order; `room` is LDS that no one reads any more.
template <int kN>
__device__ __forceinline__ void join_waves(float (&x)[kN], float* room) {
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  __syncthreads();
  if (wave > 0) {
#pragma unroll
    for (int k = 0; k < kN; ++k) room[((wave - 1) * kN + k) * 64 + lane] = x[k];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int k = 0; k < kN; ++k)
#pragma unroll
    for (int w = 0; w < kBwdWaves - 1; ++w) x[k] += room[(w * kN + k) * 64 + lane];
}

// kColumns > 0: at most two chunks of keys (T <= 128), with the bucket sums; 0: any number, without.
// kSplit (few_groups): a workgroup has 16 rows, and its wavefronts every fourth chunk of keys each.
template <bool kHalf, int HD, int kColumns, bool kSplit>
__global__ void __launch_bounds__(256)
relative_bwd_q_kernel(Rows q, Rows k, Rows v, Rows go, Relative rel, const int32_t* __restrict__ seq_lens, int heads,
                      int64_t T, int64_t n_pa, const float2* __restrict__ stats, float scale, float root_hd,
                      float* __restrict__ delta, RowsOut dq, float* __restrict__ partial) {
  using G = Geom<kHalf, HD>;
  static_assert(!kSplit || kColumns == 0, "split rows are long ones");
  using Tile = RowTile<HD, kSplit ? 64 : 256>;
  constexpr int kRows = kSplit ? 16 : kTile, kBufs = kSplit ? kBwdWaves : 2;
  __shared__ __attribute__((aligned(16))) uint16_t sk[kBufs][kTile * Tile::kPitch], sv[kBufs][kTile * Tile::kPitch];
  __shared__ __attribute__((aligned(16))) uint32_t sc[kBufs][kTile];
  __shared__ float row_of[4][kSplit ? kBwdWaves : 1][16];  // r, weight, rest and sum p dp of a wavefront's rows
  extern __shared__ __attribute__((aligned(16))) char dynamic[];
  const int64_t n_tiles = (T + kRows - 1) / kRows;
  const Item item = item_of(n_pa, heads, n_tiles);
  if (item.pa >= n_pa) return;
  const int64_t pa = item.pa, tile = item.tile, pos = pa / heads, a = pa % heads;
  TableStage biases;
  biases.request(rel);
  int64_t L = seq_lens[pos];
  L = L < 0 ? 0 : (L > T ? T : L);
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, l16 = lane % 16, g = lane / 16;
  const int64_t first = tile * kRows + (kSplit ? 0 : 16 * wave), i = first + l16;
  const bool writer = !kSplit || wave == 0;
  const bool live = i < L;
  BucketSums<kColumns> sums(rel, dynamic);
  float* part_sums = kColumns ? partial_of(partial, rel, n_pa, heads, n_tiles, pos, a, tile) : nullptr;
  f32x4_t acc[G::kDt];
#pragma unroll
  for (int dt = 0; dt < G::kDt; ++dt) acc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if (tile * kRows >= L) {  // no live row
    if (i < T && writer) {
      store_row<kHalf, HD, true>(dq.row(pos, a, i), g, acc, 0.f, false);
      if (g == 0) delta[pa * T + i] = 0.f;
    }
    if (kColumns)
      for (int b = threadIdx.x; b < rel.n_buckets; b += 256) part_sums[b] = 0.f;
    return;
  }
  const i32x4_t krs = rows_of(k, pos, a, L), vrs = rows_of(v, pos, a, L);
  struct Held {
    Tile k, v;
    uint32_t c;
  } held[kColumns ? 2 : 1];  // (both chunks of a short row are requested at once)
  auto fetch = [&](Held& h, int64_t kb) {
    h.k.fetch(krs, int32_t(kb));
    h.v.fetch(vrs, int32_t(kb));
    h.c = kSplit || threadIdx.x < kTile ? coords_of(rel, pos, T, kb + lane, L) : 0u;
  };
  auto stage = [&](const Held& h, int buf) {
    h.k.stage(sk[buf]);
    h.v.stage(sv[buf]);
    if (kSplit || threadIdx.x < kTile) sc[buf][lane] = h.c;
  };
  fetch(held[0], kSplit ? wave * kTile : 0);
  if (kColumns) fetch(held[kColumns != 0], kTile);
  biases.biases(rel, a);
  uint4 qf[G::kKs], gf[G::kKs];
  row_frags<kHalf, HD>(rows_of(q, pos, a, L), i, g, qf);
  row_frags<kHalf, HD>(rows_of(go, pos, a, L), i, g, gf);
  const float2 st = live ? stats[pa * T + i] : make_float2(0.f, INFINITY);
  const Side<true, kColumns ? 8 : 4> side(rel, coords_of(rel, pos, T, i, L), i < rel.n_latents);
  const int n_latents = int(rel.n_latents);
  sums.stage(biases, rel, a, root_hd, dynamic);
  const int64_t n_chunks = (L + kTile - 1) / kTile;
  if (!kSplit) stage(held[0], 0);
  if (kColumns) stage(held[kColumns != 0], 1);
  else if (!kSplit && n_chunks > 1) fetch(held[0], kTile);
  __syncthreads();

  const float c_log2 = scale * kLog2e;
  constexpr std::true_type full{};
  constexpr std::false_type part{};
  // p and dp of this lane's query with chunk c's keys, zeros past the n-th (a full chunk has no branch)
  auto pairs = [&](auto whole, int buf, int64_t c, int n, int (&at)[4][4], f32x4_t (&p)[4], f32x4_t (&dp)[4]) {
    constexpr bool kWhole = decltype(whole)::value;
    pair_offsets(side, n_latents, sc[buf], int(c * kTile), g, at);
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int t = 0; t < 4; ++t) p[tt][t] = sums.entry(at[tt][t]);
    products_onto<kHalf, HD>(sk[buf], kWhole ? kTile : n, l16, g, qf, p);
    products<kHalf, HD>(sv[buf], kWhole ? kTile : n, l16, g, gf, dp);
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const bool in = kWhole || 16 * tt + t < n - 4 * g;
        p[tt][t] = in ? __builtin_amdgcn_exp2f(fmaf(p[tt][t] - st.x, c_log2, -st.y)) : 0.f;
        dp[tt][t] = in ? dp[tt][t] : 0.f;
      }
  };
  float dl = 0.f;
  // sums of p and p dp (a chunk's terms among themselves first: fewer roundings of the long sum)
  auto sum_terms = [](const f32x4_t (&p)[4], const f32x4_t (&dp)[4], float& weight, float& sum) {
    float w = 0.f, s = 0.f;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        w += p[tt][t];
        s = fmaf(p[tt][t], dp[tt][t], s);
      }
    weight += w;
    sum += s;
  };
  auto row_sum = [](float x) { return sum_xor32(sum_xor16(x)); };
  // A weighted mean of dp.  By the weights' own sum and not by 1: what log2 l and the exponentials
  // round is common to a row, and where dp lies far from 0 that much of it would stay in every ds.
  auto mean_of = [](float weight, float sum) { return weight == 0.f ? 0.f : sum / weight; };
  ColumnScale<kHalf> cs;
  f32x4_t p[4], dp[4];
  int at[4][4];
  const bool working = first < L;  // wavefront-uniform: a live row here
  const int tail = int(L - (n_chunks - 1) * kTile);  // rows of the last chunk
  if constexpr (kColumns > 0) {
    float weight = 0.f;
    // ds (in p's place) into the buckets' sums and dq
    auto spread = [&](auto whole, int buf, int n, const int (&at)[4][4], f32x4_t (&p)[4], const f32x4_t (&dp)[4]) {
      constexpr bool kWhole = decltype(whole)::value;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        if (!kWhole && 16 * tt >= n) break;  // uniform
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          // (a key past the last one adds nothing, whatever delta is)
          const float x = p[tt][t] * (dp[tt][t] - dl);
          p[tt][t] = kWhole || 16 * tt + t < n - 4 * g ? x : 0.f;
        }
        sums.add(at[tt], p[tt], live);
      }
      cs.apply(p, acc);
      accumulate_parts<kHalf, HD>(sk[buf], kWhole ? kTile : n, l16, g, p, acc, acc);
    };
    if (n_chunks == 1) {
      if (working) {
        pairs(part, 0, 0, tail, at, p, dp);
        sum_terms(p, dp, weight, dl);
        dl = mean_of(row_sum(weight), row_sum(dl));
        spread(part, 0, tail, at, p, dp);
      }
    } else {  // two
      f32x4_t p1[4], dp1[4];
      if (working) {
        int at1[4][4];
        pairs(full, 0, 0, kTile, at, p, dp);
        sum_terms(p, dp, weight, dl);
        pairs(part, 1, 1, tail, at1, p1, dp1);
        sum_terms(p1, dp1, weight, dl);
        dl = mean_of(row_sum(weight), row_sum(dl));
        spread(full, 0, kTile, at, p, dp);
        spread(part, 1, tail, at1, p1, dp1);
      }
    }
  } else {
    // With r the row's mean of dp by the weights met so far: acc = sum p (dp - r) k, plain = sum p k,
    // rest = sum p (dp - r); r moves after each chunk's sums, and acc and rest with it.
    f32x4_t plain[G::kDt];
#pragma unroll
    for (int dt = 0; dt < G::kDt; ++dt) plain[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float r = 0.f, weight = 0.f;             // of the row
    float lane_weight = 0.f, rest = 0.f;     // of this lane's pairs
    auto move = [&](float by) {  // r by `by`, already counted in the weights so far
#pragma unroll
      for (int dt = 0; dt < G::kDt; ++dt)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[dt][t] = fmaf(by * (-1.f / kPScale<kHalf>), plain[dt][t], acc[dt][t]);
    };
    auto step = [&](auto whole, int64_t c, int n) {
      const int buf = kSplit ? wave : int(c & 1);
      if (kSplit) {
        stage(held[0], buf);
        if (c + kBwdWaves < n_chunks) fetch(held[0], (c + kBwdWaves) * kTile);
        wave_sync();
      }
      if (working) {
        pairs(whole, buf, c, n, at, p, dp);
        float w = 0.f, s = 0.f;
        sum_terms(p, dp, w, s);
        dl += s;
        const float chunk_weight = row_sum(w);
        weight += chunk_weight;
        // (any r will do, so a quick reciprocal; a row without a weight so far keeps 0)
        const float next =
            weight == 0.f ? 0.f : fmaf(fmaf(-r, chunk_weight, row_sum(s)), __builtin_amdgcn_rcpf(weight), r);
        const float by = next - r;
        r = next;
        move(by);
        float terms = 0.f;  // (a chunk's among themselves first)
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            dp[tt][t] = p[tt][t] * (dp[tt][t] - r);
            terms += dp[tt][t];
          }
        rest = fmaf(-by, lane_weight, rest) + terms;
        lane_weight += w;
        const int rows = decltype(whole)::value ? kTile : n;
        if constexpr (kHalf) {
          const float undo = chunk_scale(dp);
          f32x4_t chunk[G::kDt];
#pragma unroll
          for (int dt = 0; dt < G::kDt; ++dt) chunk[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) p[tt] *= kPScale<kHalf>;
          accumulate_two<kHalf, HD>(sk[buf], rows, l16, g, dp, chunk, p, plain);
#pragma unroll
          for (int dt = 0; dt < G::kDt; ++dt)
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[dt][t] = fmaf(chunk[dt][t], undo, acc[dt][t]);
        } else {
          accumulate_two<kHalf, HD>(sk[buf], rows, l16, g, dp, acc, p, plain);
        }
      }
      if (kSplit) {
        wave_sync();
        return;
      }
      if (c + 1 < n_chunks) {
        stage(held[0], buf ^ 1);  // (its readers met the barrier of the step before)
        if (c + 2 < n_chunks) fetch(held[0], (c + 2) * kTile);
      }
      __syncthreads();
    };
    int64_t c = kSplit ? wave : 0;
    for (; c + 1 < n_chunks; c += kSplit ? kBwdWaves : 1) step(full, c, kTile);
    if (c + 1 == n_chunks) step(part, c, tail);
    cs.s = 1.f;
    rest = row_sum(rest);
    dl = row_sum(dl);
    if constexpr (kSplit) {
      // the wavefronts' sums brought to one r, the mean of all, and added up in their order
      if (g == 0) {
        row_of[0][wave][l16] = r;
        row_of[1][wave][l16] = weight;
        row_of[2][wave][l16] = rest;
        row_of[3][wave][l16] = dl;
      }
      __syncthreads();
      float all = 0.f, mean = 0.f;
      dl = 0.f;
#pragma unroll
      for (int w = 0; w < kBwdWaves; ++w) {
        dl += row_of[3][w][l16];
        all += row_of[1][w][l16];
        mean += fmaf(row_of[0][w][l16], row_of[1][w][l16], row_of[2][w][l16]);
      }
      mean = mean_of(all, mean);
      move(mean - r);
      float x[8 * G::kDt + 1];
      x[8 * G::kDt] = fmaf(r - mean, weight, rest);
#pragma unroll
      for (int k = 0; k < 4 * G::kDt; ++k) {
        x[k] = acc[k / 4][k % 4];
        x[4 * G::kDt + k] = plain[k / 4][k % 4];
      }
      static_assert((kBwdWaves - 1) * sizeof(x) * 64 <= sizeof(sk), "the tiles' LDS holds them");
      join_waves(x, reinterpret_cast<float*>(sk));
      if (wave > 0) return;
      r = mean;
      weight = all;
      rest = x[8 * G::kDt];
#pragma unroll
      for (int k = 0; k < 4 * G::kDt; ++k) {
        acc[k / 4][k % 4] = x[k];
        plain[k / 4][k % 4] = x[4 * G::kDt + k];
      }
    }
    const float by = mean_of(weight, rest);
    move(by);
    // (where a dp is infinite, delta is the plain sum: r has met inf - inf)
    dl = __builtin_isfinite(dl) ? r + by : dl;
  }
  if (i < T) {
    store_row<kHalf, HD, true>(dq.row(pos, a, i), g, acc, scale / cs.s, live);
    if (g == 0) delta[pa * T + i] = live ? dl : 0.f;
  }
  if constexpr (kColumns > 0) {
    __syncthreads();
    sums.flush(L - tile * kTile < kTile ? int(L - tile * kTile) : kTile, 16, part_sums);
  }
}

// dbias of one (head, bucket): the head's partial sums, each thread a fixed
// stride of them, joined in a fixed order.  The query pass's are added up by
// workgroups of the key pass's launch (a launch of their own takes 4 us), the
// key pass's by one after it.
__device__ __forceinline__ void sum_bias(const float* __restrict__ partial, int64_t n_parts, int n_buckets,
                                         uint32_t which, float* __restrict__ dbias) {
  __shared__ float sums[256];
  const int64_t a = which / n_buckets, b = which % n_buckets;
  float sum = 0.f;
  for (int64_t i = threadIdx.x; i < n_parts; i += 256) sum += partial[(a * n_parts + i) * n_buckets + b];
  sums[threadIdx.x] = sum;
  for (int o = 128; o > 0; o >>= 1) {
    __syncthreads();
    if (int(threadIdx.x) < o) sums[threadIdx.x] += sums[threadIdx.x + o];
  }
  if (threadIdx.x == 0) dbias[which] = sums[0];
}

__global__ void __launch_bounds__(256)
relative_bias_sum_kernel(const float* __restrict__ partial, int64_t n_parts, int n_buckets, float* __restrict__ dbias) {
  sum_bias(partial, n_parts, n_buckets, blockIdx.x, dbias);
}

// kColumns > 0: with the bucket sums; 0: with the workgroups that add up the query pass's.
// kSplit (few_groups): a workgroup has 16 rows, and its wavefronts every fourth chunk of queries each.
template <bool kHalf, int HD, int kColumns, bool kSplit>
__global__ void __launch_bounds__(256)
relative_bwd_kv_kernel(Rows q, Rows k, Rows v, Rows go, Relative rel, const int32_t* __restrict__ seq_lens, int heads,
                       int64_t T, int64_t n_pa, const float2* __restrict__ stats, float scale, float root_hd,
                       const float* __restrict__ delta, RowsOut dk, RowsOut dv, float* __restrict__ partial,
                       float* __restrict__ dbias, uint32_t n_item_groups) {
  if (!kColumns && blockIdx.x >= n_item_groups) {  // the workgroups after the items
    sum_bias(partial, n_pa / heads * ((T + kTile - 1) / kTile), rel.n_buckets, blockIdx.x - n_item_groups, dbias);
    return;
  }
  using G = Geom<kHalf, HD>;
  static_assert(!kSplit || kColumns > 0, "split rows are long ones");
  using Tile = RowTile<HD, kSplit ? 64 : 256>;
  constexpr int kRows = kSplit ? 16 : kTile, kBufs = kSplit ? kBwdWaves : 2;
  __shared__ __attribute__((aligned(16))) uint16_t sq[kBufs][kTile * Tile::kPitch], sg[kBufs][kTile * Tile::kPitch];
  __shared__ __attribute__((aligned(16))) float sm[kBufs][kTile], sl[kBufs][kTile], sd[kBufs][kTile];
  __shared__ __attribute__((aligned(16))) uint32_t sc[kBufs][kTile];
  extern __shared__ __attribute__((aligned(16))) char dynamic[];
  const int64_t n_tiles = (T + kRows - 1) / kRows;
  const Item item = item_of(n_pa, heads, n_tiles);
  if (item.pa >= n_pa) return;
  const int64_t pa = item.pa, tile = item.tile, pos = pa / heads, a = pa % heads;
  TableStage biases;
  biases.request(rel);
  int64_t L = seq_lens[pos];
  L = L < 0 ? 0 : (L > T ? T : L);
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, l16 = lane % 16, g = lane / 16;
  const int64_t first = tile * kRows + (kSplit ? 0 : 16 * wave), j = first + l16;
  const bool live = j < L;
  f32x4_t ak[G::kDt], av[G::kDt], ak_lo[G::kDt], av_lo[G::kDt];
#pragma unroll
  for (int dt = 0; dt < G::kDt; ++dt) ak[dt] = av[dt] = ak_lo[dt] = av_lo[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  ColumnScale<kHalf> cs;
  BucketSums<kColumns> sums(rel, dynamic);
  float* part_sums = kColumns ? partial_of(partial, rel, n_pa, heads, n_tiles, pos, a, tile) : nullptr;
  if (tile * kRows < L) {  // workgroup-uniform
    const i32x4_t qrs = rows_of(q, pos, a, L), grs = rows_of(go, pos, a, L);
    struct Held {
      Tile q, g;
      float m, l, d;
      uint32_t c;
    } held[kColumns ? 1 : 2];  // (both chunks of a short row are requested at once)
    auto fetch = [&](Held& h, int64_t qb) {
      h.q.fetch(qrs, int32_t(qb));
      h.g.fetch(grs, int32_t(qb));
      if (kSplit || threadIdx.x < kTile) {
        const int64_t i = qb + lane;
        const bool in = i < L;
        const float2 st = in ? stats[pa * T + i] : make_float2(0.f, INFINITY);
        h.m = st.x, h.l = st.y;
        h.d = in ? delta[pa * T + i] : 0.f;
        h.c = coords_of(rel, pos, T, i, L);
      }
    };
    auto stage = [&](const Held& h, int buf) {
      h.q.stage(sq[buf]);
      h.g.stage(sg[buf]);
      if (kSplit || threadIdx.x < kTile) {
        sm[buf][lane] = h.m;
        sl[buf][lane] = h.l;
        sd[buf][lane] = h.d;
        sc[buf][lane] = h.c;
      }
    };
    fetch(held[0], kSplit ? wave * kTile : 0);
    if (!kColumns) fetch(held[!kColumns], kTile);
    biases.biases(rel, a);
    uint4 kf[G::kKs], vf[G::kKs];
    row_frags<kHalf, HD>(rows_of(k, pos, a, L), j, g, kf);
    row_frags<kHalf, HD>(rows_of(v, pos, a, L), j, g, vf);
    const Side<false, kColumns ? 8 : 4> side(rel, coords_of(rel, pos, T, j, L), j < rel.n_latents);
    const int n_latents = int(rel.n_latents);
    sums.stage(biases, rel, a, root_hd, dynamic);
    const float c_log2 = scale * kLog2e;
    if (!kSplit) stage(held[0], 0);
    if (!kColumns) stage(held[!kColumns], 1);
    else if (!kSplit && kTile < L) fetch(held[0], kTile);
    __syncthreads();
    auto chunk = [&](auto whole, int64_t qb, int n) {
      constexpr bool kWhole = decltype(whole)::value;  // (a full chunk has no branch)
      const int buf = kSplit ? wave : int(qb / kTile & 1);
      if (kSplit) {
        stage(held[0], buf);
        if (qb + kBwdWaves * kTile < L) fetch(held[0], qb + kBwdWaves * kTile);
        wave_sync();
      }
      if (first < L) {  // wavefront-uniform
        f32x4_t p[4], ds[4];
        int at[4][4];
        pair_offsets(side, n_latents, sc[buf], int(qb), g, at);  // (a latent key's pairs keep its own entry)
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int t = 0; t < 4; ++t) p[tt][t] = sums.entry(at[tt][t]);
        products_onto<kHalf, HD>(sq[buf], kWhole ? kTile : n, l16, g, kf, p);
        products<kHalf, HD>(sg[buf], kWhole ? kTile : n, l16, g, vf, ds);
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const f32x4_t m4 = *reinterpret_cast<const f32x4_t*>(&sm[buf][16 * tt + 4 * g]);
          const f32x4_t l4 = *reinterpret_cast<const f32x4_t*>(&sl[buf][16 * tt + 4 * g]);
          const f32x4_t d4 = *reinterpret_cast<const f32x4_t*>(&sd[buf][16 * tt + 4 * g]);
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const bool in = kWhole || 16 * tt + t < n - 4 * g;
            p[tt][t] = in ? __builtin_amdgcn_exp2f(fmaf(p[tt][t] - m4[t], c_log2, -l4[t])) : 0.f;
            ds[tt][t] = in ? p[tt][t] * (ds[tt][t] - d4[t]) : 0.f;
          }
        }
        if constexpr (kColumns > 0) {
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) {
            if (!kWhole && 16 * tt >= n) break;  // uniform
            sums.add(at[tt], ds[tt], live);
          }
        }
        if constexpr (kHalf) {
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) p[tt] *= kPScale<kHalf>;
        }
        accumulate_parts<kHalf, HD>(sg[buf], kWhole ? kTile : n, l16, g, p, av, av_lo);
        cs.apply(ds, ak, ak_lo);
        accumulate_parts<kHalf, HD>(sq[buf], kWhole ? kTile : n, l16, g, ds, ak, ak_lo);
      }
      if (kSplit) wave_sync();
      if (!kColumns || kSplit) return;
      if (qb + kTile < L) {
        stage(held[0], buf ^ 1);  // (its readers met the barrier of the chunk before)
        if (qb + 2 * kTile < L) fetch(held[0], qb + 2 * kTile);
      }
      __syncthreads();
    };
    const int64_t last = (L - 1) / kTile * kTile;
    int64_t qb = kSplit ? wave * kTile : 0;
    for (; qb < last; qb += kSplit ? kBwdWaves * kTile : kTile) chunk(std::true_type{}, qb, kTile);
    if (qb == last) chunk(std::false_type{}, last, int(L - last));
    join_parts(ak, ak_lo);
    join_parts(av, av_lo);
    if constexpr (kSplit) {
      float x[8 * G::kDt];
#pragma unroll
      for (int k = 0; k < 4 * G::kDt; ++k) {
        x[k] = ak[k / 4][k % 4] / cs.s;
        x[4 * G::kDt + k] = av[k / 4][k % 4];
      }
      static_assert((kBwdWaves - 1) * sizeof(x) * 64 <= sizeof(sq), "the tiles' LDS holds them");
      join_waves(x, reinterpret_cast<float*>(sq));
      cs.s = 1.f;
#pragma unroll
      for (int k = 0; k < 4 * G::kDt; ++k) {
        ak[k / 4][k % 4] = x[k];
        av[k / 4][k % 4] = x[4 * G::kDt + k];
      }
    }
    sums.flush(L - tile * kRows < kRows ? int(L - tile * kRows) : kRows, kSplit ? 0 : 16, part_sums);
  } else if (kColumns) {
    for (int b = threadIdx.x; b < rel.n_buckets; b += 256) part_sums[b] = 0.f;
  }
  if (j < T && (!kSplit || wave == 0)) {
    store_row<kHalf, HD, true>(dk.row(pos, a, j), g, ak, scale / cs.s, live);
    store_row<kHalf, HD, true>(dv.row(pos, a, j), g, av, 1.f / kPScale<kHalf>, live);
  }
}

// static LDS of the passes (the key pass's, the larger)
template <int HD>
constexpr size_t static_lds(bool split) {
  const int bufs = split ? kBwdWaves : 2;
  return size_t(2 * bufs * kTile * (HD + 8)) * 2 + bufs * kTile * 4 * 4 + 1024;
}

// the dynamic LDS that a kernel may ask for, set once per kernel and device
template <auto kKernel>
bool allow_lds(size_t bytes) {
  static std::atomic<bool> done[64] = {};  // (threads may launch at once; setting it twice does no harm)
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) return false;
  if (dev < 64 && done[dev]) return true;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(kKernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                          int(bytes)) != hipSuccess)
    return false;
  if (dev < 64) done[dev] = true;
  return true;
}

template <bool kHalf, int HD>
int32_t launch(const Rows& q, const Rows& k, const Rows& v, const Rows& go, const Relative& rel,
               const int32_t* seq_lens, int64_t n_pos, int heads, int64_t t, const float2* stats, float* delta,
               float* partial, const RowsOut& dq, const RowsOut& dk, const RowsOut& dv, float* dbias, hipStream_t st) {
  const int n_disp = rel.nq * rel.nr;
  bool split = few_groups(n_pos, heads, t, HD);
  auto total = [&](int columns) {
    return static_lds<HD>(split) + table_bytes(n_disp, 8) + column_bytes(rel.n_buckets, columns);
  };
  if (split && total(16) > kLdsBytes) split = false;
  const int64_t rows = split ? 16 : kTile, n_tiles = (t + rows - 1) / rows, n_pa = n_pos * heads;
  const int64_t grid = item_grid(n_pos, heads, n_tiles);
  if (grid + heads * rel.n_buckets > 2147483647LL) return MANTIS_E_ARG;
  const float root = sqrtf(float(HD)), scale = 1.f / root;
  // Columns per wavefront: 64 where that table leaves room for three workgroups on a CU
  // (with 64 dims, whose registers allow two, for two; with 64 split, for one), else 32 with the lane groups in two
  // turns where two fit, else 16 or 8 in four or eight.  With 64 / 32 / 16 columns: the query
  // pass of 192 positions of 44-124 rows, 32 dims, 28 buckets, 31 / 25 / 28 us; the key pass of
  // 64 positions of 150-300 rows 50 / 43 / 59, of 16 positions of 511-1,021 rows, 16
  // dims, 52 buckets, 258 / 171 / 185, of two lines of 2,049-4,096, 64 dims, 32 buckets, 352 / 396 / 475.
  const size_t fixed = static_lds<HD>(split), wide = kLdsBytes / (HD < 64 ? 3 : split ? 1 : 2);
  const int columns = total(64) <= wide ? 64 : total(32) <= kLdsBytes / 2 ? 32 : total(16) <= kLdsBytes ? 16 : 8;
  if (total(columns) > kLdsBytes) return MANTIS_E_ARG;
  const size_t sums_lds = total(columns) - fixed, plain_lds = table_bytes(n_disp, 4);
  const bool few = t <= 2 * kTile;  // the bucket sums go with the query pass
  auto passes = [&](auto query, auto key, bool allowed) {
    if (!allowed) return false;
    query<<<unsigned(grid), 256, few ? sums_lds : plain_lds, st>>>(q, k, v, go, rel, seq_lens, heads, t, n_pa, stats,
                                                                   scale, root, delta, dq, partial);
    key<<<unsigned(few ? grid + heads * rel.n_buckets : grid), 256, few ? plain_lds : sums_lds, st>>>(
        q, k, v, go, rel, seq_lens, heads, t, n_pa, stats, scale, root, delta, dk, dv, partial, dbias, uint32_t(grid));
    return true;
  };
  const size_t most = kLdsBytes - fixed;
#define MANTIS_PASSES(C)                                                                                         \
  (few     ? passes(relative_bwd_q_kernel<kHalf, HD, C, false>, relative_bwd_kv_kernel<kHalf, HD, 0, false>,     \
                    allow_lds<relative_bwd_q_kernel<kHalf, HD, C, false>>(most))                                 \
   : split ? passes(relative_bwd_q_kernel<kHalf, HD, 0, true>, relative_bwd_kv_kernel<kHalf, HD, C, true>,       \
                    allow_lds<relative_bwd_q_kernel<kHalf, HD, 0, true>>(most) &&                                \
                        allow_lds<relative_bwd_kv_kernel<kHalf, HD, C, true>>(most))                             \
           : passes(relative_bwd_q_kernel<kHalf, HD, 0, false>, relative_bwd_kv_kernel<kHalf, HD, C, false>,     \
                    allow_lds<relative_bwd_kv_kernel<kHalf, HD, C, false>>(most)))
  const bool queued = columns == 64   ? MANTIS_PASSES(64)
                      : columns == 32 ? MANTIS_PASSES(32)
                      : columns == 16 ? MANTIS_PASSES(16)
                                      : MANTIS_PASSES(8);
#undef MANTIS_PASSES
  if (!queued) return MANTIS_E_LAUNCH;
  if (!few)
    relative_bias_sum_kernel<<<unsigned(heads * rel.n_buckets), 256, 0, st>>>(partial, n_pos * n_tiles, rel.n_buckets,
                                                                             dbias);
  return launched();
}

}  // namespace
}  // namespace mantis

using namespace mantis;

extern "C" int64_t mantis_relative_attention_backward_workspace(int64_t n_pos, int32_t heads, int64_t t,
                                                                int64_t n_buckets) {
  if (n_pos <= 0 || heads <= 0 || t <= 0 || n_buckets <= 0) return 0;
  // delta, then the partial bias sums
  const int64_t rows = few_groups(n_pos, heads, t, 16) ? 16 : kTile;  // (enough for every width)
  return 4 * (n_pos * heads * t + n_pos * heads * ((t + rows - 1) / rows) * n_buckets);
}

extern "C" int32_t mantis_relative_attention_backward(
    const void* q, const int64_t* qs, const void* k, const int64_t* ks, const void* v, const int64_t* vs,
    const void* grad_out, const int64_t* gs, const float* stats, int32_t dtype, const float* bias, int64_t n_buckets,
    const int32_t* coords, const int32_t* buckets, int64_t nq, int64_t nr, int64_t n_latents, const int32_t* seq_lens,
    int64_t n_pos, int32_t heads, int64_t t, int32_t hd, void* workspace, int64_t workspace_bytes, void* dq,
    const int64_t* dqs, void* dk, const int64_t* dks, void* dv, const int64_t* dvs, float* dbias, int32_t* err_flag,
    void* stream) {
  if (n_pos < 0 || t < 0 || heads <= 0) return MANTIS_E_ARG;
  if (n_pos == 0 || t == 0) return MANTIS_OK;
  if (!q || !k || !v || !grad_out || !stats || !seq_lens || !workspace || !dq || !dk || !dv || !dbias) return MANTIS_E_ARG;
  if (!qs || !ks || !vs || !gs || !dqs || !dks || !dvs) return MANTIS_E_ARG;
  if ((hd != 16 && hd != 32 && hd != 64) || (dtype != MANTIS_BF16 && dtype != MANTIS_F16)) return MANTIS_E_ARG;
  if (nq > kMaxDisplacements || nr > kMaxDisplacements || n_buckets > kMaxBuckets) return MANTIS_E_ARG;
  for (const int64_t* st : {qs, ks, vs, gs, dqs, dks, dvs}) {
    if (st[3] != 1) return MANTIS_E_ARG;
    if ((st[0] | st[1] | st[2]) % 8) return MANTIS_E_ARG;
  }
  for (const int64_t* st : {qs, ks, vs, gs})  // (buffer descriptors, as in the forward)
    if (st[2] < hd || st[2] >= 8192 || t * st[2] * 2 > 2147483647LL) return MANTIS_E_ARG;
  for (const void* ptr : {q, k, v, grad_out, static_cast<const void*>(dq), static_cast<const void*>(dk),
                          static_cast<const void*>(dv), static_cast<const void*>(stats),
                          static_cast<const void*>(workspace)})
    if (!aligned16(ptr)) return MANTIS_E_ARG;
  const Relative rel{coords, buckets, bias, int(nq), int(nr), int(n_buckets), n_latents, err_flag};
  if (!good_relative(rel, t)) return MANTIS_E_ARG;
  if (workspace_bytes < mantis_relative_attention_backward_workspace(n_pos, heads, t, n_buckets)) return MANTIS_E_ARG;
  auto rows = [](const void* ptr, const int64_t* st) {
    return Rows{static_cast<const uint16_t*>(ptr), st[0], st[1], st[2]};
  };
  auto outs = [](void* ptr, const int64_t* st) { return RowsOut{static_cast<uint16_t*>(ptr), st[0], st[1], st[2]}; };
  const Rows Q = rows(q, qs), K = rows(k, ks), V = rows(v, vs), GO = rows(grad_out, gs);
  const RowsOut DQ = outs(dq, dqs), DK = outs(dk, dks), DV = outs(dv, dvs);
  const float2* sp = reinterpret_cast<const float2*>(stats);
  float* delta = static_cast<float*>(workspace);
  float* partial = delta + n_pos * heads * t;
  hipStream_t st = as_stream(stream);
#define MANTIS_BWD(HD_)                                                                                               \
  return dtype == MANTIS_F16 ? launch<true, HD_>(Q, K, V, GO, rel, seq_lens, n_pos, heads, t, sp, delta, partial, DQ, \
                                                 DK, DV, dbias, st)                                                   \
                             : launch<false, HD_>(Q, K, V, GO, rel, seq_lens, n_pos, heads, t, sp, delta, partial, DQ, \
                                                  DK, DV, dbias, st)
  if (hd == 16) MANTIS_BWD(16);
  if (hd == 32) MANTIS_BWD(32);
  MANTIS_BWD(64);
#undef MANTIS_BWD
}
