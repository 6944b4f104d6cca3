// Ragged attention with a learned bias by relative position, on 16-bit MFMA
// for gfx950.  For the live rows i and keys j < L of a position and head:
//   s_ij = q_i . k_j / sqrt(hd) + bias[bucket(i, j)],  out_i = softmax_j(s_ij) v_j,
//   lse_i = log sum_j exp s_ij
// A live row whose every key has bias -inf gives zeros and lse -inf; rows past L
// give zeros and lse 0.
//
// One workgroup serves an item (position, head, query tile of 4 kSub 16 rows);
// each of its four wavefronts owns kSub 16-query sub-tiles and the keys stream
// through LDS in 64-key chunks, double-buffered, the next one's rows in
// registers meanwhile (where such tiles are few, few_groups, an item has 16
// queries, each wavefront its own chunks, and their sums join at the end).  The
// transposed products S^T = K Q^T and O^T += V^T P^T keep a lane on one query, and
// a score fragment is the next product's B operand as it stands.  The bias is the
// score product's C operand (relative_bias.hpp), so adding it costs the lookup alone.
//
// Softmax: p = exp2(c (s - m)), c = log2(e) / sqrt(hd), over the raw scores
// (bias * sqrt(hd) included), in fp32 and with the difference first, so a row
// of scores at the type's lowest value is still uniform; m moves only when a
// score passes it by more than 8 in log2 units.  The probabilities enter the
// value product rounded to 16 bits, half a step of each as the output rounds once
// more: 2^-8 of it in bf16, 2^-11 in fp16 and there, under 2^-14 beside a largest one of 1
// to 2^8, 2^-25 outright (under that it counts as 0, beside an infinite value too).  The
// output is divided by the sum of the rounded ones, so a row of one key is that key's
// value, and lse is the log of the unrounded fp32 sum.
//
// Bound by the pairs' vector work (table offset, lookup, maximum, exp2, sum, pack:
// some 20 instructions for each, against 4 hd matrix operations), not by memory.
// Measured: 512 positions of 44-124 rows, 4 heads, 32 dims, 27 us (q, k, v and out
// at the rate of a large copy: 10); 192 of them 14.6; 16 of 511-1,021 rows, 8 heads
// of 16 dims, 58; two lines of 2,049-4,096 rows, 8 heads of 64 dims, 131.
#include <type_traits>

#include "attention_rows.hpp"
#include "relative_bias.hpp"

namespace mantis {
namespace {

constexpr int kWaves = 4;
constexpr int kKChunk = 64;
constexpr float kLazyLog2 = 8.f;  // probabilities up to 2^8 before the reference point moves

struct Operand {  // (P, A, T, hd): base and element strides
  const uint16_t* p;
  int64_t sp, sa, st;
};

// kSplit (kSub 1): an item has 16 queries, and its wavefronts every fourth chunk of keys each.
template <bool kHalf, int HD, int kSub, bool kSplit>
__global__ void __launch_bounds__(256)
relative_attention_kernel(Operand q, Operand k, Operand v, Relative rel, const int32_t* __restrict__ seq_lens,
                          int heads, int64_t T, uint16_t* __restrict__ out, int64_t osp, int64_t osa, int64_t ost,
                          float* __restrict__ lse, float2* __restrict__ stats, float c_log2, float root_hd, int64_t n_pa) {
  constexpr int kQTile = (kSplit ? 1 : kWaves) * 16 * kSub;
  constexpr int kStagers = kSplit ? 64 : 256, kBufs = kSplit ? kWaves : 2;
  constexpr int kKPitch = HD + 8;              // 16-bit elements per staged K or V row
  constexpr int kKs = HD < 32 ? 1 : HD / 32;   // K steps of the score product
  constexpr int kDt = HD / 16;                 // 16-dim output tiles
  constexpr int kPieces = kKChunk * HD / 8;    // 16-byte pieces of a chunk's K (or V) rows
  constexpr int kPer = kPieces < kStagers ? 1 : kPieces / kStagers;
  extern __shared__ float table[];  // the head's bias per displacement
  __shared__ __attribute__((aligned(16))) uint16_t sk[kBufs][kKChunk * kKPitch];
  __shared__ __attribute__((aligned(16))) uint16_t sv[kBufs][kKChunk * kKPitch];
  __shared__ __attribute__((aligned(16))) uint32_t sc[kBufs][kKChunk];
  const int64_t n_qt = (T + kQTile - 1) / kQTile;
  const Item item = item_of(n_pa, heads, n_qt);
  if (item.pa >= n_pa) return;
  const int64_t pa = item.pa, qt = item.tile, p = pa / heads, a = pa % heads;
  TableStage bias_table;
  bias_table.request(rel);
  int64_t L = seq_lens[p];
  L = L < 0 ? 0 : (L > T ? T : L);
  const int64_t q0 = qt * kQTile;
  uint16_t* op = out + p * osp + a * osa;
  float* lp = lse + (p * heads + a) * T;
  float2* sp = stats + (p * heads + a) * T;

  if (q0 >= L) {  // a tile past the live rows
    for (int i = threadIdx.x; i < kQTile * (HD / 8); i += 256) {
      const int64_t row = q0 + i / (HD / 8);
      const int c = (i % (HD / 8)) * 8;
      if (row < T) {
        *reinterpret_cast<uint4*>(op + row * ost + c) = make_uint4(0u, 0u, 0u, 0u);
        if (c == 0) {
          lp[row] = 0.f;
          sp[row] = make_float2(0.f, INFINITY);
        }
      }
    }
    return;
  }

  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int l16 = lane % 16, g = lane / 16;
  using FR = Frag<kHalf>;
  // rows through buffer descriptors over the live rows: one at or past L reads
  // zeros without a memory access
  const i32x4_t qrs = rows_rsrc(q.p + p * q.sp + a * q.sa, uint32_t(q.st * 2), uint32_t(L));
  const i32x4_t krs = rows_rsrc(k.p + p * k.sp + a * k.sa, uint32_t(k.st * 2), uint32_t(L));
  const i32x4_t vrs = rows_rsrc(v.p + p * v.sp + a * v.sa, uint32_t(v.st * 2), uint32_t(L));
  // the K slots of a score step: dims 32 ks + 8 g .. +7 (HD = 16: lanes g >= 2 hold zeros on both sides)
  auto kdim = [&](int ks) { return HD < 32 ? 8 * (g & 1) : 32 * ks + 8 * g; };
  const bool upper = HD < 32 && g >= 2;
  typename FR::vec qf[kSub][kKs];
  int64_t qrow[kSub];
#pragma unroll
  for (int j = 0; j < kSub; ++j) {
    qrow[j] = q0 + (kSplit ? 0 : kWaves * j + wave) * 16 + l16;  // (sub-tiles dealt over the wavefronts)
#pragma unroll
    for (int ks = 0; ks < kKs; ++ks) {
      uint4 u = row_load16(qrs, int32_t(qrow[j]), 2 * kdim(ks));
      if (upper) u = make_uint4(0u, 0u, 0u, 0u);
      qf[j][ks] = FR::cast(u);
    }
  }

  // staging role of this thread: kPer 16-byte pieces of a chunk's K and V rows, a row's coordinates.
  // kSub 2 holds a position of at most two chunks: both are requested at once and met without a
  // barrier in between; else the next chunk's are in registers while one is met.
  constexpr bool kAll = kSub == 2;
  const int stager = int(threadIdx.x) % kStagers;
  struct Pieces {
    uint4 k[kPer], v[kPer];
    uint32_t c;
  } held[kAll ? 2 : 1];
  auto fetch = [&](Pieces& h, int64_t kb) {
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const int i = stager + kStagers * r;
      const int32_t row = i < kPieces ? int32_t(kb) + i / (HD / 8) : -1;
      h.k[r] = row_load16(krs, row, 16 * (i % (HD / 8)));
      h.v[r] = row_load16(vrs, row, 16 * (i % (HD / 8)));
    }
    h.c = stager < kKChunk ? coords_of(rel, p, T, kb + stager, L) : 0u;
  };
  auto stage = [&](const Pieces& h, int buf) {
    if (stager < kKChunk) sc[buf][stager] = h.c;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const int i = stager + kStagers * r;
      if (i >= kPieces) break;
      const int st_key = i / (HD / 8), st_d = 8 * (i % (HD / 8));
      *reinterpret_cast<uint4*>(&sk[buf][st_key * kKPitch + st_d]) = h.k[r];
      *reinterpret_cast<uint4*>(&sv[buf][st_key * kKPitch + st_d]) = h.v[r];
    }
  };
  fetch(held[0], kSplit ? wave * kKChunk : 0);
  if (kAll) fetch(held[kAll], kKChunk);
  bias_table.biases(rel, a);
  uint32_t qc[kSub];
#pragma unroll
  for (int j = 0; j < kSub; ++j) qc[j] = coords_of(rel, p, T, qrow[j], L);
  bias_table.finish(rel, a, root_hd, [&](int i, float x, int) { table[i] = x; });
  const Side<true, 4> side[2] = {{rel, qc[0], qrow[0] < rel.n_latents},
                                {rel, qc[kSub - 1], qrow[kSub - 1] < rel.n_latents}};
  const int n_latents = int(rel.n_latents);

  // per sub-tile: the exponent's reference point (raw-score units), O^T tiles,
  // the rounded probabilities' sum (a product with an all-ones A operand, every
  // row of it) and this lane's share of the unrounded sum
  float m[kSub], thr[kSub], lreal[kSub];
  const float lazy_raw = kLazyLog2 / c_log2;
  f32x4_t o[kSub][kDt], lsum[kSub];
#pragma unroll
  for (int j = 0; j < kSub; ++j) {
    m[j] = thr[j] = -INFINITY;
    lreal[j] = 0.f;
    lsum[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < kDt; ++dt) o[j][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t one2 = FR::pack_unit(1.f, 1.f);
  const typename FR::vec ones = FR::cast(make_uint4(one2, one2, one2, one2));

  // one chunk for the first kNJ sub-tiles (those with a live query)
  auto chunk = [&](auto nj, auto masked, int buf, int64_t kb, bool more) {
    constexpr int kNJ = decltype(nj)::value;
    if (kSplit) {
      stage(held[0], buf);
      if (kb + kWaves * kKChunk < L) fetch(held[0], kb + kWaves * kKChunk);
      wave_sync();
    } else if (!kAll && more) {
      fetch(held[0], kb + kKChunk);
    }
    if constexpr (kNJ > 0) {
      // keys of the last chunk: tiles of 16 past the last one are left out (uniform)
      constexpr bool kMasked = decltype(masked)::value;
      const int n = kMasked ? int(L - kb) : kKChunk;
      f32x4_t s[kNJ][4];
#pragma unroll
      for (int j = 0; j < kNJ; ++j) {
        int at[4][4];
        pair_offsets(side[j], n_latents, sc[buf], int(kb), g, at);
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          s[j][tt] = f32x4_t{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          if (kMasked && 16 * tt >= n) continue;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            s[j][tt][t] = entry(table, at[tt][t]);
            if (kMasked) s[j][tt][t] = 16 * tt + t < n - 4 * g ? s[j][tt][t] : -INFINITY;
          }
        }
      }
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        if (kMasked && 16 * tt >= n) {
          around_products();
          continue;
        }
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks) {
          uint4 ku = *reinterpret_cast<const uint4*>(&sk[buf][(16 * tt + l16) * kKPitch + kdim(ks)]);
          if (upper) ku = make_uint4(0u, 0u, 0u, 0u);
          const typename FR::vec kf = FR::cast(ku);
#pragma unroll
          for (int j = 0; j < kNJ; ++j) s[j][tt] = mfma16x16x32(kf, qf[j][ks], s[j][tt]);
        }
      }
      typename FR::vec pf[kNJ][2];
#pragma unroll
      for (int j = 0; j < kNJ; ++j) {
        float lmax = s[j][0][0];
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int t = 0; t < 4; ++t) lmax = fmaxf(lmax, s[j][tt][t]);
        if (__builtin_amdgcn_ballot_w64(lmax > thr[j])) {  // wavefront-uniform
          const float cmax = max_xor32(max_xor16(fmaxf(m[j], lmax)));
          // (a row without a finite score keeps m = -inf and its zero sums)
          const float alpha = m[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[j] - cmax) * c_log2);
          m[j] = cmax;
          thr[j] = cmax + lazy_raw;
          lreal[j] *= alpha;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            lsum[j][t] *= alpha;
#pragma unroll
            for (int dt = 0; dt < kDt; ++dt) o[j][dt][t] *= alpha;
          }
        }
        const float m0 = m[j] == -INFINITY ? 0.f : m[j];
        uint32_t pw[4][2];
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          pw[tt][0] = pw[tt][1] = 0u;
          if (kMasked && 16 * tt >= n) continue;
          float pr[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            pr[t] = __builtin_amdgcn_exp2f((s[j][tt][t] - m0) * c_log2);
            lreal[j] += pr[t];
          }
          pw[tt][0] = FR::pack_unit(pr[0], pr[1]);
          pw[tt][1] = FR::pack_unit(pr[2], pr[3]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
          pf[j][h] = FR::cast(make_uint4(pw[2 * h][0], pw[2 * h][1], pw[2 * h + 1][0], pw[2 * h + 1][1]));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (kMasked && 32 * h >= n) {
          around_products();
          continue;
        }
#pragma unroll
        for (int dt = 0; dt < kDt; ++dt) {
          const typename FR::vec vf = FR::cast(transposed_frag<HD>(sv[buf], h, dt, l16, g));
#pragma unroll
          for (int j = 0; j < kNJ; ++j) o[j][dt] = mfma16x16x32(vf, pf[j][h], o[j][dt]);
        }
#pragma unroll
        for (int j = 0; j < kNJ; ++j) lsum[j] = mfma16x16x32(ones, pf[j][h], lsum[j]);
      }
    }
    if (kSplit) wave_sync();
    if (kAll || kSplit) return;
    if (more) stage(held[0], buf ^ 1);
    __syncthreads();
  };

  const int64_t n_chunks = (L + kKChunk - 1) / kKChunk;
  auto run = [&](auto nj) {
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    const int64_t last = n_chunks - 1;  // only the last chunk can hold padding keys
    if constexpr (kSplit) {
      int64_t ch = wave;
      for (; ch < last; ch += kWaves) chunk(nj, no, wave, ch * kKChunk, true);
      if (ch == last) chunk(nj, yes, wave, last * kKChunk, false);
    } else {
      for (int64_t ch = 0; ch < last; ++ch) chunk(nj, no, int(ch & 1), ch * kKChunk, true);
      chunk(nj, yes, int(last & 1), last * kKChunk, false);
    }
  };
  if (!kSplit) stage(held[0], 0);
  if (kAll) stage(held[kAll], 1);
  __syncthreads();
  const int64_t subs = (L - q0 + 15) / 16;  // with a live query (wavefront-uniform)
  if (kSplit) run(std::integral_constant<int, 1>{});
  else if (kSub > 1 && subs > kWaves + wave) run(std::integral_constant<int, kSub>{});
  else if (subs > wave) run(std::integral_constant<int, 1>{});
  else if (!kAll) run(std::integral_constant<int, 0>{});
  if constexpr (kSplit) {
    // the wavefronts' sums, in their order, brought to the largest of their reference points
    constexpr int kN = 4 * kDt + 3;
    static_assert((kWaves - 1) * kN * 64 * 4 <= sizeof(sk), "the tiles' LDS holds them");
    float* room = reinterpret_cast<float*>(sk);
    __syncthreads();
    if (wave > 0) {
      float* mine = room + (wave - 1) * kN * 64 + lane;
      mine[0] = m[0];
      mine[64] = lreal[0];
      mine[128] = lsum[0][0];
#pragma unroll
      for (int i = 0; i < 4 * kDt; ++i) mine[(3 + i) * 64] = o[0][i / 4][i % 4];
    }
    __syncthreads();
    if (wave > 0) return;
    float top = m[0];
#pragma unroll
    for (int w = 0; w < kWaves - 1; ++w) top = fmaxf(top, room[w * kN * 64 + lane]);
    auto factor = [&](float mw) { return mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw - top) * c_log2); };
    const float own = factor(m[0]);
    lreal[0] *= own;
    lsum[0][0] *= own;
#pragma unroll
    for (int i = 0; i < 4 * kDt; ++i) o[0][i / 4][i % 4] *= own;
#pragma unroll
    for (int w = 0; w < kWaves - 1; ++w) {
      const float* theirs = room + w * kN * 64 + lane;
      const float f = factor(theirs[0]);
      lreal[0] = fmaf(theirs[64], f, lreal[0]);
      lsum[0][0] = fmaf(theirs[128], f, lsum[0][0]);
#pragma unroll
      for (int i = 0; i < 4 * kDt; ++i) o[0][i / 4][i % 4] = fmaf(theirs[(3 + i) * 64], f, o[0][i / 4][i % 4]);
    }
    m[0] = top;
  }
#pragma unroll
  for (int j = 0; j < kSub; ++j) {
    const float lt = lsum[j][0], lr = sum_xor32(sum_xor16(lreal[j]));
    if (qrow[j] < T) {
      const bool live = qrow[j] < L;
      const float inv = live && lt != 0.f ? 1.f / lt : 0.f;
#pragma unroll
      for (int dt = 0; dt < kDt; ++dt) {
        uint2 w = make_uint2(0u, 0u);
        if (live) {
          w.x = FR::pack_unit(o[j][dt][0] * inv, o[j][dt][1] * inv);
          w.y = FR::pack_unit(o[j][dt][2] * inv, o[j][dt][3] * inv);
        }
        *reinterpret_cast<uint2*>(op + qrow[j] * ost + 16 * dt + 4 * g) = w;
      }
      if (g == 0) {
        const float m0 = m[j] == -INFINITY ? 0.f : m[j], log2l = log2f(lr);  // (an empty row's sum is 0)
        // (a row of scores at the lowest finite value has that as its lse, unless a NaN is among them)
        lp[qrow[j]] = !live                                 ? 0.f
                      : fabsf(m0) == kLargest && lr == lr ? m0
                                                          : fmaf(m0, 1.f / root_hd, log2l * 0.6931471805599453f);
        sp[qrow[j]] = live && lr != 0.f ? make_float2(m0, log2l) : make_float2(0.f, INFINITY);
      }
    }
  }
}

template <bool kHalf, int HD, int kSub, bool kSplit>
int32_t launch(const Operand& q, const Operand& k, const Operand& v, const Relative& rel, const int32_t* seq_lens,
               int64_t n_pos, int heads, int64_t t, uint16_t* out, const int64_t* os, float* lse, float2* stats, hipStream_t st) {
  constexpr int kQTile = (kSplit ? 1 : kWaves) * 16 * kSub;
  const int64_t grid = item_grid(n_pos, heads, (t + kQTile - 1) / kQTile);
  if (grid > 2147483647LL) return MANTIS_E_ARG;
  const size_t lds = size_t(rel.nq * rel.nr + 2) * sizeof(float);
  const float root = sqrtf(float(HD));
  relative_attention_kernel<kHalf, HD, kSub, kSplit><<<unsigned(grid), 256, lds, st>>>(
      q, k, v, rel, seq_lens, heads, t, out, os[0], os[1], os[2], lse, stats, 1.4426950408889634f / root, root, n_pos * heads);
  return launched();
}

}  // namespace
}  // namespace mantis

using namespace mantis;

extern "C" int32_t mantis_relative_attention(const void* q, const int64_t* qs, const void* k, const int64_t* ks,
                                             const void* v, const int64_t* vs, int32_t dtype, const float* bias,
                                             int64_t n_buckets, const int32_t* coords, const int32_t* buckets,
                                             int64_t nq, int64_t nr, int64_t n_latents, const int32_t* seq_lens,
                                             int64_t n_pos, int32_t heads, int64_t t, int32_t hd, void* out,
                                             const int64_t* os, float* lse, float* stats, int32_t* err_flag,
                                             void* stream) {
  if (n_pos == 0 || t == 0) return MANTIS_OK;
  if (!q || !k || !v || !out || !lse || !stats || !seq_lens || !qs || !ks || !vs || !os) return MANTIS_E_ARG;
  if ((hd != 16 && hd != 32 && hd != 64) || heads <= 0 || n_pos < 0 || t < 0 || t > 2147483647LL) return MANTIS_E_ARG;
  if (dtype != MANTIS_BF16 && dtype != MANTIS_F16) return MANTIS_E_ARG;
  if (nq > kMaxDisplacements || nr > kMaxDisplacements || n_buckets > kMaxBuckets) return MANTIS_E_ARG;
  for (const int64_t* st : {qs, ks, vs, os}) {
    if (st[3] != 1) return MANTIS_E_ARG;
    if ((st[0] | st[1] | st[2]) % 8) return MANTIS_E_ARG;
  }
  // a position's q, k and v rows are read through buffer descriptors: a row
  // pitch of hd to 8,191 elements and 32-bit byte offsets
  for (const int64_t* st : {qs, ks, vs})
    if (st[2] < hd || st[2] >= 8192 || t * st[2] * 2 > 2147483647LL) return MANTIS_E_ARG;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(stats)) return MANTIS_E_ARG;
  const Relative rel{coords, buckets, bias, int(nq), int(nr), int(n_buckets), n_latents, err_flag};
  if (!good_relative(rel, t)) return MANTIS_E_ARG;
  auto operand = [](const void* ptr, const int64_t* st) {
    return Operand{static_cast<const uint16_t*>(ptr), st[0], st[1], st[2]};
  };
  const Operand Q = operand(q, qs), K = operand(k, ks), V = operand(v, vs);
  uint16_t* o = static_cast<uint16_t*>(out);
  float2* sp = reinterpret_cast<float2*>(stats);
  hipStream_t st = as_stream(stream);
#define MANTIS_FWD(HD_, ...)                                                                                       \
  return dtype == MANTIS_F16                                                                                      \
             ? launch<true, HD_, __VA_ARGS__>(Q, K, V, rel, seq_lens, n_pos, heads, t, o, os, lse, sp, st)        \
             : launch<false, HD_, __VA_ARGS__>(Q, K, V, rel, seq_lens, n_pos, heads, t, o, os, lse, sp, st)
  // Two sub-tiles of 16 queries per wavefront read a key fragment once for both, and 128 queries hold
  // a usual position whole; one leaves the registers for twice the wavefronts: 192 positions of
  // 44-124 rows, 32 dims, 14.5 against 16.7 us, 64 of 150-300 rows 21.6 against 19.7; two lines of
  // 2,049-4,096 rows, 64 dims, 137 against 131, 16 positions of 511-1,021, 16 dims, 72 against 58.
  const bool split = few_groups(n_pos, heads, t, hd);
  if (hd == 16 && split) MANTIS_FWD(16, 1, true);
  if (hd == 16) MANTIS_FWD(16, 1, false);
  if (hd == 32 && split) MANTIS_FWD(32, 1, true);
  if (hd == 32 && t <= 128) MANTIS_FWD(32, 2, false);
  if (hd == 32) MANTIS_FWD(32, 1, false);
  if (split) MANTIS_FWD(64, 1, true);
  MANTIS_FWD(64, 1, false);
#undef MANTIS_FWD
}
