// Backward of the relative attention on 16-bit MFMA for gfx950.  With the
// forward's statistics (m, log2 l) per row, s_ij the raw scores with their bias
// (relative_bias.hpp) and c = log2(e) / sqrt(hd):
//   p_ij = exp2(c (s_ij - m_i) - log2 l_i),  dp_ij = go_i . v_j,
//   delta_i = sum_j p_ij dp_ij,  ds_ij = p_ij (dp_ij - delta_i),
//   dq_i = sum_j ds_ij k_j / sqrt(hd),  dk_j = sum_i ds_ij q_i / sqrt(hd),
//   dv_j = sum_i p_ij go_i,  dbias[a, b] = sum of ds_ij over the pairs of bucket b.
//
// Two passes, each a workgroup per (position, head, 64 rows), 16 rows per
// wavefront, the other side's rows in 64-row chunks through LDS:
//   query-major  S^T = K Q^T and dP^T = V dO^T, then dQ^T += K^T dS^T and the buckets' sums
//   key-major    S = Q K^T and dP = dO V^T, then dV^T += dO^T P, dK^T += Q^T dS
// The query pass goes over the keys twice: delta first, from the fp32 products
// (the 16-bit output's rounding would stay in every ds of its row, and in the
// bias gradient's long sums), then ds; the rows of one chunk stay in
// registers and LDS in between.
//
// The bias gradient: every lane adds its ds to its own column of the
// workgroup's LDS table (a row of 64 lanes per bucket and wavefront: no two
// lanes meet, no bank is asked twice), or, where that table does not fit, the
// four lane groups in turn to 16 columns.  The columns join in a fixed order into the
// workgroup's partial sums, those of a head in a second launch.  Every sum is
// fp32 in a fixed order: two calls agree bitwise.
//
// The probabilities and ds are fp32 and enter their products, with the rows
// widened, as fp32 MFMA operands.
#include "attention_rows.hpp"
#include "relative_bias.hpp"

namespace mantis {
namespace {

constexpr int kBwdWaves = 4;
constexpr size_t kLdsBytes = 160 * 1024;

// fp32 add to LDS, no value back
__device__ __forceinline__ void lds_add(float* p, float x) {
  __hip_atomic_fetch_add(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

// Dynamic LDS: the bias table, then (query pass) the bucket table and the columns.
__host__ __device__ constexpr size_t table_bytes(int n_disp) { return (size_t(n_disp + 2) * 4 + 15) / 16 * 16; }
__host__ __device__ constexpr size_t bucket_bytes(int n_disp) { return (size_t(n_disp + 2) * 2 + 15) / 16 * 16; }
__host__ __device__ constexpr size_t column_bytes(int n_buckets, int columns) {
  return size_t(kBwdWaves) * (n_buckets + 1) * columns * 4;  // (a row for the pairs of no bucket)
}

template <bool kHalf, int HD, int kColumns>
__global__ void __launch_bounds__(256)
relative_bwd_q_kernel(Rows q, Rows k, Rows v, Rows go, Relative rel, const int32_t* __restrict__ seq_lens, int heads,
                      int64_t T, const float2* __restrict__ stats, float scale, float root_hd,
                      float* __restrict__ delta, RowsOut dq, float* __restrict__ partial) {
  using G = Geom<kHalf, HD>;
  __shared__ __attribute__((aligned(16))) uint16_t sk[kTile * G::kPitch], sv[kTile * G::kPitch];
  __shared__ __attribute__((aligned(16))) uint16_t skt[HD * kTPitch];
  __shared__ __attribute__((aligned(16))) uint32_t sc[kTile];
  extern __shared__ __attribute__((aligned(16))) char dynamic[];
  const int n_disp = rel.nq * rel.nr;
  float* table = reinterpret_cast<float*>(dynamic);
  uint16_t* bucket = reinterpret_cast<uint16_t*>(dynamic + table_bytes(n_disp));
  float* columns = reinterpret_cast<float*>(dynamic + table_bytes(n_disp) + bucket_bytes(n_disp));
  const int64_t n_tiles = (T + kTile - 1) / kTile;
  const int64_t pa = blockIdx.x / n_tiles, tile = blockIdx.x % n_tiles;
  const int64_t pos = pa / heads, a = pa % heads;
  int64_t L = seq_lens[pos];
  L = L < 0 ? 0 : (L > T ? T : L);
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, l16 = lane % 16, g = lane / 16;
  const int64_t first = tile * kTile + 16 * wave, i = first + l16;
  const bool live = i < L;
  const int n_rows = rel.n_buckets + 1;
  // partial sums: (head, position, tile, bucket)
  float* part = partial + ((a * (gridDim.x / n_tiles / heads) + pos) * n_tiles + tile) * rel.n_buckets;
  if (tile * kTile >= L) {  // no live row
    if (i < T) {
      const f32x4_t zero[G::kDt] = {};
      store_row<kHalf, HD, true>(dq.row(pos, a, i), g, zero, 0.f, false);
      if (g == 0) delta[pa * T + i] = 0.f;
    }
    for (int b = threadIdx.x; b < rel.n_buckets; b += 256) part[b] = 0.f;
    return;
  }
  uint4 qf[G::kKs], gf[G::kKs];
  load_frags<kHalf, HD>(q.at(pos, a) + i * q.st, live, g, qf);
  load_frags<kHalf, HD>(go.at(pos, a) + i * go.st, live, g, gf);
  const float2 st = live ? stats[pa * T + i] : make_float2(0.f, INFINITY);
  const Side<true> side(rel, coords_of(rel, pos, T, i, L), i < rel.n_latents);
  stage_bias(rel, a, root_hd, table);
  for (int d = threadIdx.x; d < n_disp + 2; d += 256) bucket[d] = uint16_t(bucket_of(rel, d));
  for (int c = threadIdx.x; c < kBwdWaves * n_rows * kColumns; c += 256) columns[c] = 0.f;
  float* column = columns + wave * n_rows * kColumns + lane % kColumns;

  f32x4_t acc[G::kDt];
#pragma unroll
  for (int dt = 0; dt < G::kDt; ++dt) acc[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const uint16_t* kp = k.at(pos, a);
  const uint16_t* vp = v.at(pos, a);
  Chunk<kHalf, HD> ck, cv;
  uint32_t cc = 0u;
  auto fetch = [&](int64_t kb) {
    ck.fetch(kp, k.st, kb, L);
    cv.fetch(vp, v.st, kb, L);
    if (threadIdx.x < kTile) cc = coords_of(rel, pos, T, kb + threadIdx.x, L);
  };
  auto stage = [&](bool transposed) {
    __syncthreads();  // the last chunk's readers are done
    ck.stage_rows(sk);
    if (transposed) ck.stage_transposed(skt);
    cv.stage_rows(sv);
    if (threadIdx.x < kTile) sc[threadIdx.x] = cc;
    __syncthreads();
  };
  const float c_log2 = scale * kLog2e;
  int at[4][4];  // the pairs' table entries, as byte offsets
  // p and dp of the staged chunk's keys for this lane's query, zeros at or past L
  auto pairs = [&](int64_t kb, int n, float (&p)[4][4], f32x4_t (&dp)[4]) {
    const int lim = n - 4 * g;  // keys 16 tt + t below it are live
    f32x4_t s[4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      const uint4 kc = *reinterpret_cast<const uint4*>(&sc[16 * tt + 4 * g]);
      const uint32_t kcs[4] = {kc.x, kc.y, kc.z, kc.w};
#pragma unroll
      for (int t = 0; t < 4; ++t) at[tt][t] = side.at(kcs[t]);
    }
    if (kb < rel.n_latents) {  // uniform
      const int64_t lat = rel.n_latents - kb - 4 * g;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int t = 0; t < 4; ++t) at[tt][t] = 16 * tt + t < lat ? side.latent_other : at[tt][t];
    }
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int t = 0; t < 4; ++t) s[tt][t] = entry(table, at[tt][t]);
    products_onto<kHalf, HD>(sk, n, l16, g, qf, s);
    products<kHalf, HD>(sv, n, l16, g, gf, dp);
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const bool in = 16 * tt + t < lim;
        p[tt][t] = in ? __builtin_amdgcn_exp2f(fmaf(s[tt][t] - st.x, c_log2, -st.y)) : 0.f;
        dp[tt][t] = in ? dp[tt][t] : 0.f;
      }
  };
  float dl = 0.f;
  auto sum_delta = [&](const float (&p)[4][4], const f32x4_t (&dp)[4]) {
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int t = 0; t < 4; ++t) dl = fmaf(p[tt][t], dp[tt][t], dl);
  };
  auto spread = [&](int n, const float (&p)[4][4], const f32x4_t (&dp)[4]) {
    const int lim = n - 4 * g;
    float ds[4][4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        ds[tt][t] = p[tt][t] * (dp[tt][t] - dl);
        const bool in = live && 16 * tt + t < lim;
        float* to = column + (in ? int(bucket[at[tt][t] / 4]) : rel.n_buckets) * kColumns;
        if constexpr (kColumns == 64) {
          lds_add(to, ds[tt][t]);
        } else {
#pragma unroll
          for (int turn = 0; turn < 4; ++turn)
            if (g == turn) lds_add(to, ds[tt][t]);
        }
      }
    accumulate<kHalf, HD>(skt, n, l16, g, ds, acc);
  };
  float p[4][4];
  f32x4_t dp[4];
  fetch(0);
  if (L <= kTile) {
    stage(true);
    if (first < L) {  // wavefront-uniform: a live row here
      pairs(0, int(L), p, dp);
      sum_delta(p, dp);
      dl = sum_xor32(sum_xor16(dl));
      spread(int(L), p, dp);
    }
  } else {
    for (int64_t kb = 0; kb < L; kb += kTile) {
      stage(false);
      fetch(kb + kTile < L ? kb + kTile : 0);
      if (first >= L) continue;
      pairs(kb, int(L - kb < kTile ? L - kb : kTile), p, dp);
      sum_delta(p, dp);
    }
    dl = sum_xor32(sum_xor16(dl));
    for (int64_t kb = 0; kb < L; kb += kTile) {
      stage(true);
      if (kb + kTile < L) fetch(kb + kTile);
      if (first >= L) continue;
      const int n = int(L - kb < kTile ? L - kb : kTile);
      pairs(kb, n, p, dp);
      spread(n, p, dp);
    }
  }
  if (i < T) {
    store_row<kHalf, HD, true>(dq.row(pos, a, i), g, acc, scale, live);
    if (g == 0) delta[pa * T + i] = live ? dl : 0.f;
  }
  __syncthreads();
  // the columns of a bucket, from the bucket's own on so that the threads meet other banks
  for (int b = threadIdx.x; b < rel.n_buckets; b += 256) {
    float sum = 0.f;
    for (int w = 0; w < kBwdWaves; ++w)
      for (int c = 0; c < kColumns; ++c) sum += columns[(w * n_rows + b) * kColumns + (c + b) % kColumns];
    part[b] = sum;
  }
}

template <bool kHalf, int HD>
__global__ void __launch_bounds__(256)
relative_bwd_kv_kernel(Rows q, Rows k, Rows v, Rows go, Relative rel, const int32_t* __restrict__ seq_lens, int heads,
                       int64_t T, const float2* __restrict__ stats, float scale, float root_hd,
                       const float* __restrict__ delta, RowsOut dk, RowsOut dv) {
  using G = Geom<kHalf, HD>;
  __shared__ __attribute__((aligned(16))) uint16_t sq[kTile * G::kPitch], sg[kTile * G::kPitch];
  __shared__ __attribute__((aligned(16))) uint16_t sqt[HD * kTPitch], sgt[HD * kTPitch];
  __shared__ __attribute__((aligned(16))) float sm[kTile], sl[kTile], sd[kTile];
  __shared__ __attribute__((aligned(16))) uint32_t sc[kTile];
  extern __shared__ __attribute__((aligned(16))) char dynamic[];
  float* table = reinterpret_cast<float*>(dynamic);
  const int64_t n_tiles = (T + kTile - 1) / kTile;
  const int64_t pa = blockIdx.x / n_tiles, tile = blockIdx.x % n_tiles;
  const int64_t pos = pa / heads, a = pa % heads;
  int64_t L = seq_lens[pos];
  L = L < 0 ? 0 : (L > T ? T : L);
  const int lane = threadIdx.x % 64, l16 = lane % 16, g = lane / 16;
  const int64_t first = tile * kTile + 16 * (threadIdx.x / 64), j = first + l16;
  const bool live = j < L;
  f32x4_t ak[G::kDt], av[G::kDt];
#pragma unroll
  for (int dt = 0; dt < G::kDt; ++dt) ak[dt] = av[dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if (tile * kTile < L) {  // workgroup-uniform
    uint4 kf[G::kKs], vf[G::kKs];
    load_frags<kHalf, HD>(k.at(pos, a) + j * k.st, live, g, kf);
    load_frags<kHalf, HD>(v.at(pos, a) + j * v.st, live, g, vf);
    const bool latent = j < rel.n_latents;
    const Side<false> side(rel, coords_of(rel, pos, T, j, L), latent);
    stage_bias(rel, a, root_hd, table);
    const uint16_t* qp = q.at(pos, a);
    const uint16_t* gp = go.at(pos, a);
    const float c_log2 = scale * kLog2e;
    Chunk<kHalf, HD> cq, cg;
    float rm = 0.f, rl = INFINITY, rd = 0.f;
    uint32_t cc = 0u;
    auto fetch = [&](int64_t qb) {
      cq.fetch(qp, q.st, qb, L);
      cg.fetch(gp, go.st, qb, L);
      if (threadIdx.x < kTile) {
        const int64_t i = qb + threadIdx.x;
        const bool in = i < L;
        const float2 st = in ? stats[pa * T + i] : make_float2(0.f, INFINITY);
        rm = st.x, rl = st.y;
        rd = in ? delta[pa * T + i] : 0.f;
        cc = coords_of(rel, pos, T, i, L);
      }
    };
    fetch(0);
    for (int64_t qb = 0; qb < L; qb += kTile) {
      __syncthreads();
      cq.stage_rows(sq);
      cq.stage_transposed(sqt);
      cg.stage_rows(sg);
      cg.stage_transposed(sgt);
      if (threadIdx.x < kTile) {
        sm[threadIdx.x] = rm;
        sl[threadIdx.x] = rl;
        sd[threadIdx.x] = rd;
        sc[threadIdx.x] = cc;
      }
      __syncthreads();
      if (qb + kTile < L) fetch(qb + kTile);
      if (first >= L) continue;  // wavefront-uniform
      const int n = int(L - qb < kTile ? L - qb : kTile);
      f32x4_t s[4], dp[4];
      int at[4][4];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const uint4 qc = *reinterpret_cast<const uint4*>(&sc[16 * tt + 4 * g]);
        const uint32_t qcs[4] = {qc.x, qc.y, qc.z, qc.w};
#pragma unroll
        for (int t = 0; t < 4; ++t) at[tt][t] = side.at(qcs[t]);
      }
      if (qb < rel.n_latents) {  // uniform (a latent key's pairs keep its own entry)
        const int64_t lat = rel.n_latents - qb - 4 * g;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int t = 0; t < 4; ++t) at[tt][t] = 16 * tt + t < lat ? side.latent_other : at[tt][t];
      }
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int t = 0; t < 4; ++t) s[tt][t] = entry(table, at[tt][t]);
      products_onto<kHalf, HD>(sq, n, l16, g, kf, s);
      products<kHalf, HD>(sg, n, l16, g, vf, dp);
      const int lim = n - 4 * g;  // queries 16 tt + t below it are live
      float p[4][4], ds[4][4];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const float4 m4 = *reinterpret_cast<const float4*>(&sm[16 * tt + 4 * g]);
        const float4 l4 = *reinterpret_cast<const float4*>(&sl[16 * tt + 4 * g]);
        const float4 d4 = *reinterpret_cast<const float4*>(&sd[16 * tt + 4 * g]);
        const float mv[4] = {m4.x, m4.y, m4.z, m4.w}, lv[4] = {l4.x, l4.y, l4.z, l4.w},
                    dv4[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float e = __builtin_amdgcn_exp2f(fmaf(s[tt][t] - mv[t], c_log2, -lv[t]));
          p[tt][t] = 16 * tt + t < lim ? e : 0.f;
          ds[tt][t] = 16 * tt + t < lim ? e * (dp[tt][t] - dv4[t]) : 0.f;
        }
      }
      accumulate<kHalf, HD>(sgt, n, l16, g, p, av);
      accumulate<kHalf, HD>(sqt, n, l16, g, ds, ak);
    }
  }
  if (j < T) {
    store_row<kHalf, HD, true>(dk.row(pos, a, j), g, ak, scale, live);
    store_row<kHalf, HD, true>(dv.row(pos, a, j), g, av, 1.f, live);
  }
}

// dbias[a, b]: the head's partial sums, each thread a fixed stride of them,
// joined in a fixed order.  One workgroup per (head, bucket).
__global__ void __launch_bounds__(256)
relative_bias_sum_kernel(const float* __restrict__ partial, int64_t n_parts, int n_buckets, float* __restrict__ dbias) {
  __shared__ float sums[256];
  const int64_t a = blockIdx.x / n_buckets, b = blockIdx.x % n_buckets;
  float sum = 0.f;
  for (int64_t i = threadIdx.x; i < n_parts; i += 256) sum += partial[(a * n_parts + i) * n_buckets + b];
  sums[threadIdx.x] = sum;
  for (int o = 128; o > 0; o >>= 1) {
    __syncthreads();
    if (int(threadIdx.x) < o) sums[threadIdx.x] += sums[threadIdx.x + o];
  }
  if (threadIdx.x == 0) dbias[blockIdx.x] = sums[0];
}

template <bool kHalf, int HD>
constexpr size_t static_lds() {
  return size_t(2 * kTile * Geom<kHalf, HD>::kPitch + HD * kTPitch) * 2 + kTile * 4;
}

// the dynamic LDS that a kernel may ask for, set once per kernel and device
template <auto kKernel>
bool allow_lds(size_t bytes) {
  static bool done[64] = {};
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
  const int64_t n_tiles = (t + kTile - 1) / kTile, grid = n_pos * heads * n_tiles;
  if (grid > 2147483647LL) return MANTIS_E_ARG;
  const float root = sqrtf(float(HD)), scale = 1.f / root;
  const int n_disp = rel.nq * rel.nr;
  const size_t tables = table_bytes(n_disp) + bucket_bytes(n_disp);
  const size_t wide = tables + column_bytes(rel.n_buckets, 64), narrow = tables + column_bytes(rel.n_buckets, 16);
  const bool fits = static_lds<kHalf, HD>() + wide <= kLdsBytes;
  if (!fits && static_lds<kHalf, HD>() + narrow > kLdsBytes) return MANTIS_E_ARG;
  auto first = fits ? relative_bwd_q_kernel<kHalf, HD, 64> : relative_bwd_q_kernel<kHalf, HD, 16>;
  constexpr size_t most = kLdsBytes - static_lds<kHalf, HD>();
  if (!(fits ? allow_lds<relative_bwd_q_kernel<kHalf, HD, 64>>(most)
             : allow_lds<relative_bwd_q_kernel<kHalf, HD, 16>>(most)))
    return MANTIS_E_LAUNCH;
  first<<<unsigned(grid), 256, fits ? wide : narrow, st>>>(q, k, v, go, rel, seq_lens, heads, t, stats, scale, root,
                                                           delta, dq, partial);
  relative_bwd_kv_kernel<kHalf, HD><<<unsigned(grid), 256, table_bytes(n_disp), st>>>(
      q, k, v, go, rel, seq_lens, heads, t, stats, scale, root, delta, dk, dv);
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
  return 4 * (n_pos * heads * t + n_pos * heads * ((t + kTile - 1) / kTile) * n_buckets);
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
