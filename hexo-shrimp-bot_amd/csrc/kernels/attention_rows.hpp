// Row chunks and products shared by the ragged attentions' passes: a workgroup
// of four wavefronts, 16 rows of its own side each, meets the other side's rows
// in 64-row chunks through LDS.
#pragma once

#include "common.hpp"
#include "mfma.hpp"

namespace mantis {
namespace {

constexpr int kTile = 64;                // rows of a workgroup, and of a chunk
constexpr int kTPitch = kTile + 8;       // 16-bit elements per transposed row
constexpr float kLog2e = 1.4426950408889634f;

struct Rows {  // one (P, A, T, HD) operand: base and element strides
  const uint16_t* p;
  int64_t sp, sa, st;
  __device__ const uint16_t* at(int64_t pos, int64_t a) const { return p + pos * sp + a * sa; }
};
struct RowsOut {
  uint16_t* p;
  int64_t sp, sa, st;
  __device__ uint16_t* row(int64_t pos, int64_t a, int64_t t) const { return p + pos * sp + a * sa + t * st; }
};

template <bool kHalf>
__device__ __forceinline__ float widen(uint32_t bits) {
  if constexpr (kHalf) return float(__builtin_bit_cast(_Float16, uint16_t(bits)));
  else return __uint_as_float(bits << 16);
}

template <bool kHalf, int HD>
struct Geom {
  static constexpr int kPitch = HD + 8;                 // 16-bit elements per staged row
  static constexpr int kKs = HD < 32 ? 1 : HD / 32;     // K steps of a product over dims
  static constexpr int kDt = HD / 16;                   // 16-dim output tiles
  static constexpr int kPieces = kTile * HD / 8;        // 16-byte pieces of a chunk
  static constexpr int kPer = kPieces < 256 ? 1 : kPieces / 256;
  // the dims of this lane in K step ks (HD = 16: lanes g >= 2 hold zeros)
  static __device__ __forceinline__ int kdim(int ks, int g) { return HD < 32 ? 8 * (g & 1) : 32 * ks + 8 * g; }
};

// A 64-row chunk of one operand: fetched to registers (zeros at or past L),
// staged as rows, as transposed rows, or both.
template <bool kHalf, int HD>
struct Chunk {
  using G = Geom<kHalf, HD>;
  uint4 reg[G::kPer];
  __device__ __forceinline__ void fetch(const uint16_t* base, int64_t st, int64_t first, int64_t L) {
#pragma unroll
    for (int r = 0; r < G::kPer; ++r) {
      const int i = int(threadIdx.x) + 256 * r;
      const int64_t row = first + i / (HD / 8);
      reg[r] = make_uint4(0u, 0u, 0u, 0u);
      if (i < G::kPieces && row < L) reg[r] = *reinterpret_cast<const uint4*>(base + row * st + 8 * (i % (HD / 8)));
    }
  }
  __device__ __forceinline__ void stage_rows(uint16_t* s) const {
#pragma unroll
    for (int r = 0; r < G::kPer; ++r) {
      const int i = int(threadIdx.x) + 256 * r;
      if (i < G::kPieces)
        *reinterpret_cast<uint4*>(s + (i / (HD / 8)) * G::kPitch + 8 * (i % (HD / 8))) = reg[r];
    }
  }
  __device__ __forceinline__ void stage_transposed(uint16_t* s) const {
#pragma unroll
    for (int r = 0; r < G::kPer; ++r) {
      const int i = int(threadIdx.x) + 256 * r;
      if (i >= G::kPieces) continue;
      uint16_t* col = s + 8 * (i % (HD / 8)) * kTPitch + i / (HD / 8);
      const uint32_t w[4] = {reg[r].x, reg[r].y, reg[r].z, reg[r].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        col[2 * e * kTPitch] = uint16_t(w[e]);
        col[(2 * e + 1) * kTPitch] = uint16_t(w[e] >> 16);
      }
    }
  }
};

// this lane's row of one side as B fragments, zeros when it is not live
template <bool kHalf, int HD>
__device__ __forceinline__ void load_frags(const uint16_t* row, bool live, int g,
                                           uint4 (&u)[Geom<kHalf, HD>::kKs]) {
  using G = Geom<kHalf, HD>;
#pragma unroll
  for (int ks = 0; ks < G::kKs; ++ks) {
    u[ks] = make_uint4(0u, 0u, 0u, 0u);
    if (live && (HD >= 32 || g < 2)) u[ks] = *reinterpret_cast<const uint4*>(row + G::kdim(ks, g));
  }
}

// d += 4 tiles of 16 staged rows times this lane's row, those with a row below n (HD = 16: the upper K slots
// are zeros on both sides, so an infinite row meets none of them)
template <bool kHalf, int HD>
__device__ __forceinline__ void products_onto(const uint16_t* s, int n, int l16, int g,
                                              const uint4 (&b)[Geom<kHalf, HD>::kKs], f32x4_t (&d)[4]) {
  using G = Geom<kHalf, HD>;
  using FR = Frag<kHalf>;
#pragma unroll
  for (int tt = 0; tt < 4; ++tt) {
    if (16 * tt >= n) {  // uniform
      around_products();
      continue;
    }
#pragma unroll
    for (int ks = 0; ks < G::kKs; ++ks) {
      uint4 a = *reinterpret_cast<const uint4*>(s + (16 * tt + l16) * G::kPitch + G::kdim(ks, g));
      if (HD < 32 && g >= 2) a = make_uint4(0u, 0u, 0u, 0u);
      d[tt] = mfma16x16x32(FR::cast(a), FR::cast(b[ks]), d[tt]);
    }
  }
}
template <bool kHalf, int HD>
__device__ __forceinline__ void products(const uint16_t* s, int n, int l16, int g,
                                         const uint4 (&b)[Geom<kHalf, HD>::kKs], f32x4_t (&d)[4]) {
#pragma unroll
  for (int tt = 0; tt < 4; ++tt) d[tt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  products_onto<kHalf, HD>(s, n, l16, g, b, d);
}

// acc (HD dims x this lane's row) += transposed rows . x over a chunk's tiles with
// a row below n, x the 16 fp32 values of this lane (rows 16 tt + 4 g + t), on the fp32 MFMA
// (16 x 16 x 4: lane group g holds K slot g of both operands)
template <bool kHalf, int HD>
__device__ __forceinline__ void accumulate(const uint16_t* st, int n, int l16, int g, const float (&x)[4][4],
                                           f32x4_t (&acc)[Geom<kHalf, HD>::kDt]) {
#pragma unroll
  for (int tt = 0; tt < 4; ++tt) {
    if (16 * tt >= n) {  // uniform
      around_fp32_products();
      continue;
    }
    uint2 a[Geom<kHalf, HD>::kDt];
#pragma unroll
    for (int dt = 0; dt < Geom<kHalf, HD>::kDt; ++dt)
      a[dt] = *reinterpret_cast<const uint2*>(st + (16 * dt + l16) * kTPitch + 16 * tt + 4 * g);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int dt = 0; dt < Geom<kHalf, HD>::kDt; ++dt) {
        const uint32_t w = t < 2 ? a[dt].x : a[dt].y;
        const float v = widen<kHalf>(t % 2 ? w >> 16 : w & 0xffffu);
        acc[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, x[tt][t], acc[dt], 0, 0, 0);
      }
  }
}

// a lane's row of HD gradients (dims 16 dt + 4 g + t), zeros when not live; fp16
// saturates, or with kOverflow overflows to an infinity and keeps NaN
template <bool kHalf, int HD, bool kOverflow = false>
__device__ __forceinline__ void store_row(uint16_t* row, int g, const f32x4_t (&acc)[Geom<kHalf, HD>::kDt],
                                          float scale, bool live) {
#pragma unroll
  for (int dt = 0; dt < Geom<kHalf, HD>::kDt; ++dt) {
    uint2 w = make_uint2(0u, 0u);
    if (live) {
      auto pack = [](float lo, float hi) {
        return kOverflow ? Frag<kHalf>::pack_unit(lo, hi) : Frag<kHalf>::pack(lo, hi);
      };
      w.x = pack(acc[dt][0] * scale, acc[dt][1] * scale);
      w.y = pack(acc[dt][2] * scale, acc[dt][3] * scale);
    }
    *reinterpret_cast<uint2*>(row + 16 * dt + 4 * g) = w;
  }
}

// the A fragment (16 dims x 32 rows) of the transposed rows 32 h .. of a tile
// at pitch HD + 8, dims 16 dt .., its K slots the rows 4 g + t and 16 + 4 g + t: the transposing
// read gives lane i of 16 the i-th of the 16 dims of four rows whose 8-byte
// pieces the 16 lanes name
typedef short lds_s16x4_t __attribute__((ext_vector_type(4)));
template <int HD>
__device__ __forceinline__ uint4 transposed_frag(const uint16_t* s, int h, int dt, int l16, int g) {
  using Shared = __attribute__((address_space(3))) lds_s16x4_t;
  const uint16_t* at = s + (32 * h + 4 * g + l16 / 4) * (HD + 8) + 16 * dt + 4 * (l16 % 4);
  const lds_s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Shared*)at);
  const lds_s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Shared*)(at + 16 * (HD + 8)));
  const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
  return make_uint4(a.x, a.y, b.x, b.y);
}

}  // namespace
}  // namespace mantis
