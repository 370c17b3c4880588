// fna2_rope_dev.h — what the rotary kernels share: element types, 16-byte
// chunks, the walk over tokens, sums over a row's lanes.
#pragma once

#include "fna2_kernels.h"

namespace fna2 {

// Products and sums that are never fused into a multiply-add (the
// reference evaluates them as separate elementwise ops).
__device__ __forceinline__ float mul_rn(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}
__device__ __forceinline__ float add_rn(float a, float b) {
#pragma clang fp contract(off)
  return a + b;
}

// Rounding to the element type, as a float.
template <int DT>
__device__ __forceinline__ float rnd(float x) {
  if constexpr (DT == kRopeBF16) {
    return bf16_lo(pack_bf16(x, 0.f));
  } else if constexpr (DT == kRopeF16) {
    return (float)(_Float16)x;
  } else {
    return x;
  }
}

// 16 bytes <-> EPL floats.
template <int DT>
struct Chunk {
  static constexpr int EPL = DT == kRopeF32 ? 4 : 8;
  float v[EPL];
  __device__ __forceinline__ void load(const void* p) {
    const u32x4 w = *(const u32x4*)p;
    if constexpr (DT == kRopeF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u = w[i];  // (a vector element is copied out first)
        v[i] = __builtin_bit_cast(float, u);
      }
    } else if constexpr (DT == kRopeBF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(w[i]), v[2 * i + 1] = bf16_hi(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const _Float16 lo = __builtin_bit_cast(_Float16, (uint16_t)(w[i] & 0xffffu));
        const _Float16 hi = __builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
        v[2 * i] = (float)lo, v[2 * i + 1] = (float)hi;
      }
    }
  }
  __device__ __forceinline__ void store(void* p) const {
    u32x4 w;
    if constexpr (DT == kRopeF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = v[i];
        w[i] = __builtin_bit_cast(uint32_t, f);
      }
    } else if constexpr (DT == kRopeBF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) |
               ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) << 16);
    }
    *(u32x4*)p = w;
  }
};

// 16 bytes as loaded (EPL elements), unpacked on use: rows in flight cost
// half the registers of their fp32 values.
template <int DT>
struct Raw {
  static constexpr int EPL = Chunk<DT>::EPL;
  u32x4 w;
  __device__ __forceinline__ void load(const void* p) { w = *(const u32x4*)p; }
  __device__ __forceinline__ void store(void* p) const { *(u32x4*)p = w; }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (DT == kRopeF32) {
      return __builtin_bit_cast(float, (uint32_t)w[e]);
    } else if constexpr (DT == kRopeBF16) {
      return (e & 1) ? bf16_hi(w[e >> 1]) : bf16_lo(w[e >> 1]);
    } else {
      const uint32_t u = w[e >> 1];
      return (float)__builtin_bit_cast(_Float16, (uint16_t)((e & 1) ? (u >> 16) : (u & 0xffffu)));
    }
  }
};

// Lane layout and the token -> sequence walk shared by the kernels: lane
// owns columns [col, col + EPL) of both halves of row lrow + j * rpw of a
// token; a wave covers P.tpw consecutive tokens from t0.
template <int DT>
struct RopeLanes {
  static constexpr int EPL = Chunk<DT>::EPL;
  int lane, half, lpr, rpw, col, lrow, nrows, t0, b;
  __device__ __forceinline__ RopeLanes(const RopeParams& P, int wave_id) {
    lane = threadIdx.x & 63;
    half = P.D / 2;
    lpr = half / EPL;  // lanes per row (divides 64)
    rpw = 64 / lpr;    // rows per wave pass
    col = (lane % lpr) * EPL;
    lrow = lane / lpr;
    nrows = P.Hq + P.Hk;
    t0 = wave_id * P.tpw;
    // Largest b with cu[b] <= t0 (b = -1: before the first sequence).
    const auto cu = const_space(P.cu);
    const int n = P.nseq;
    int lo = -1, hi = n;  // cu[lo] <= t0 < cu[hi]
    if (t0 < P.T) {
      if (uni(cu[n]) <= t0) lo = n;
      else
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (uni(cu[mid]) <= t0) lo = mid;
          else hi = mid;
        }
    }
    b = lo;
  }
  // Step to token t; returns its position, or -1 outside every sequence.
  __device__ __forceinline__ int position(const RopeParams& P, int t) {
    const auto cu = const_space(P.cu);
    while (b < P.nseq && uni(cu[b + 1]) <= t) ++b;
    return (b >= 0 && b < P.nseq) ? t - uni(cu[b]) : -1;
  }
  // Row pointers (q rows first, then k rows).
  __device__ __forceinline__ const char* in_row(const RopeParams& P, const void* q, const void* k,
                                                int64_t qs, int64_t qh, int64_t ks, int64_t kh,
                                                int t, int r) const {
    constexpr int ES = DT == kRopeF32 ? 4 : 2;
    const bool isq = r < P.Hq;
    const int h = isq ? r : r - P.Hq;
    return (const char*)(isq ? q : k) +
           ((int64_t)t * (isq ? qs : ks) + (int64_t)h * (isq ? qh : kh)) * ES;
  }
};

// Sum over the lpr lanes of a row (lanes lrow * lpr .. + lpr - 1); every
// lane of the wave takes part.
__device__ __forceinline__ float row_sum(float v, int lpr) {
  for (int m = 1; m < lpr; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

}  // namespace fna2
