// fna2_paged_dev.h — what the packed and the tile kernel of the paged
// attention share in their key steps.
#pragma once

#include "fna2_paged.h"
#include "fna2_tile.h"

namespace fna2 {

// The page ids of a part of a sequence, 64 at a time in a register's lanes: a
// step reads its own with no memory access, so none waits in the steps' way
// (a scalar load a step ahead did: its counter is the LDS reads' too).
struct PageIds {
  const int* row;  // of the block table
  int ids, base, last;
  // Pages base .. base + 63; `last` is the last one that holds rows (-1: none).
  __device__ __forceinline__ void load(int lane, int first) {
    base = first;
    ids = last >= 0 ? row[min(first + lane, last)] : -1;
  }
  __device__ __forceinline__ int at(int lane, int page) {
    if (page - base >= 64) load(lane, page);
    return __builtin_amdgcn_readlane(ids, page - base);
  }
};

// e^(x) in powers of two for the weight of an accumulator, never zero: an
// infinity in it stays one (a sum's start, x = -inf, holds zeros).
__device__ __forceinline__ float weight2(float x) {
  return fmaxf(__builtin_amdgcn_exp2f(x), 1.17549435e-38f);
}

// P in two parts (as the decode kernel): the first cut to the element
// type, the second what that cut off, so that the result does not
// depend on where a tile is split.  No part of a visible key is
// zero (an infinite V stays infinite; in fp16 from a p of 2^-24 on, below which the first is),
// both of a hidden key's are.  The second
// part's lowest bit, which sees to that, is 2^-24 in fp16 (p's scale: the
// largest is 1), which is then each key's error at most; in bf16 nothing.
template <bool F16>
__device__ __forceinline__ void split_p(float p0, float p1, u32x4& first, u32x4& second, int i) {
  if constexpr (F16) {
    first[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p0, p1));
    second[i] = pack_e<true>(p0 - elt_lo<true>(first[i]), p1 - elt_hi<true>(first[i]));
  } else {
    const uint32_t u0 = __builtin_bit_cast(uint32_t, p0);
    const uint32_t u1 = __builtin_bit_cast(uint32_t, p1);
    first[i] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);  // their upper halves
    second[i] = pack_bf16(p0 - __builtin_bit_cast(float, u0 & 0xffff0000u),
                          p1 - __builtin_bit_cast(float, u1 & 0xffff0000u));
  }
  second[i] |= (p0 > 0.f ? 1u : 0u) | (p1 > 0.f ? 0x10000u : 0u);
}

// Hidden V rows.  In a step whose rows some columns see and others do not, a
// hidden row's probability is 0, and 0 times an infinity or a NaN in it (a later
// token's V) is NaN.  So such a step looks through its V tile first
// (tile_odd); where it finds one, those values are added to the accumulators
// of the columns that see their row (add_odd), and then zeroed in the tile
// (tile_clean).  (A second product with cleaned operands instead: 240
// registers spilled.)

// Bits of an element-type word's two halves that are infinite or NaN.
template <bool F16>
__device__ __forceinline__ uint32_t odd_bits(uint32_t w) {
  constexpr uint32_t E = F16 ? 0x7c00u : 0x7f80u;
  return ((w & E) == E ? 0xffffu : 0u) | ((w & (E << 16)) == (E << 16) ? 0xffff0000u : 0u);
}

// Whether the wave finds an infinity or a NaN in KB kilobytes of a tile, and
// the zeroing of those.
template <int KB, bool F16>
__device__ __forceinline__ bool tile_odd(const uint8_t* tile, int lane) {
  // (the largest exponents, and one comparison: a comparison a word would take
  // a pair of scalar registers each)
  constexpr uint32_t E = F16 ? 0x7c00u : 0x7f80u;
  uint32_t lo = 0, hi = 0;
#pragma unroll
  for (int i = 0; i < KB; ++i) {
    const u32x4 w = *(const u32x4*)(tile + 1024 * i + 16 * lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      lo = max(lo, w[j] & E);
      hi = max(hi, w[j] & (E << 16));
    }
  }
  return __builtin_amdgcn_ballot_w64(lo == E || hi == (E << 16)) != 0;
}
template <int KB, bool F16>
__device__ __forceinline__ void tile_clean(uint8_t* tile, int lane) {
#pragma unroll 1
  for (int i = 0; i < KB; ++i) {
    u32x4* at = (u32x4*)(tile + 1024 * i + 16 * lane);
    u32x4 w = *at;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] &= ~odd_bits<F16>(w[j]);
    *at = w;
  }
}

// Adds the odd values of a V tile of BN rows, the first of them row `kbase`
// of the cache, to the accumulators O^T of a column that sees rows up to `lim`
// (a positive probability times an infinity or a NaN is that).
template <int D, int BN, bool F16>
__device__ __forceinline__ void add_odd(const uint8_t* tile, int kbase, int lim, int hl,
                                        f32x16 (&oacc)[D / 32]) {
#pragma unroll 1
  for (int r = 0; r < BN; ++r) {
    const bool see = kbase + r <= lim;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const u32x2 w = *(const u32x2*)(tile + tile_off<BN>(r, 4 * d + g) + 8 * hl);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t o = see ? w[i] & odd_bits<F16>(w[i]) : 0u;
          oacc[d][4 * g + 2 * i] += elt_lo<F16>(o);
          oacc[d][4 * g + 2 * i + 1] += elt_hi<F16>(o);
        }
        __builtin_amdgcn_sched_barrier(0);  // (few registers, not speed)
      }
  }
}

}  // namespace fna2
