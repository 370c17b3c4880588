// fna2_paged_tile.hip — attention of long chunks of new tokens over a paged cache.
//
// The operator of fna2_paged_attn.hip for chunks whose (token, head) pairs
// fill more than one column tile.  A workgroup is 4 waves that share the K
// and V tiles of one KV head; each wave has 32 tokens of one query head, hw of
// the KV head's in all: (tokens, heads) = (128, 1), (64, 2) or (32, 4).  With
// grouped heads a tile of 4 heads reads K and V once for them all however short the chunk.
// The waves compute as the forward kernel's do: S^T = Ka Qa^T with the rank
// chain first, the lazily rescaled online softmax by column, O^T += V^T P^T with
// P in the element type.
//
// Work and pages as in fna2_paged_attn.hip: the tiles' key steps laid end to
// end, an equal run for each resident workgroup, parts of cut tiles joined by
// a second kernel.  Workgroups whose runs are neighbours share an XCD's L2.  A
// wave DMAs the same 16 rows of every K, V and R_k tile, so it follows one
// page.
//
// Bound by the matrix cores and, between their products, by the exponentials and the
// rounding of P: 1024 tokens over 16,384 rows, 32 heads over 8 KV heads of 128, R = 64,
// 346 to 362 us with the merge of the parts, up to 0.96 10^15 operations a second of the
// 1.23 10^15 of a large matrix product (matrix cores 52% of the cycles, at the 1.85 GHz
// that the power leaves; spread evenly at 2.4 GHz products 132 us, other vector
// instructions 125).  A step of 256 tokens beside 32 decoding sequences over 4096 rows
// is bound by reading K, V and R_k (5.7 TB/s): 123 us and 12 us.  At d = 64, R = 16
// (2 chunks of 509 tokens over 7001 rows, 16 heads) by neither, 48 us and 9: products
// 10 us, vector instructions 19, waves waiting 37% of their time on two workgroups a CU,
// and the ranks padded to 32.  P is rounded once, off by
// half a step (bf16 2^-8) of each p at most, on top of the output's own rounding (1.4 times
// the error of an output alone); in two parts the products with V would double.
#include <algorithm>

#include "fna2_paged_tile_dev.h"

namespace fna2 {

namespace {

// Joins the parts of a tile that runs cut: workgroup (i, y) takes 32 features
// of the tile that run i's end cuts, four parts at a time.  A wave takes the tokens
// of one wave of the tile; where a tile has many parts (by_part) the
// workgroup does, its waves every fourth group of parts each, joined in LDS.  The
// order of the sums goes by the parts alone.
template <int D, bool F16>
__global__ __launch_bounds__(256) void paged_tile_merge_kernel(const PagedParams) {
  KArg P = kargs();
  __shared__ f32x4_t part[4][4][64];
  __shared__ float stat[4][2][32];
  const int lane = threadIdx.x & 63, own = uni(threadIdx.x >> 6);
  const bool by_part = P->merge_by_part != 0;
  const int d = blockIdx.y % (D / 32), wv = by_part ? blockIdx.y / (D / 32) : own;
  const int l32 = lane & 31, hl = lane >> 5;
  const int i0 = blockIdx.x;
  const auto rec = const_space(P->cuts + i0);
  const int n = uni(rec->parts);
  if (blockIdx.y == 0) clear_loose_tokens(P, blockIdx.x, gridDim.x);
  if (n <= 0) return;
  const int hb = uni(rec->head), qt = uni(rec->tile);
  const PagedSeq e = paged_seq_uniform(P, rec->b);
  const int hblk = cdiv(P->group, P->hw), kvh = hb / hblk, h_in = (hb - kvh * hblk) * P->hw + wv % P->hw;
  const int tok = qt * TilePlan::tokens(P) + 32 * (wv / P->hw) + l32;
  const bool live = tok < e.lq && h_in < P->group;
  const int h = kvh * P->group + h_in;
  const float c2 = P->c2;
  float M = kNegInf, L = 0.f;
  f32x4_t o[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) o[g] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;  // parts in flight
  if (live) {
    for (int j0 = by_part ? U * own : 0; j0 < n; j0 += by_part ? 4 * U : U) {
      f32x4_t x[U][4];
      f32x2 ml[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int j = min(j0 + k, n - 1);  // (past the last: not added below)
        const int64_t slot = (int64_t)(j == 0 ? 2 * i0 + 1 : 2 * (i0 + j)) * 4 + wv;
        const float* src = P->part + slot * 32 * D + d * 1024 + 4 * lane;
        ml[k] = *(const f32x2*)(P->ml + 2 * (slot * 32 + l32));
#pragma unroll
        for (int g = 0; g < 4; ++g) x[k][g] = *(const f32x4_t*)(src + g * 256);
      }
      float m = M;
#pragma unroll
      for (int k = 0; k < U; ++k) m = fmaxf(m, ml[k][0]);
      const float ref = m == kNegInf ? 0.f : m;
      const float wa = weight2((M - ref) * c2);
      L *= wa;
#pragma unroll
      for (int g = 0; g < 4; ++g) o[g] *= wa;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (j0 + k >= n) break;  // (uniform)
        const float wb = weight2((ml[k][0] - ref) * c2);
        L += ml[k][1] * wb;
#pragma unroll
        for (int g = 0; g < 4; ++g) o[g] += x[k][g] * wb;
      }
      M = m;
    }
  }
  if (by_part) {
#pragma unroll
    for (int g = 0; g < 4; ++g) part[own][g][lane] = o[g];
    if (hl == 0) stat[own][0][l32] = M, stat[own][1][l32] = L;
    __syncthreads();
    if (own != 0) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float mw = stat[w][0][l32], m = fmaxf(M, mw);
      const float ref = m == kNegInf ? 0.f : m;
      const float wa = weight2((M - ref) * c2), wb = weight2((mw - ref) * c2);
      L = L * wa + stat[w][1][l32] * wb;
#pragma unroll
      for (int g = 0; g < 4; ++g) o[g] = o[g] * wa + part[w][g][lane] * wb;
      M = m;
    }
  }
  if (!live) return;
  const float inv = 1.f / (L + 1e-6f);
  uint16_t* orow = (uint16_t*)P->o.ptr + (int64_t)(e.q0 + tok) * P->o.ss + (int64_t)h * P->o.sh;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    u32x2 val;
    val[0] = pack_e<F16>(o[g][0] * inv, o[g][1] * inv);
    val[1] = pack_e<F16>(o[g][2] * inv, o[g][3] * inv);
    *(u32x2*)(orow + d * 32 + 8 * g + 4 * hl) = val;
  }
  if (d == 0 && hl == 0 && P->lse.ptr)
    ((float*)P->lse.ptr)[(int64_t)(e.q0 + tok) * P->lse.ss + (int64_t)h * P->lse.sh] =
        M == kNegInf ? kNegInf : M * P->c + __builtin_amdgcn_logf(L + 1e-6f) * kLn2;
}

#define FNA2_TILE(D, RPL, HW)                                                               \
  __global__ __launch_bounds__(256, tile_occ(D, RPL, HW)) void paged_tile_d##D##_r##RPL##_h##HW( \
      const PagedParams) {                                                                \
    tile_body<D, RPL, HW, false, false>();                                                         \
  }                                                                                         \
  __global__ __launch_bounds__(256, tile_occ(D, RPL, HW)) void                              \
      paged_tile_d##D##_r##RPL##_h##HW##_f16(const PagedParams) {                         \
    tile_body<D, RPL, HW, true, false>();                                                          \
  }
FNA2_TILE(64, 0, 1)
FNA2_TILE(64, 32, 1)
FNA2_TILE(64, 32, 2)
FNA2_TILE(64, 32, 4)
FNA2_TILE(64, 64, 1)
FNA2_TILE(64, 64, 2)
FNA2_TILE(64, 64, 4)
FNA2_TILE(128, 0, 1)
FNA2_TILE(128, 32, 1)
FNA2_TILE(128, 32, 2)
FNA2_TILE(128, 32, 4)
FNA2_TILE(128, 64, 1)
FNA2_TILE(128, 64, 2)
FNA2_TILE(128, 64, 4)
#undef FNA2_TILE

}  // namespace

int paged_tile_per_cu(int D, int rpl, int hw, bool two) { return tile_occ(D, rpl, hw, two); }

size_t paged_tile_slot(int D) { return (size_t)128 * D * 4; }

hipError_t launch_paged_tile(const PagedParams& P, int rpl, hipStream_t s) {
  void (*k)(const PagedParams) = nullptr;
#define FNA2_TILE_OF(D, RPL, HW) \
  (P.f16 ? paged_tile_d##D##_r##RPL##_h##HW##_f16 : paged_tile_d##D##_r##RPL##_h##HW)
#define FNA2_TILE_HW(D, RPL)                             \
  (P.hw == 1   ? FNA2_TILE_OF(D, RPL, 1)                 \
   : P.hw == 2 ? FNA2_TILE_OF(D, RPL, 2)                 \
   : P.hw == 4 ? FNA2_TILE_OF(D, RPL, 4)                 \
               : nullptr)
  if (P.D == 64)
    k = rpl == 0 ? FNA2_TILE_OF(64, 0, 1) : rpl == 32 ? FNA2_TILE_HW(64, 32) : FNA2_TILE_HW(64, 64);
  if (P.D == 128)
    k = rpl == 0 ? FNA2_TILE_OF(128, 0, 1) : rpl == 32 ? FNA2_TILE_HW(128, 32) : FNA2_TILE_HW(128, 64);
#undef FNA2_TILE_HW
#undef FNA2_TILE_OF
  if (!k) return hipErrorInvalidValue;
  hipLaunchKernelGGL(k, dim3((uint32_t)P.waves), dim3(256), 0, s, P);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid((uint32_t)P.waves, (uint32_t)(P.D / 32 * (P.merge_by_part ? 4 : 1)));
  void (*m)(const PagedParams) =
      P.D == 64 ? (P.f16 ? paged_tile_merge_kernel<64, true> : paged_tile_merge_kernel<64, false>)
                : (P.f16 ? paged_tile_merge_kernel<128, true> : paged_tile_merge_kernel<128, false>);
  hipLaunchKernelGGL(m, grid, dim3(256), 0, s, P);
  return hipGetLastError();
}

}  // namespace fna2
