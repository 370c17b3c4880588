// fna2_paged_shared.hip — attention over a paged cache in which groups of
// sequences share their first rows.
//
// Rows that a group of sequences shares (one prompt, one document, many
// questions) are attended to once for the tokens of all of them: softmax over
// the shared rows and over a sequence's own are two parts of one, joined as
// parts of rows are,
//     m = max(m1, m2),  l = l1 e^{m1-m} + l2 e^{m2-m},
//     O = (O1 e^{m1-m} + O2 e^{m2-m}) / (l + 1e-6).
// A group shares the rows that lie before every chunk of its tokens, so that no
// token's mask cuts them, in whole key steps of 32; what is left over is each
// sequence's own.
//
// The plan forms the units, key steps of tiles of 128 (token, head) columns, of the
// groups' shared rows with all the group's tokens and of the sequences' own rows, and cuts
// them into equal runs: every workgroup for itself where 64 sequences and 64 groups at
// most fit its LDS, else in a launch of its own, in one workgroup's registers up to 1024 (5 groups of
// 22 sequences: the call 48 us with the general form, 39 so).  The tile kernel
// (fna2_paged_tile_dev.h) takes a run a workgroup, with P in two parts for chunks that
// fna2_paged_attn's packed kernel would take, which has it so: a layer that begins to share is
// then as precise as before (P in one part: 1.4 times the error of the output's rounding alone; two
// cost 64 tokens over 16384 shared rows 104 us for 99, 4 over 2000 18.3 for 17.4).  A tile that runs cut, or
// that is one of two for its tokens, leaves unnormalised parts; the join, another
// launch, adds a token's parts up in a fixed order.
//
// Bound by memory where the sequences' own rows are many: 64 tokens over 16384 shared and up
// to 1000 own rows, 32 heads over 8 of 128, rank 32 96 + 8 us (tiles + join; 406 MB at 4.2 TB/s, the
// least that it can read being 395); by the matrix cores where chunks are long: 16 x up to 128 tokens
// over 8192, rank 64 333 to 352, up to 0.87 10^15 operations a second, 24 of them the join's; by chains of dependent loads (plan, page
// ids, rows, parts, join) where there is little: 4 tokens over 2000 rows 13 + 6.
#include <algorithm>

#include "fna2_paged_tile_dev.h"

namespace fna2 {

namespace {

// The plan where a workgroup has no room for it in LDS.
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void paged_shared_plan_kernel(const PagedSharedParams) {
  SArg S = sargs();
  __shared__ int64_t sums[kPlanThreads / 64];
  shared_plan<kPlanThreads>(S, SharedPlanRef{S->meta, S->groups, S->group_ends, S->seqs, S->ends}, sums);
}

__global__ __launch_bounds__(kSharedMid) void paged_shared_plan_mid_kernel(const PagedSharedParams) {
  SArg S = sargs();
  __shared__ SharedMidPlan mid;
  shared_plan_mid(S, SharedPlanRef{S->meta, S->groups, S->group_ends, S->seqs, S->ends}, mid);
}

// The join: a workgroup takes 32 tokens, a query head and 32 features; its NW
// waves every NW-th group of four parts each.  Column = lane % 32, as in a
// tile, so that the parts of tokens that are neighbours in a tile are read as they lie.
// Four waves where there are few workgroups, so that many parts are in flight (the whole call,
// one wave against four: 32 sequences of 5 tokens over 3001 shared rows 41.0 us, 34.5; 4 of 1
// over 2000 23.7, 18.8), one where the workgroups alone fill the chip (10 of 100 tokens over 1024
// rows 38.9, 42.3; 24 of 195 over 131 43.9, 48.3).
template <int D, bool F16, int NW>
__global__ __launch_bounds__(64 * NW) void paged_shared_join_kernel(const PagedSharedParams) {
  SArg S = sargs();
  KArg P = &S->p;
  __shared__ f32x4_t part[NW][4][64];
  __shared__ float stat[NW][2][32];
  const int lane = threadIdx.x & 63, own = uni(threadIdx.x >> 6);
  const int l32 = lane & 31, hl = lane >> 5;
  const int h = uni(blockIdx.y / (D / 32)), d = uni(blockIdx.y % (D / 32));
  const int tok = 32 * blockIdx.x + l32;
  const int hw = P->hw, hblk = cdiv(P->group, hw);
  const int kvh = h / P->group, h_in = h - kvh * P->group;
  const int hb = kvh * hblk + h_in / hw, hin = h_in % hw;
  const int t0 = min(max(uni(*const_space(P->cu)), 0), P->T);
  const int t1 = min(max(uni(*const_space(P->cu + P->N)), t0), P->T);
  const bool loose = tok < P->T && (tok < t0 || tok >= t1);
  // (loaded with the bounds, not behind them: a token of no sequence has no record, and
  // none is used)
  SharedRec a{}, b{};
  if (tok < P->T) {
    a = S->recs[(int64_t)hb * P->T + tok];
    b = S->recs[(int64_t)(P->H_KV * hblk + hb) * P->T + tok];
  }
  const bool live = tok >= t0 && tok < t1 && a.parts >= 0, has = live && (a.at & kSharedHas);
  auto parts = [&](int x) { return min(max(x, 0), P->waves); };  // (whatever cu holds, the loop ends)
  const int na = live ? max(parts(a.parts), 1) : 0, nc = has ? parts(a.full) : 0;
  const int nb = has && (a.at & kSharedRest) ? max(parts(b.parts), 1) : 0, n = nc + nb + na;
  const float c2 = P->c2;
  float M = kNegInf, L = 0.f;
  f32x4_t o[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) o[g] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;  // parts in flight
  for (int j0 = U * own; __builtin_amdgcn_ballot_w64(j0 < n) != 0; j0 += NW * U) {
    f32x4_t x[U][4];
    f32x2 ml[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      ml[k] = f32x2{kNegInf, 0.f};
#pragma unroll
      for (int g = 0; g < 4; ++g) x[k][g] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      int j = j0 + k;
      if (j >= n) continue;
      // the shared rows' chunks, their rest, the token's own rows
      const int which = j < nc ? 0 : j < nc + nb ? 1 : 2;
      const SharedRec& r = which == 1 ? b : a;
      j -= which == 0 ? 0 : which == 1 ? nc : nc + nb;
      const float *src, *src_ml;
      int step;
      if (which != 0 && r.parts == 0) {
        const int64_t row = ((int64_t)(which == 1) * P->T + tok) * P->H + h;
        src = S->whole + row * D + 32 * d + 4 * hl;
        src_ml = S->whole_ml + 2 * row;
        step = 8;
      } else {
        const int at = which == 0 ? a.at0 & 0x7f : (r.at >> 16) & 0x7f;
        const int run = which == 0 ? a.run0 + j * a.stride : (r.at & 0xffff) + j;
        const int wv = ((at >> 5) * hw + hin) & 3;
        const int64_t slot = (2 * (int64_t)min(max(run, 0), P->waves - 1) + (which == 0 || j == 0 ? 1 : 0)) * 4 + wv;
        src = P->part + slot * 32 * D + d * 1024 + 4 * ((at & 31) + 32 * hl);
        src_ml = P->ml + 2 * (slot * 32 + (at & 31));
        step = 256;
      }
      ml[k] = *(const f32x2*)src_ml;
#pragma unroll
      for (int g = 0; g < 4; ++g) x[k][g] = *(const f32x4_t*)(src + g * step);
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
      const float wb = weight2((ml[k][0] - ref) * c2);
      L += ml[k][1] * wb;
#pragma unroll
      for (int g = 0; g < 4; ++g) o[g] += x[k][g] * wb;
    }
    M = m;
  }
#pragma unroll
  for (int g = 0; g < 4; ++g) part[own][g][lane] = o[g];
  if (hl == 0) stat[own][0][l32] = M, stat[own][1][l32] = L;
  __syncthreads();
  if (own != 0 || !(live || loose)) return;
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    const float mw = stat[w][0][l32], m = fmaxf(M, mw);
    const float ref = m == kNegInf ? 0.f : m;
    const float wa = weight2((M - ref) * c2), wb = weight2((mw - ref) * c2);
    L = L * wa + stat[w][1][l32] * wb;
#pragma unroll
    for (int g = 0; g < 4; ++g) o[g] = o[g] * wa + part[w][g][lane] * wb;
    M = m;
  }
  const float inv = 1.f / (L + 1e-6f);
  uint16_t* orow = (uint16_t*)P->o.ptr + (int64_t)tok * P->o.ss + (int64_t)h * P->o.sh;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    u32x2 val;
    val[0] = pack_e<F16>(o[g][0] * inv, o[g][1] * inv);
    val[1] = pack_e<F16>(o[g][2] * inv, o[g][3] * inv);
    *(u32x2*)(orow + d * 32 + 8 * g + 4 * hl) = val;
  }
  if (d == 0 && hl == 0 && P->lse.ptr)
    ((float*)P->lse.ptr)[(int64_t)tok * P->lse.ss + (int64_t)h * P->lse.sh] =
        M == kNegInf ? kNegInf : M * P->c + __builtin_amdgcn_logf(L + 1e-6f) * kLn2;
}

#define FNA2_SHARED(D, RPL, HW)                                                                   \
  __global__ __launch_bounds__(256, tile_occ(D, RPL, HW)) void                                    \
      paged_shared_d##D##_r##RPL##_h##HW(const PagedSharedParams) {                               \
    tile_body<D, RPL, HW, false, true>();                                                         \
  }                                                                                               \
  __global__ __launch_bounds__(256, tile_occ(D, RPL, HW)) void                                    \
      paged_shared_d##D##_r##RPL##_h##HW##_f16(const PagedSharedParams) {                         \
    tile_body<D, RPL, HW, true, true>();                                                          \
  }                                                                                               \
  __global__ __launch_bounds__(256, tile_occ(D, RPL, HW, true)) void                              \
      paged_shared_d##D##_r##RPL##_h##HW##_p2(const PagedSharedParams) {                          \
    tile_body<D, RPL, HW, false, true, true>();                                                   \
  }                                                                                               \
  __global__ __launch_bounds__(256, tile_occ(D, RPL, HW, true)) void                              \
      paged_shared_d##D##_r##RPL##_h##HW##_p2_f16(const PagedSharedParams) {                      \
    tile_body<D, RPL, HW, true, true, true>();                                                    \
  }
FNA2_SHARED(64, 0, 1)
FNA2_SHARED(64, 32, 1)
FNA2_SHARED(64, 32, 2)
FNA2_SHARED(64, 32, 4)
FNA2_SHARED(64, 64, 1)
FNA2_SHARED(64, 64, 2)
FNA2_SHARED(64, 64, 4)
FNA2_SHARED(128, 0, 1)
FNA2_SHARED(128, 32, 1)
FNA2_SHARED(128, 32, 2)
FNA2_SHARED(128, 32, 4)
FNA2_SHARED(128, 64, 1)
FNA2_SHARED(128, 64, 2)
FNA2_SHARED(128, 64, 4)
#undef FNA2_SHARED

}  // namespace

hipError_t launch_paged_shared(const PagedSharedParams& S, int rpl, hipStream_t s) {
  const PagedParams& P = S.p;
  void (*k)(const PagedSharedParams) = nullptr;
#define FNA2_SHARED_OF(D, RPL, HW) \
  (S.two ? (P.f16 ? paged_shared_d##D##_r##RPL##_h##HW##_p2_f16 : paged_shared_d##D##_r##RPL##_h##HW##_p2) \
         : (P.f16 ? paged_shared_d##D##_r##RPL##_h##HW##_f16 : paged_shared_d##D##_r##RPL##_h##HW))
#define FNA2_SHARED_HW(D, RPL)                             \
  (P.hw == 1   ? FNA2_SHARED_OF(D, RPL, 1)                 \
   : P.hw == 2 ? FNA2_SHARED_OF(D, RPL, 2)                 \
   : P.hw == 4 ? FNA2_SHARED_OF(D, RPL, 4)                 \
               : nullptr)
  if (P.D == 64)
    k = rpl == 0 ? FNA2_SHARED_OF(64, 0, 1) : rpl == 32 ? FNA2_SHARED_HW(64, 32) : FNA2_SHARED_HW(64, 64);
  if (P.D == 128)
    k = rpl == 0 ? FNA2_SHARED_OF(128, 0, 1) : rpl == 32 ? FNA2_SHARED_HW(128, 32) : FNA2_SHARED_HW(128, 64);
#undef FNA2_SHARED_HW
#undef FNA2_SHARED_OF
  if (!k) return hipErrorInvalidValue;
  hipError_t e = hipSuccess;
  if (!S.small) {
    const int most = std::max(P.N, S.G);
    if (most <= kSharedMid)
      hipLaunchKernelGGL(paged_shared_plan_mid_kernel, dim3(1), dim3((most + 63) / 64 * 64), 0, s, S);
    else
      hipLaunchKernelGGL(paged_shared_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, S);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(k, dim3((uint32_t)P.waves), dim3(256), 0, s, S);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid((uint32_t)((P.T + 31) / 32), (uint32_t)(P.H * (P.D / 32)));
  const bool one = (int64_t)grid.x * grid.y >= 1024;  // (4 a CU)
#define FNA2_JOIN(D, F16) (one ? paged_shared_join_kernel<D, F16, 1> : paged_shared_join_kernel<D, F16, 4>)
  void (*m)(const PagedSharedParams) = P.D == 64 ? (P.f16 ? FNA2_JOIN(64, true) : FNA2_JOIN(64, false))
                                                 : (P.f16 ? FNA2_JOIN(128, true) : FNA2_JOIN(128, false));
#undef FNA2_JOIN
  hipLaunchKernelGGL(m, grid, dim3(one ? 64 : 256), 0, s, S);
  return hipGetLastError();
}

}  // namespace fna2
