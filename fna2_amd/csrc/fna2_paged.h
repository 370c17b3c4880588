// fna2_paged.h — the paged cache's kernels: parameters, and the parts of the
// device code that they share.
#pragma once

#include "fna2_device.h"

namespace fna2 {

// A paged cache and the chunk of new tokens that belongs to it.  Row j of
// sequence b: row j % ps of page table[b * tstride + j / ps]; page p, head
// h, row r of a pool at ptr + p * sb + h * sh + r * ss.
struct PagedParams {
  int N, T;
  int H, H_KV, H_G, D, R, group;
  int ps, npages, width;
  int64_t tstride;
  const int* table;
  const int* lens;
  const int* cu;
  TView k, v, rk;  // pools: sb page, sh head, ss row
  TView q, rq, o, lse;  // [T, heads, .]: ss token, sh head; lse.ptr may be null
  const float* gs;
  int causal, f16;
  float c, c2, qa;  // as in Problem
  // Column tiles (the packed kernel): gsub query heads of a KV head times
  // tpt tokens are the columns of a tile; nsub such groups a KV head.
  int gsub, nsub, tpt;
  int waves;      // resident waves that share the work
  int min_steps;  // key steps a wave takes at least
  float* part;    // [2 * waves][cols][D] unnormalised numerators of split tiles
  float* ml;      // [2 * waves][cols] (max, sum)
};

// A sequence's tokens and rows, clamped so that no access leaves [0, T) or
// its row of the table.
struct PagedSeq {
  int q0, lq, lk;
};
__device__ __forceinline__ PagedSeq paged_clamp(const PagedParams& P, int qs, int qe, int lk) {
  PagedSeq s;
  qs = min(max(qs, 0), P.T);
  qe = min(max(qe, qs), P.T);
  s.q0 = qs;
  s.lq = qe - qs;
  s.lk = min(max(lk, 0), P.width * P.ps);
  return s;
}
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& P, int b) {
  return paged_clamp(P, P.cu[b], P.cu[b + 1], P.lens[b]);
}
__device__ __forceinline__ PagedSeq paged_seq_uniform(const PagedParams& P, int b) {
  b = uni(b);
  const auto cu = const_space(P.cu);
  return paged_clamp(P, uni(cu[b]), uni(cu[b + 1]), uni(*const_space(P.lens + b)));
}

// Work that the host cannot count (the lengths are on the device): the
// sequences' units, laid end to end, are found again by every wave from the
// lengths alone.  `units(s)` is a sequence's count.
template <typename F>
__device__ __forceinline__ int64_t wave_total(const PagedParams& P, int lane, F&& units) {
  int64_t sum = 0;
  for (int b = lane; b < P.N; b += 64) sum += units(paged_seq(P, b));
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
  return sum;
}

// The sequence that holds unit u (0 <= u < total), and u's place in it.
struct PagedAt {
  int b;
  int64_t rem;
};
template <typename F>
__device__ __forceinline__ PagedAt wave_locate(const PagedParams& P, int lane, int64_t u,
                                               F&& units) {
  int64_t base = 0;
  for (int b0 = 0; b0 < P.N; b0 += 64) {
    const int b = b0 + lane;
    const int64_t mine = b < P.N ? units(paged_seq(P, b)) : 0;
    int64_t end = mine;  // inclusive sum over the lanes
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const int64_t o = __shfl_up(end, m);
      if (lane >= m) end += o;
    }
    const uint64_t past = __builtin_amdgcn_ballot_w64(base + end > u);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int64_t start = __shfl(end - mine, l) + base;
      PagedAt at;
      at.b = uni(b0 + l);
      const int64_t rem = u - start;
      at.rem = (int64_t)(((uint64_t)(uint32_t)uni((int)(rem >> 32)) << 32) | (uint32_t)uni((int)rem));
      return at;
    }
    base += __shfl(end, 63);
  }
  return PagedAt{P.N, 0};
}

// The page of row group `row` (a multiple of 16, below lk) and the row's
// place in it, stepped 16 rows at a time.
struct PageCursor {
  int page, off;
  __device__ __forceinline__ void at(const PagedParams& P, int row) {
    page = row / P.ps;
    off = row - page * P.ps;
  }
  __device__ __forceinline__ void next(const PagedParams& P) {
    off += 16;
    if (off >= P.ps) {
      off = 0;
      ++page;
    }
  }
};

__device__ __forceinline__ int64_t uni64(int64_t x) {
  return (int64_t)(((uint64_t)(uint32_t)uni((int)(x >> 32)) << 32) | (uint32_t)uni((int)x));
}

// The packed kernel's units (key steps of 32 rows of a column tile) and the
// share of each wave: shared with the kernel that joins split tiles.
struct PackedPlan {
  int64_t total, per;
  __device__ __forceinline__ static int steps(const PagedSeq& s) { return max(cdiv(s.lk, 32), 1); }
  __device__ __forceinline__ static int64_t units(const PagedParams& P, const PagedSeq& s) {
    return (int64_t)cdiv(s.lq, P.tpt) * (P.H_KV * P.nsub) * steps(s);
  }
  __device__ __forceinline__ PackedPlan(const PagedParams& P, int lane) {
    total = uni64(wave_total(P, lane, [&](const PagedSeq& s) { return units(P, s); }));
    per = max((total + P.waves - 1) / P.waves, (int64_t)P.min_steps);
  }
};

// Kernel launches (fna2_paged_attn.hip, fna2_paged_rows.hip).
int paged_rank_chunks(int rch);      // as decode_rank_chunks
int paged_waves_per_cu(int D, int rc);  // resident waves of the packed kernel
hipError_t launch_paged_packed(const PagedParams& P, int rc, hipStream_t s);
hipError_t launch_paged_merge(const PagedParams& P, hipStream_t s);

struct PagedWeightsParams {
  PagedParams p;
  float* w;
  int64_t w_sb, w_sh;
  int cap;
  int grid;
};
hipError_t launch_paged_weights(const PagedWeightsParams& P, hipStream_t s);

struct PagedAppendParams {
  PagedParams p;  // q, k, v pools and the chunk; o is q_out
  TView kn, vn, rkn;  // the new rows [T, heads, .]
  const int* pos;
  const float* inv_freq;
  const float* wq;
  const float* wk;
  float eps;
};
hipError_t launch_paged_append(const PagedAppendParams& P, hipStream_t s);

struct PagedEvictParams {
  PagedParams p;
  int budget, recent, first;
  const float* w;
  int64_t w_sb, w_sh;
  int cap;
  float* w_out;
  int* kept;
  int* new_lens;
};
hipError_t launch_paged_select(const PagedEvictParams& P, hipStream_t s);
hipError_t launch_paged_compact(const PagedEvictParams& P, hipStream_t s);

}  // namespace fna2
