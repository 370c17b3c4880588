// fna2_paged_shared.h — attention over a paged cache whose groups of sequences
// share their first rows: the plan that the tile kernel runs on.
#pragma once

#include "fna2_paged.h"

namespace fna2 {

// What the tiles of a virtual sequence are of: rows that a group shares, of
// all its tokens; the rows behind them, of one sequence; a sequence that shares
// none.
constexpr int kSharedAlone = 0, kSharedOwn = 1, kSharedPrefix = 2;

// A virtual sequence: s.lq tokens from s.q0 on over s.lk rows, the first of
// them row row0 of row `table` of the block table; s.off counts from there.
struct __attribute__((aligned(16))) SharedSeq {
  PagedSeq s;
  int row0, table, kind, pad;
};

// Where a token's part of a tile lies: the run in which the tile begins, the
// token's place in it (<< 16), and whether its sequence shares rows.  parts: 0
// where one run did the whole tile (SharedParams::whole), else as many as runs
// cut it into; -1: the output is written.
struct __attribute__((aligned(8))) SharedRec {
  int at, parts;
};
constexpr int kSharedHas = 1 << 24;

struct PagedSharedParams {
  PagedParams p;
  int G, V;  // groups; virtual sequences: the groups' rows, then the N sequences'
  const int* cu_groups;
  const int* shared_rows;
  SharedSeq* seqs;  // [V]
  int64_t* ends;    // [V] units up to and including a virtual sequence's
  SharedRec* recs;  // [own, prefix][blocks of heads][T]
  float* whole;     // [own, prefix][T][H][D] numerators of tiles that one run did
  float* whole_ml;  // [own, prefix][T][H] (max, sum)
};
typedef const __attribute__((address_space(4))) PagedSharedParams* SArg;
__device__ __forceinline__ SArg sargs() {
  SArg p = (SArg)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

__device__ __forceinline__ SharedSeq shared_seq_uniform(SArg S, int v) {
  const auto r = const_space((const int*)(S->seqs + uni(v)));
  SharedSeq x;
  x.s = PagedSeq{uni(r[0]), uni(r[1]), uni(r[2]), uni(r[3])};
  x.row0 = uni(r[4]);
  x.table = uni(r[5]);
  x.kind = uni(r[6]);
  x.pad = 0;
  return x;
}

// The virtual sequence that holds unit u (below the last end), and u's place in it:
// 64 ends at a time.
__device__ __forceinline__ int shared_seek(SArg S, int lane, int64_t u, int64_t& rem) {
  int lo = 0, n = S->V;
  const int64_t* ends = S->ends;
  while (n > 64) {
    const int step = (n + 63) / 64;
    const int64_t end = ends[lo + min((lane + 1) * step, n) - 1];
    const int l = uni(__builtin_ctzll(__builtin_amdgcn_ballot_w64(end > u) | ((uint64_t)1 << 63)));
    lo += l * step;
    n = min(step, n - l * step);
  }
  const int64_t end = ends[lo + min(lane, n - 1)];
  const int64_t before = lo + min(lane, n - 1) > 0 ? ends[lo + min(lane, n - 1) - 1] : 0;
  const int l = uni(__builtin_ctzll(__builtin_amdgcn_ballot_w64(end > u) | ((uint64_t)1 << 63)));
  rem = u - lane64(before, l);
  return lo + min(l, n - 1);
}

// Kernel launches (fna2_paged_shared.hip): the plan, the tiles, the join.
hipError_t launch_paged_shared(const PagedSharedParams& P, int rpl, hipStream_t s);

}  // namespace fna2
