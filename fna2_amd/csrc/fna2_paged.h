// fna2_paged.h — the paged cache's kernels: parameters, and the parts of the
// device code that they share.
#pragma once

#include "fna2_device.h"

namespace fna2 {

// A tile that the end of run i cuts (parts > 0), if no earlier run's end does:
// what the merge needs to join its parts, which lie with runs i .. i + parts - 1.
struct __attribute__((aligned(16))) PagedCut {
  int b, head, tile, parts;  // sequence; block of heads; tile of tokens
};

// A paged cache and the chunk of new tokens that belongs to it.  Row j of
// sequence b: row j % ps of page table[b * tstride + j / ps]; page p, head
// h, row r of a pool at ptr + p * sb + h * sh + r * ss.
struct PagedParams {
  int N, T;
  int H, H_KV, H_G, D, R, group;
  int ps, npages, width;
  uint32_t ps_mul;  // row / ps = (row / 16) ps_mul >> ps_shift
  int ps_shift;
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
  int waves;      // resident waves (workgroups of the tile kernel) that share the work
  int min_steps;  // tile kernel: key steps a run takes at least
  int hw;         // tile kernel: query heads of a KV head that a workgroup's waves take
  struct PagedCut* cuts;  // [waves]
  int merge_runs;     // runs that a workgroup of the merge looks through (<= 64)
  int merge_by_part;  // ... with a workgroup for every column
  float* part;    // [2 * waves] slots of unnormalised numerators of split tiles
  float* ml;      // [2 * waves][columns of a tile] (max, sum)
  // Scores that the packed kernel leaves for the weights: [N][H_KV * nsub][columns
  // of a tile][srows], of the sequences whose chunk one tile holds; or null.
  float* scores;
  int srows;  // rows of the table, rounded up to 32
};

// The kernels read their parameters where the launch put them, through a
// pointer that the compiler cannot see through (kargs()): it then loads a field
// where that is used.  Read as an ordinary argument, all of the block stays in
// scalar registers through the key loop and pushes the loop's own out (100
// spilled).  PagedParams is the first member of every parameter block here.
typedef const __attribute__((address_space(4))) PagedParams* KArg;
__device__ __forceinline__ KArg kargs() {
  KArg p = (KArg)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// The scores of group `sg` (kvh * nsub + sub) of sequence b.
__device__ __forceinline__ float* paged_scores(KArg P, int b, int sg) {
  return P->scores + ((int64_t)b * (P->H_KV * P->nsub) + sg) * (P->gsub * P->tpt) * P->srows;
}

// A sequence's tokens and rows, clamped so that no access leaves [0, T) or
// its row of the table.  off: the first token's row, lk - lq; more where the
// sequence has outgrown its table (whose rows the tokens past it all see).
struct PagedSeq {
  int q0, lq, lk, off;
};
__device__ __forceinline__ PagedSeq paged_clamp(KArg P, int qs, int qe, int len) {
  PagedSeq s;
  qs = min(max(qs, 0), P->T);
  qe = min(max(qe, qs), P->T);
  s.q0 = qs;
  s.lq = qe - qs;
  const int rows = P->width * P->ps;
  len = max(len, 0);
  s.lk = min(len, rows);
  s.off = min(len - s.lq, rows);
  return s;
}
__device__ __forceinline__ PagedSeq paged_seq(KArg P, int b) {
  return paged_clamp(P, P->cu[b], P->cu[b + 1], P->lens[b]);
}
__device__ __forceinline__ PagedSeq paged_seq_uniform(KArg P, int b) {
  b = uni(b);
  const auto cu = const_space(P->cu);
  return paged_clamp(P, uni(cu[b]), uni(cu[b + 1]), uni(*const_space(P->lens + b)));
}

__device__ __forceinline__ int64_t lane64(int64_t x, int l) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)x, l);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(x >> 32), l);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t uni64(int64_t x) { return lane64(x, 0); }

// Sum over the lanes up to and including this one, in moves between lanes'
// registers (shuffles go through LDS: 1 us for the six).
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t dpp_add64(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, false);
  return x + (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t lane_scan64(int64_t x) {
  x = dpp_add64<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8: within 16 lanes
  x = dpp_add64<0x112, 0xf>(x);
  x = dpp_add64<0x114, 0xf>(x);
  x = dpp_add64<0x118, 0xf>(x);
  x = dpp_add64<0x142, 0xa>(x);  // row_bcast 15: rows 1 and 3 take the row before
  return dpp_add64<0x143, 0xc>(x);  // row_bcast 31: rows 2 and 3 the first two
}

// Quotient of nonnegative numbers, by 32-bit division where they fit.
__device__ __forceinline__ int64_t div64(int64_t a, int64_t b) {
  if (((uint64_t)(a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

// Work that the host cannot count (the lengths are on the device): the
// sequences' units, laid end to end, are found again by every wave from the
// lengths alone.  `units(s)` is a sequence's count.  seek(u): the sequence that holds
// unit u (0 <= u < total) and u's place in it.
struct PagedAt {
  int b;
  int64_t rem;
  PagedSeq s;
};
template <typename F>
struct SeqWork {
  F units;
  int64_t total, base, mine, end;  // of the block of 64 sequences scanned last
  PagedSeq s;
  __device__ __forceinline__ void scan(KArg P, int lane, int b0, int64_t before) {
    const int b = b0 + lane;
    s = PagedSeq{0, 0, 0, 0};
    if (b < P->N) s = paged_seq(P, b);
    base = before;
    mine = b < P->N ? units(s) : 0;
    end = before + lane_scan64(mine);
  }
  __device__ __forceinline__ SeqWork(KArg P, int lane, F f) : units(f), total(0) {
    for (int b0 = 0; b0 < P->N; b0 += 64) {
      scan(P, lane, b0, total);
      total = lane64(end, 63);
    }
  }
  __device__ __forceinline__ PagedAt seek(KArg P, int lane, int64_t u) {
    int b0 = 0;
    if (P->N > 64) {
      int64_t sum = 0;
      while (true) {
        scan(P, lane, b0, sum);
        sum = lane64(end, 63);
        if (sum > u || b0 + 64 >= P->N) break;
        b0 += 64;
      }
    }
    const int l = uni(__builtin_ctzll(__builtin_amdgcn_ballot_w64(end > u) | ((uint64_t)1 << 63)));
    PagedAt at;
    at.b = b0 + l;
    at.rem = u - lane64(end - mine, l);
    at.s = PagedSeq{__builtin_amdgcn_readlane(s.q0, l), __builtin_amdgcn_readlane(s.lq, l),
                    __builtin_amdgcn_readlane(s.lk, l), __builtin_amdgcn_readlane(s.off, l)};
    return at;
  }
};

// Zeros, and LSE -inf, for the tokens of no sequence: workgroup `i` of `n`.
__device__ __forceinline__ void clear_loose_tokens(KArg P, int i, int n) {
  const int t0 = min(max(uni(*const_space(P->cu)), 0), P->T);
  const int t1 = min(max(uni(*const_space(P->cu + P->N)), t0), P->T);
  const int64_t rows = (int64_t)(t0 + P->T - t1) * P->H;
  for (int64_t r = i; r < rows; r += n) {
    const int h = (int)(r % P->H);
    int t = (int)(r / P->H);
    if (t >= t0) t += t1 - t0;
    uint16_t* o = (uint16_t*)P->o.ptr + (int64_t)t * P->o.ss + (int64_t)h * P->o.sh;
    if (threadIdx.x < P->D / 8) *(u32x4*)(o + 8 * threadIdx.x) = u32x4{0, 0, 0, 0};
    if (threadIdx.x == 0 && P->lse.ptr)
      ((float*)P->lse.ptr)[(int64_t)t * P->lse.ss + (int64_t)h * P->lse.sh] = kNegInf;
  }
}

// The page of row `row` (below 2^30).
__device__ __forceinline__ int page_of(uint32_t mul, int shift, int row) {
  return (int)(((uint64_t)(uint32_t)(row >> 4) * mul) >> shift);
}

// x / d and x % d for lane numbers (x < 64) and d <= 64.
__device__ __forceinline__ int small_div(int x, int d) {
  return (x * (65536 / d + 1)) >> 16;
}

// The units of a run: an equal share for each of the resident waves
// (workgroups), `least` at least.
__device__ __forceinline__ int64_t run_units(KArg P, int64_t total, int64_t least) {
  return max(div64(total + P->waves - 1, P->waves), least);
}

// The packed kernel's units: key steps of 32 rows of a column tile.
struct PackedPlan {
  __device__ __forceinline__ static int steps(const PagedSeq& s) { return max(cdiv(s.lk, 32), 1); }
  __device__ __forceinline__ static int64_t units(KArg P, const PagedSeq& s) {
    return (int64_t)cdiv(s.lq, P->tpt) * (P->H_KV * P->nsub) * steps(s);
  }
};

// The tile kernel's units: key steps of 32 rows of a tile of 32 * (4 / hw)
// tokens and hw query heads of a KV head (a block; the last one of a KV head
// may be short of heads).  Tile i of a sequence sees, causal, the rows up to
// its last token's: ceil((off + min((i + 1) TB, lq)) / 32) units, one at least.
struct TilePlan {
  __device__ __forceinline__ static int tokens(KArg P) { return 128 / P->hw; }
  __device__ __forceinline__ static int blocks(KArg P) {
    return P->H_KV * cdiv(P->group, P->hw);
  }
  // Units of tiles 0 .. m - 1, none of them the sequence's last.
  __device__ __forceinline__ static int64_t before(KArg P, const PagedSeq& s, int m) {
    if (!P->causal) return (int64_t)m * max(cdiv(s.lk, 32), 1);
    const int t = 4 / P->hw, off = s.off;
    if (off + m * tokens(P) > s.lk) {  // (the last ones of a sequence past its table see all its rows)
      const int n = min(max(s.lk - off, 0) / tokens(P), m);
      return before_end(t, off, n) + (int64_t)(m - n) * max(cdiv(s.lk, 32), 1);
    }
    return before_end(t, off, m);
  }
  __device__ __forceinline__ static int64_t before_end(int t, int off, int m) {
    const int64_t a = off >= 0 ? (off + 31) / 32 : -(-off / 32);  // ceil(off / 32)
    const int64_t n0 = a > 0 ? 0 : min((int64_t)m, -a / t);       // tiles that see no row
    return n0 + a * (m - n0) + t * ((int64_t)m * (m + 1) - n0 * (n0 + 1)) / 2;
  }
  __device__ __forceinline__ static int steps(KArg P, const PagedSeq& s, int i) {
    int vis = s.lk;
    if (P->causal) vis = min(vis, s.off + (i + 1) * tokens(P));
    return max(cdiv(max(vis, 0), 32), 1);
  }
  __device__ __forceinline__ static int64_t head_units(KArg P, const PagedSeq& s) {
    if (s.lq <= 0) return 0;
    const int n = cdiv(s.lq, tokens(P));
    return before(P, s, n - 1) + steps(P, s, n - 1);
  }
  __device__ __forceinline__ static int64_t units(KArg P, const PagedSeq& s) {
    return head_units(P, s) * blocks(P);
  }
  // The tile of unit r (of one block of heads) and the unit's place in it.
  __device__ __forceinline__ static int find(KArg P, const PagedSeq& s, int64_t& r) {
    int lo = 0, hi = cdiv(s.lq, tokens(P)) - 1;  // before(lo) <= r
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (before(P, s, mid) <= r) lo = mid;
      else hi = mid - 1;
    }
    r -= before(P, s, lo);
    return lo;
  }
};

// Kernel launches (fna2_paged_attn.hip, fna2_paged_tile.hip, fna2_paged_rows.hip).
int paged_tile_per_cu(int D, int rpl, int hw);  // resident workgroups of the tile kernel
size_t paged_tile_slot(int D);                  // bytes of a split tile's part
hipError_t launch_paged_tile(const PagedParams& P, int rpl, hipStream_t s);
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
  int key_waves;  // kernel for long chunks: waves of a workgroup on keys of their own, 4 or 2
};
int paged_weigh_per_cu(int D, int rc);  // resident workgroups
int paged_glance_per_cu(int D, int rc);  // ... waves of the kernel for short chunks
hipError_t launch_paged_glance(const PagedWeightsParams& P, int rc, hipStream_t s);
hipError_t launch_paged_weights(const PagedWeightsParams& P, int rc, hipStream_t s);

struct PagedAppendParams {
  PagedParams p;  // q, k, v pools and the chunk; o is q_out
  TView kn, vn, rkn;  // the new rows [T, heads, .]
  const int* pos;
  const int* shift;  // [N] added to a sequence's positions, or null
  const float* inv_freq;
  const float* wq;
  const float* wk;
  float eps;
  int share;  // waves of a token (set by the launch)
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
  int strip;  // (set by the launch)
};
hipError_t launch_paged_select(const PagedEvictParams& P, hipStream_t s);
hipError_t launch_paged_compact(const PagedEvictParams& P, hipStream_t s);

}  // namespace fna2
