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
  int row0, table, kind, group;
};

// A group's shared rows.  All its tiles have as many steps, of which the first
// full * chunk are cut alike: chunk c of block of heads hb of tile qt is the
// whole of run run0 + (c * blocks + hb) * tiles + qt.  So the runs of one KV head and
// chunk, which lie together on an XCD, read the same rows at the same time.  The
// rest of the rows is a virtual sequence like others.
struct __attribute__((aligned(16))) SharedGroup {
  PagedSeq s;  // of all the shared rows
  int64_t run0, end;  // the first of its full runs, and behind the last
  int table, tiles;
  int64_t full;
};

// Where a token's parts of a tile lie: the run in which the tile begins, the
// token's place in it (<< 16), flags.  parts: 0 where one run did the whole
// tile (PagedSharedParams::whole), else as many as runs cut it into; -1: the
// output is written.  With kSharedHas, of the shared rows: `full` chunks in runs run0, run0 +
// stride, ..., the token's place in their tiles, and with kSharedRest the rest.
struct __attribute__((aligned(16))) SharedRec {
  int at, parts, run0, stride, full, at0, pad[2];
};
constexpr int kSharedHas = 1 << 24, kSharedRest = 1 << 25;

struct __attribute__((aligned(16))) SharedMeta {
  int64_t per;    // units of a run: a tile's steps, and `start` for its start
  int64_t full;   // runs of the groups' full chunks, which come first
  int64_t units;  // of the virtual sequences, in the runs behind
};

// Where a plan lies.
struct SharedPlanRef {
  SharedMeta* meta;
  SharedGroup* groups;  // [G]
  int64_t* group_ends;  // [G] full runs up to and including a group's
  SharedSeq* seqs;      // [V]
  int64_t* ends;        // [V] units up to and including a virtual sequence's
};

constexpr int kSharedSmall = 64;  // sequences, and groups, of a plan in LDS
struct SharedSmallPlan {
  SharedMeta meta;
  SharedGroup groups[kSharedSmall];
  int64_t group_ends[kSharedSmall];
  SharedSeq seqs[2 * kSharedSmall];
  int64_t ends[2 * kSharedSmall];
};

constexpr int kSharedStart = 8;  // PagedSharedParams::start

struct PagedSharedParams {
  PagedParams p;
  int start;  // what starting and ending a tile costs, in steps
  float worth;
  int G, V;  // groups; virtual sequences: the rests of the groups' rows, then the N sequences'
  const int* cu_groups;
  const int* shared_rows;
  int small;  // every workgroup makes the plan in its LDS
  int two;    // P in two parts (set where fna2_paged_attn's packed kernel would run)
  SharedMeta* meta;  // ... else as in SharedPlanRef
  SharedGroup* groups;
  int64_t* group_ends;
  SharedSeq* seqs;
  int64_t* ends;
  SharedRec* recs;      // [own, rest][blocks of heads][T]
  float* whole;         // [own, rest][T][H][D] numerators of tiles that one run did
  float* whole_ml;      // [own, rest][T][H] (max, sum)
};
typedef const __attribute__((address_space(4))) PagedSharedParams* SArg;
__device__ __forceinline__ SArg sargs() {
  SArg p = (SArg)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

__device__ __forceinline__ SharedSeq shared_seq_uniform(const SharedSeq* seqs, int v) {
  SharedSeq x = seqs[uni(v)];
  x.s = PagedSeq{uni(x.s.q0), uni(x.s.lq), uni(x.s.lk), uni(x.s.off)};
  x.row0 = uni(x.row0);
  x.table = uni(x.table);
  x.kind = uni(x.kind);
  x.group = uni(x.group);
  return x;
}

// Units of a virtual sequence: TilePlan's steps, and S->start for every tile.
struct SharedUnits {
  __device__ __forceinline__ static int64_t head_units(SArg S, const PagedSeq& s) {
    if (s.lq <= 0) return 0;
    return TilePlan::head_units(&S->p, s) + (int64_t)S->start * cdiv(s.lq, TilePlan::tokens(&S->p));
  }
  __device__ __forceinline__ static int64_t units(SArg S, const PagedSeq& s) {
    return head_units(S, s) * TilePlan::blocks(&S->p);
  }
  // The tile of unit r (of one block of heads) and the unit's place in it.
  __device__ __forceinline__ static int find(SArg S, const PagedSeq& s, int64_t& r) {
    KArg P = &S->p;
    auto before = [&](int m) { return TilePlan::before(P, s, m) + (int64_t)m * S->start; };
    int lo = 0, hi = cdiv(s.lq, TilePlan::tokens(P)) - 1;  // before(lo) <= r
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (before(mid) <= r) lo = mid;
      else hi = mid - 1;
    }
    r -= before(lo);
    return lo;
  }
};

// The first of n ends that is above u (the last is), and u's distance from the one
// before: 64 ends at a time.
__device__ __forceinline__ int shared_seek(const int64_t* ends, int n, int lane, int64_t u, int64_t& rem) {
  int lo = 0;
  while (n > 64) {
    const int step = (n + 63) / 64;
    const int64_t end = ends[lo + min((lane + 1) * step, n) - 1];
    const int l = uni(__builtin_ctzll(__builtin_amdgcn_ballot_w64(end > u) | ((uint64_t)1 << 63)));
    lo += l * step;
    n = min(step, n - l * step);
  }
  const int at = lo + min(lane, n - 1);
  const int64_t end = ends[at], before = at > 0 ? ends[at - 1] : 0;
  const int l = uni(__builtin_ctzll(__builtin_amdgcn_ballot_w64(end > u) | ((uint64_t)1 << 63)));
  rem = u - lane64(before, l);
  return lo + min(l, n - 1);
}

// The units of a run, to begin with: as few as the runs that there are can do of A units and B
// steps in chunks.  A unit is a step or a tile's start's share.  A run starts somewhere, in a
// chunk or inside a tile, and pays for it once; tiles that it goes on to are counted, so that a run takes
// as long as a chunk of as many steps.  (What does not fit then takes a little more.)
__device__ __forceinline__ int64_t shared_per(SArg S, int64_t A, int64_t B) {
  return max(div64(A + B + S->p.waves - 1, S->p.waves), (int64_t)S->p.min_steps);
}

// How many of `rows` rows, that n sequences with tokens in all share, are worth it.  Sharing saves
// reading their K, V and R_k n - 1 times and costs every token and head a second part, written
// and read in fp32, which is worth it from `worth` elements for each of it on.
__device__ __forceinline__ int shared_worth(SArg S, int rows, int n, int tokens) {
  KArg P = &S->p;
  rows = n > 1 && rows > 0 ? rows & ~31 : 0;
  const float saved = (float)(n - 1) * (float)rows * (float)(2 * P->H_KV * P->D + P->H_G * P->R);
  return saved >= S->worth * (float)tokens * (float)(P->H * P->D) ? rows : 0;
}

// Sum of x over the threads before this one, and over all (total), in one workgroup.
template <int NT>
__device__ __forceinline__ int64_t plan_scan(int64_t x, int64_t* sums, int64_t& total) {
  const int lane = threadIdx.x & 63, wv = uni(threadIdx.x >> 6);
  const int64_t end = lane_scan64(x);
  __syncthreads();  // (the last scan's sums have been read)
  if (lane == 63) sums[wv] = end;
  __syncthreads();
  int64_t before = end - x;
  total = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wv) before += sums[w];
    total += sums[w];
  }
  return before;
}

// The plan, made by one workgroup of NT threads.  A wave per group: the rows that it
// shares.  Then all threads: what is left of each sequence (of one group at most, whatever
// cu_groups holds), the units of all tiles, what a run takes of them, the
// groups' full chunks, and the units that are left, added up.  (R: in LDS or in memory.)
template <int NT>
__device__ __forceinline__ void shared_plan(SArg S, const SharedPlanRef R, int64_t* sums) {
  KArg P = &S->p;
  const int lane = threadIdx.x & 63, wv = uni(threadIdx.x >> 6), tid = threadIdx.x;
  const int N = P->N, G = S->G, V = S->V;
  SharedSeq* const seqs = R.seqs;
  SharedGroup* const groups = R.groups;
  for (int b = tid; b < N; b += NT)
    seqs[G + b] = SharedSeq{paged_seq(P, b), 0, b, kSharedAlone, 0};
  __threadfence_block();
  __syncthreads();
  for (int g = wv; g < G; g += NT / 64) {
    const int c0 = min(max(uni(S->cu_groups[g]), 0), N);
    const int c1 = min(max(uni(S->cu_groups[g + 1]), c0), N);
    // the least number of rows before a chunk, the sequences that have one, and the first of them
    int least = 0x7fffffff, first = c1, n = 0;
    for (int b = c0 + lane; b < c1; b += 64) {
      const PagedSeq s = seqs[G + b].s;
      if (s.lq <= 0) continue;
      least = min(least, s.off);
      first = min(first, b);
      ++n;
    }
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) {
      least = min(least, __shfl_xor(least, k));
      first = min(first, __shfl_xor(first, k));
      n += __shfl_xor(n, k);
    }
    SharedGroup x{};
    int rows = 0;
    if (n > 1) {
      x.s.q0 = seqs[G + c0].s.q0;
      const PagedSeq last = seqs[G + c1 - 1].s;
      x.s.lq = max(last.q0 + last.lq - x.s.q0, 0);
      rows = shared_worth(S, min(least, uni(S->shared_rows[g])), n, x.s.lq);
    }
    if (rows > 0) {
      x.s.lk = x.s.off = rows;
      x.table = first;
      x.tiles = cdiv(x.s.lq, TilePlan::tokens(P));
    }
    if (rows <= 0) x = SharedGroup{};
    if (lane == 0) groups[g] = x;
  }
  __threadfence_block();
  __syncthreads();
  for (int b = tid; b < N && G > 0; b += NT) {
    SharedSeq y = seqs[G + b];
    if (y.s.lq <= 0 || S->cu_groups[0] > b || S->cu_groups[G] <= b) continue;
    int lo = 0, hi = G;  // cu_groups[lo] <= b < cu_groups[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (S->cu_groups[mid] <= b) lo = mid;
      else hi = mid;
    }
    const int rows = groups[lo].s.lk;
    if (rows <= 0) continue;
    y.s.lk = max(y.s.lk - rows, 0);
    y.s.off -= rows;
    y.row0 = rows;
    y.kind = kSharedOwn;
    y.group = lo;
    seqs[G + b] = y;
  }
  __threadfence_block();
  __syncthreads();
  int64_t own = 0, steps = 0, starts = 0, sum;
  for (int v0 = 0; v0 < N; v0 += NT) {
    const int v = v0 + tid;
    plan_scan<NT>(v < N ? SharedUnits::units(S, seqs[G + v].s) : 0, sums, sum);
    own += sum;
  }
  const int64_t blocks = TilePlan::blocks(P), start = S->start;
  for (int g0 = 0; g0 < G; g0 += NT) {
    const int g = g0 + tid;
    const int64_t tiles = g < G ? groups[g].tiles * blocks : 0;
    plan_scan<NT>(g < G ? tiles * (groups[g].s.lk / 32) : 0, sums, sum);
    steps += sum;
    plan_scan<NT>(tiles * start, sums, sum);
    starts += sum;
  }
  int64_t per = shared_per(S, own + starts, steps);
  while (true) {
    int64_t runs = 0, units = own;
    for (int g0 = 0; g0 < G; g0 += NT) {
      const int g = g0 + tid;
      const int64_t n = g < G ? groups[g].s.lk / 32 : 0, tiles = g < G ? groups[g].tiles * blocks : 0;
      const int64_t full = div64(n, per), left = n - full * per;
      plan_scan<NT>(full * tiles, sums, sum);
      runs += sum;
      plan_scan<NT>(left > 0 ? (left + start) * tiles : 0, sums, sum);
      units += sum;
    }
    if (runs + div64(units + per - 1, per) <= P->waves) break;
    per += 1 + per / 32;
  }
  int64_t runs = 0;
  for (int g0 = 0; g0 < G; g0 += NT) {
    const int g = g0 + tid;
    SharedGroup x{};
    if (g < G) x = groups[g];
    x.full = div64(x.s.lk / 32, per);
    const int64_t mine = x.full * x.tiles * blocks;
    x.run0 = runs + plan_scan<NT>(mine, sums, sum);
    x.end = x.run0 + mine;
    runs += sum;
    if (g >= G) continue;
    groups[g] = x;
    R.group_ends[g] = x.end;
    SharedSeq y{x.s, (int)(x.full * per * 32), x.table, kSharedPrefix, g};
    y.s.lk = y.s.off = x.s.lk - y.row0;
    if (y.s.lk <= 0) y.s.lq = 0;
    seqs[g] = y;
  }
  __threadfence_block();
  __syncthreads();
  int64_t before = 0;
  for (int v0 = 0; v0 < V; v0 += NT) {
    const int v = v0 + tid;
    const int64_t mine = v < V ? SharedUnits::units(S, seqs[v].s) : 0;
    const int64_t end = before + plan_scan<NT>(mine, sums, sum) + mine;
    if (v < V) R.ends[v] = end;
    before += sum;
  }
  if (tid == 0) *R.meta = SharedMeta{per, runs, before};
}

// Smallest of the wave's values, in moves between lanes' registers.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_min(int x) {
  return min(x, __builtin_amdgcn_update_dpp(0x7fffffff, x, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ int wave_min(int x) {
  x = dpp_min<0x111, 0xf>(x);  // as lane_scan64
  x = dpp_min<0x112, 0xf>(x);
  x = dpp_min<0x114, 0xf>(x);
  x = dpp_min<0x118, 0xf>(x);
  x = dpp_min<0x142, 0xa>(x);
  x = dpp_min<0x143, 0xc>(x);
  return __builtin_amdgcn_readlane(x, 63);
}

// The same by one wave, for at most 64 sequences and 64 groups: lane i has
// sequence i and group i in registers.  (1.3 us; the other form, in LDS by four waves, 5.)
__device__ __forceinline__ void shared_plan_small(SArg S, SharedSmallPlan& R, int lane) {
  KArg P = &S->p;
  const int N = P->N, G = S->G;
  PagedSeq s{0, 0, 0, 0};
  int c0 = N, c1 = N, said = 0;
  if (lane < N) s = paged_seq(P, lane);
  if (lane < G) {
    c0 = S->cu_groups[lane], c1 = S->cu_groups[lane + 1];
    said = S->shared_rows[lane];
  }
  c0 = min(max(c0, 0), N);
  c1 = min(max(c1, c0), N);
  int row0 = 0, group = -1;           // of the lane's sequence
  int rows = 0, q0 = 0, lq = 0, first = 0;  // of the lane's group
  const uint64_t have = __builtin_amdgcn_ballot_w64(s.lq > 0);
  // (groups of two sequences with tokens and more, and rows to share)
  const uint64_t below1 = c1 >= 64 ? ~(uint64_t)0 : ((uint64_t)1 << c1) - 1;
  const uint64_t below0 = c0 >= 64 ? ~(uint64_t)0 : ((uint64_t)1 << c0) - 1;
  const uint64_t members = have & below1 & ~below0;
  uint64_t todo = __builtin_amdgcn_ballot_w64(said > 0 && __builtin_popcountll(members) > 1);
  while (todo) {
    const int g = uni(__builtin_ctzll(todo));
    todo &= todo - 1;
    const uint64_t m = (uint64_t)lane64((int64_t)members, g);
    const bool in = (m >> lane) & 1;
    const int b0 = __builtin_amdgcn_readlane(c0, g), b1 = __builtin_amdgcn_readlane(c1, g) - 1;
    const int t0 = __builtin_amdgcn_readlane(s.q0, b0);
    const int t1 = __builtin_amdgcn_readlane(s.q0, b1) + __builtin_amdgcn_readlane(s.lq, b1);
    const int least = min(wave_min(in ? s.off : 0x7fffffff), __builtin_amdgcn_readlane(said, g));
    const int n = shared_worth(S, least, __builtin_popcountll(m), max(t1 - t0, 0));
    if (n <= 0) continue;
    if (lane == g) rows = n, q0 = t0, lq = max(t1 - t0, 0), first = __builtin_ctzll(m);
    if (in) row0 = n, group = g;
  }
  if (row0 > 0) s.lk = max(s.lk - row0, 0), s.off -= row0;
  const int64_t blocks = TilePlan::blocks(P), start = S->start;
  const int64_t mine = lane < N ? SharedUnits::units(S, s) : 0;
  const int64_t own_end = lane_scan64(mine), own = lane64(own_end, 63);
  const int tiles1 = rows > 0 ? cdiv(lq, TilePlan::tokens(P)) : 0, n = rows / 32;
  const int64_t tiles = tiles1 * blocks;
  int64_t per = own, full = 0, runs = 0, run_end = 0, rest = 0, rest_end = 0, rests = 0;
  const bool any = __builtin_amdgcn_ballot_w64(rows > 0) != 0;
  per = any ? shared_per(S, own + lane64(lane_scan64(tiles * start), 63), lane64(lane_scan64(tiles * n), 63))
            : shared_per(S, own, 0);
  while (any) {
    full = div64(n, per);
    const int64_t left = n - full * per;
    run_end = lane_scan64(full * tiles);
    runs = lane64(run_end, 63);
    rest = left > 0 ? (left + start) * tiles : 0;
    rest_end = lane_scan64(rest);
    rests = lane64(rest_end, 63);
    if (runs + div64(rests + own + per - 1, per) <= P->waves) break;
    per += 1 + per / 32;
  }
  if (lane < G) {
    R.groups[lane] = SharedGroup{PagedSeq{q0, lq, rows, rows}, run_end - full * tiles, run_end, first, tiles1, full};
    R.group_ends[lane] = run_end;
    const int at = (int)(full * per * 32), lk = rows - at;
    R.seqs[lane] = SharedSeq{PagedSeq{q0, lk > 0 ? lq : 0, lk, lk}, at, first, kSharedPrefix, lane};
    R.ends[lane] = rest_end;
  }
  if (lane < N) {
    R.seqs[G + lane] = SharedSeq{s, row0, lane, row0 > 0 ? kSharedOwn : kSharedAlone, group};
    R.ends[G + lane] = rests + own_end;
  }
  if (lane == 0) R.meta = SharedMeta{per, runs, rests + own};
}

// Sums of K values over the threads up to and including this one, and over all, of NW waves.
template <int K>
__device__ __forceinline__ void plan_scans(int64_t (&x)[K], int64_t (&total)[K], int64_t (*sums)[16], int nw) {
  const int lane = threadIdx.x & 63, wv = uni(threadIdx.x >> 6);
#pragma unroll
  for (int k = 0; k < K; ++k) x[k] = lane_scan64(x[k]);
  __syncthreads();  // (the last scan's sums have been read)
  if (lane == 63) {
#pragma unroll
    for (int k = 0; k < K; ++k) sums[k][wv] = x[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) total[k] = 0;
  for (int w = 0; w < nw; ++w) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t v = sums[k][w];
      if (w < wv) x[k] += v;
      total[k] += v;
    }
  }
}

// The same by one workgroup for at most 1024 sequences and 1024 groups: thread i has sequence i
// and group i in registers.
constexpr int kSharedMid = 1024;
struct SharedMidPlan {
  int cu[kSharedMid + 1], least[kSharedMid], first[kSharedMid], n[kSharedMid], rows[kSharedMid];
  int q0[kSharedMid], lq[kSharedMid];
  int64_t sums[3][16];
};
__device__ __forceinline__ void shared_plan_mid(SArg S, const SharedPlanRef R, SharedMidPlan& L) {
  KArg P = &S->p;
  const int tid = threadIdx.x, nw = blockDim.x >> 6, N = P->N, G = S->G;
  PagedSeq s{0, 0, 0, 0};
  int c0 = N, said = 0;
  if (tid < N) s = paged_seq(P, tid);
  if (tid <= G) c0 = min(max(S->cu_groups[tid], 0), N);
  if (tid < G) said = S->shared_rows[tid];
  if (tid <= G) L.cu[tid] = c0;
  if (tid == 0 && G >= (int)blockDim.x) L.cu[G] = min(max(S->cu_groups[G], 0), N);
  L.least[tid] = L.first[tid] = 0x7fffffff, L.n[tid] = 0;
  L.q0[tid] = s.q0, L.lq[tid] = s.lq;
  __syncthreads();
  int g = -1;
  if (s.lq > 0 && G > 0 && L.cu[0] <= tid && tid < L.cu[G]) {
    int lo = 0, hi = G;  // cu[lo] <= tid < cu[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (L.cu[mid] <= tid) lo = mid;
      else hi = mid;
    }
    g = lo;
    atomicMin(&L.least[g], s.off);
    atomicMin(&L.first[g], tid);
    atomicAdd(&L.n[g], 1);
  }
  __syncthreads();
  int rows = 0, q0 = 0, lq = 0, first = 0;
  if (tid < G && L.n[tid] > 1) {
    const int b0 = L.cu[tid], b1 = max(L.cu[tid + 1] - 1, b0);
    q0 = L.q0[b0];
    lq = max(L.q0[b1] + L.lq[b1] - q0, 0);
    first = L.first[tid];
    rows = shared_worth(S, min(L.least[tid], said), L.n[tid], lq);
  }
  L.rows[tid] = rows;
  __syncthreads();
  const int row0 = g >= 0 ? L.rows[g] : 0;
  if (row0 > 0) s.lk = max(s.lk - row0, 0), s.off -= row0;
  const int64_t blocks = TilePlan::blocks(P), start = S->start;
  const int tiles1 = rows > 0 ? cdiv(lq, TilePlan::tokens(P)) : 0, n = rows / 32;
  const int64_t tiles = tiles1 * blocks, mine = tid < N ? SharedUnits::units(S, s) : 0;
  int64_t sum[3], total[3], own, own_end;
  {
    int64_t x[3] = {mine, tiles * n, tiles * start};
    plan_scans<3>(x, total, L.sums, nw);
    own = total[0], own_end = x[0];
  }
  int64_t per = shared_per(S, own + total[2], total[1]), full, end[2];
  while (true) {
    full = div64(n, per);
    const int64_t left = n - full * per;
    int64_t x[2] = {full * tiles, left > 0 ? (left + start) * tiles : 0}, t[2];
    plan_scans<2>(x, t, L.sums, nw);
    end[0] = x[0], end[1] = x[1], sum[0] = t[0], sum[1] = t[1];
    if (sum[0] + div64(sum[1] + own + per - 1, per) <= P->waves) break;
    per += 1 + per / 32;
  }
  if (tid < G) {
    R.groups[tid] = SharedGroup{PagedSeq{q0, lq, rows, rows}, end[0] - full * tiles, end[0], first, tiles1, full};
    R.group_ends[tid] = end[0];
    const int at = (int)(full * per * 32), lk = rows - at;
    R.seqs[tid] = SharedSeq{PagedSeq{q0, lk > 0 ? lq : 0, lk, lk}, at, first, kSharedPrefix, tid};
    R.ends[tid] = end[1];
  }
  if (tid < N) {
    R.seqs[G + tid] = SharedSeq{s, row0, tid, row0 > 0 ? kSharedOwn : kSharedAlone, g};
    R.ends[G + tid] = sum[1] + own_end;
  }
  if (tid == 0) *R.meta = SharedMeta{per, sum[0], sum[1] + own};
}

// Kernel launches (fna2_paged_shared.hip): the plan, the tiles, the join.
hipError_t launch_paged_shared(const PagedSharedParams& P, int rpl, hipStream_t s);

}  // namespace fna2
