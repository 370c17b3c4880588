// fna2_paged_books.hip — the books of a paged cache on the GPU: which pages hold
// the rows of which sequence, and who shares them.
//
// Integers only, and all results fixed by the inputs: the pages of a step go to
// the sequences in their order, from the top of a stack of free ones.
//
// Bound by latency: a launch and a few dependent loads.  Extend 5.6 us for 256 sequences of a token,
// 5.9 for 64 of up to 2048; groups 3.5 + 2.2 for 512 rows of 256 entries.
#include <algorithm>

#include "fna2_paged_books.h"

namespace fna2 {

namespace {

constexpr int kBooksThreads = 256, kBooksWaves = kBooksThreads / 64;
constexpr int kBooksChunk = 1024;  // sequences whose sums are formed at once
constexpr int kBooksEach = kBooksChunk / kBooksThreads;
constexpr int kBooksMax = 1 << 30;  // rows of a sequence, tokens of a step

// ceil(rows / ps), or one more than the table has room for.
__device__ __forceinline__ int books_pages(const BooksParams& P, int64_t rows) {
  if (rows <= 0) return 0;
  if (rows > (int64_t)P.width * P.ps) return P.width + 1;
  return page_of(P.ps_mul, P.ps_shift, (int)rows - 1) + 1;
}

// A workgroup's sums over a chunk of sequences, thread by thread four of them in order:
// a and b become the sums of all before.
struct BooksScan {
  int64_t (*sums)[kBooksWaves];
  int64_t total[2];
  __device__ __forceinline__ void run(int64_t (&a)[kBooksEach], int64_t (&b)[kBooksEach]) {
    const int lane = threadIdx.x & 63, wv = uni(threadIdx.x >> 6);
    int64_t sa = 0, sb = 0;
#pragma unroll
    for (int i = 0; i < kBooksEach; ++i) {
      const int64_t x = a[i], y = b[i];
      a[i] = sa, b[i] = sb;
      sa += x, sb += y;
    }
    const int64_t ea = lane_scan64(sa), eb = lane_scan64(sb);
    __syncthreads();  // (the last run's sums have been read)
    if (lane == 63) sums[0][wv] = ea, sums[1][wv] = eb;
    __syncthreads();
    int64_t ba = ea - sa, bb = eb - sb;
    total[0] = total[1] = 0;
#pragma unroll
    for (int w = 0; w < kBooksWaves; ++w) {
      if (w < wv) ba += sums[0][w], bb += sums[1][w];
      total[0] += sums[0][w], total[1] += sums[1][w];
    }
#pragma unroll
    for (int i = 0; i < kBooksEach; ++i) a[i] += ba, b[i] += bb;
  }
};

// The last of n (>= 1) ascending numbers that is <= x; the first is.
__device__ __forceinline__ int books_find(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// ── Extend ────────────────────────────────────────────────────────────────────
// With have = ceil(len / ps) and more = ceil((len + c) / ps) - have, the k-th new
// page over all sequences is free[F - 1 - k], and token t of sequence b sits at
// row len_b + t - cu_b.  Every workgroup forms the sums of all sequences for
// itself (they are few, and one launch is what a step waits for) and then takes
// its share of the new pages and of the tokens, whose sequence it finds by
// halving the sums in LDS.  No workgroup reads what another writes: a token's page
// comes from the table if it is old, from the stack if it is new.
__global__ __launch_bounds__(kBooksThreads) void paged_extend_kernel(const BooksParams P) {
  __shared__ int64_t sums[2][kBooksWaves];
  __shared__ int cu[kBooksChunk], first[kBooksChunk], len[kBooksChunk];
  __shared__ int wrong;
  BooksScan scan{sums};
  const int tid = threadIdx.x, F = min(max(*P.nfree, 0), P.cap);
  const int nchunks = max((P.N + kBooksChunk - 1) / kBooksChunk, 1);
  if (tid == 0) wrong = 0;
  __syncthreads();
  int64_t a[kBooksEach], b[kBooksEach];
  int l[kBooksEach], c[kBooksEach];
  auto load = [&](int c0) {
    bool wide = false;
#pragma unroll
    for (int i = 0; i < kBooksEach; ++i) {
      const int s = c0 + kBooksEach * tid + i;
      l[i] = c[i] = 0;
      a[i] = b[i] = 0;
      if (s >= P.N) continue;
      l[i] = min(max(P.lens[s], 0), kBooksMax);
      c[i] = min(max(P.counts[s], 0), kBooksMax);
      const int need = books_pages(P, (int64_t)l[i] + c[i]);
      wide |= c[i] > 0 && need > P.width;
      a[i] = c[i];
      b[i] = need - books_pages(P, l[i]);
    }
    if (wide) wrong = 1;
    scan.run(a, b);
  };
  int64_t tokens = 0, pages = 0;
  for (int k = 0; k < nchunks; ++k) {
    load(k * kBooksChunk);
    tokens += scan.total[0], pages += scan.total[1];
  }
  const int bad = wrong ? -1 : tokens > P.T ? -2 : pages > F ? (int)min(pages - F, (int64_t)kBooksMax) : 0;
  if (blockIdx.x == 0 && tid == 0) {
    *P.status = bad;
    *P.new_nfree = bad ? F : F - (int)pages;
    if (P.N == 0) P.cu[0] = 0;
  }
  const int step = gridDim.x * kBooksThreads, me = blockIdx.x * kBooksThreads + tid;
  int64_t t0 = 0, p0 = 0;  // tokens and new pages of the chunks before
  for (int k = 0; k < nchunks && P.N > 0; ++k) {
    const int c0 = k * kBooksChunk, n = min(P.N - c0, kBooksChunk);
    if (nchunks > 1) load(c0);
#pragma unroll
    for (int i = 0; i < kBooksEach; ++i) {
      const int s = kBooksEach * tid + i;
      if (s >= n) continue;
      if (blockIdx.x == 0) {
        P.cu[c0 + s] = bad ? 0 : (int)(t0 + a[i]);
        P.new_lens[c0 + s] = bad ? P.lens[c0 + s] : l[i] + c[i];
        if (c0 + s == P.N - 1) P.cu[P.N] = bad ? 0 : (int)tokens;
      }
      cu[s] = (int)a[i], first[s] = (int)b[i], len[s] = l[i];
    }
    if (bad) continue;
    __syncthreads();
    const int nt = (int)scan.total[0], np = (int)scan.total[1];
    for (int j = me; j < np; j += step) {
      const int s = books_find(first, n, j);
      const int64_t at = books_pages(P, len[s]) + (j - first[s]);
      P.table[(int64_t)(c0 + s) * P.tstride + at] = P.free[F - 1 - (p0 + j)];
    }
    for (int j = me; j < nt; j += step) {
      const int s = books_find(cu, n, j);
      const int row = len[s] + (j - cu[s]), pg = page_of(P.ps_mul, P.ps_shift, row);
      const int have = books_pages(P, len[s]);
      const int id = pg < have ? P.table[(int64_t)(c0 + s) * P.tstride + pg]
                               : P.free[F - 1 - (p0 + first[s] + (pg - have))];
      const int64_t t = t0 + j;
      P.slots[t] = id < 0 ? -1 : (int64_t)id * P.ps + (row - pg * P.ps);
      P.seq[t] = c0 + s;
      P.pos[t] = row + (P.shift ? P.shift[c0 + s] : 0);
    }
    t0 += nt, p0 += np;
    __syncthreads();  // (the sums in LDS have been read)
  }
  for (int64_t t = (bad ? 0 : tokens) + me; t < P.T; t += step) {
    P.slots[t] = -1;
    P.seq[t] = -1;
    P.pos[t] = 0;
  }
}

// ── Trim ──────────────────────────────────────────────────────────────────────
// len -> min(len, keep); the entries behind the pages that still hold rows become -1
// and, but for borrowed ones, go onto the stack, sequence by sequence, each one's last page
// first.  One workgroup: a few sequences end or shrink in a step.
__global__ __launch_bounds__(kBooksThreads) void paged_trim_kernel(const BooksParams P) {
  __shared__ int64_t sums[2][kBooksWaves];
  __shared__ int first[kBooksChunk], gone[kBooksChunk], keep[kBooksChunk], have[kBooksChunk];
  BooksScan scan{sums};
  const int tid = threadIdx.x, F = min(max(*P.nfree, 0), P.cap);
  int64_t back = 0;  // pages given back by the chunks before
  for (int c0 = 0; c0 < P.N; c0 += kBooksChunk) {
    const int n = min(P.N - c0, kBooksChunk);
    int64_t a[kBooksEach], b[kBooksEach];
    int h[kBooksEach], k[kBooksEach];
#pragma unroll
    for (int i = 0; i < kBooksEach; ++i) {
      const int s = c0 + kBooksEach * tid + i;
      h[i] = k[i] = 0;
      a[i] = b[i] = 0;
      if (s >= P.N) continue;
      const int len = P.lens[s], rows = min(max(len, 0), kBooksMax);
      const int kept = min(rows, max(P.counts[s], 0));
      h[i] = min(books_pages(P, rows), P.width);
      k[i] = min(books_pages(P, kept), h[i]);
      const int lent = P.borrowed ? min(max(P.borrowed[s], 0), h[i]) : 0;
      a[i] = h[i] - k[i];             // entries that are cleared
      b[i] = h[i] - max(k[i], lent);  // ... and given back, the last ones
      P.new_lens[s] = kept < rows ? kept : len;
    }
    scan.run(a, b);
#pragma unroll
    for (int i = 0; i < kBooksEach; ++i) {
      const int s = kBooksEach * tid + i;
      if (s < n) first[s] = (int)min(a[i], (int64_t)kBooksMax), gone[s] = (int)min(b[i], (int64_t)kBooksMax), keep[s] = k[i], have[s] = h[i];
    }
    __syncthreads();
    const int total = (int)min(scan.total[0], (int64_t)kBooksMax);
    const int64_t given = scan.total[1];
    for (int j = tid; j < total; j += kBooksThreads) {
      const int s = books_find(first, n, j);
      // the j-th cleared entry, the sequence's last page first
      const int e = j - first[s], at = have[s] - 1 - e;
      const int mine = (int)((s + 1 < n ? (int64_t)gone[s + 1] : min(given, (int64_t)kBooksMax)) - gone[s]);
      int* entry = P.table + (int64_t)(c0 + s) * P.tstride + at;
      const int64_t to = F + back + gone[s] + e;
      if (e < mine && to < P.cap) P.free[to] = *entry;
      *entry = -1;
    }
    back += given;
    __syncthreads();
  }
  if (tid == 0) *P.new_nfree = (int)min(F + back, (int64_t)P.cap);
}

// ── Groups ────────────────────────────────────────────────────────────────────
// common[b]: the leading entries that rows b - 1 and b of the table have alike (0 for b = 0).  A
// run of neighbours with at least one is a group, and shares as many as all of its
// pairs do.  A wave a pair, 64 entries a step; then one workgroup for the runs.
__global__ __launch_bounds__(256) void paged_common_kernel(const BooksParams P) {
  const int lane = threadIdx.x & 63, b = blockIdx.x * 4 + uni(threadIdx.x >> 6);
  if (b >= P.N) return;
  int n = 0;
  if (b > 0) {
    const int* x = P.table + (int64_t)b * P.tstride;
    const int* y = x - P.tstride;
    for (; n < P.width; n += 64) {
      const int j = n + lane;
      const int id = j < P.width ? x[j] : -1;
      const uint64_t apart = __builtin_amdgcn_ballot_w64(id < 0 || id != y[min(j, P.width - 1)]);
      if (apart) {
        n += __builtin_ctzll(apart);
        break;
      }
    }
  }
  if (lane == 0) P.common[b] = n;
}

__global__ __launch_bounds__(kBooksThreads) void paged_groups_kernel(const BooksParams P) {
  __shared__ int64_t sums[2][kBooksWaves];
  __shared__ int least[kBooksChunk + 1];
  BooksScan scan{sums};
  const int tid = threadIdx.x, N = P.N;
  int before = 0;      // groups that begin in the chunks before
  int open = kBooksMax;  // the last of them: the least of its pairs so far
  for (int c0 = 0; c0 < N; c0 += kBooksChunk) {
    int64_t a[kBooksEach], b[kBooksEach];
    int c[kBooksEach];
#pragma unroll
    for (int i = 0; i < kBooksEach; ++i) {
      const int s = c0 + kBooksEach * tid + i;
      c[i] = s < N ? P.common[s] : -1;
      a[i] = c[i] == 0;
      b[i] = 0;
      least[kBooksEach * tid + i + 1] = kBooksMax;
    }
    if (tid == 0) least[0] = open;
    scan.run(a, b);
#pragma unroll
    for (int i = 0; i < kBooksEach; ++i) {
      const int s = c0 + kBooksEach * tid + i;
      if (c[i] == 0) P.cu_groups[before + (int)a[i]] = s;
      else if (c[i] > 0) atomicMin(least + (int)a[i], c[i]);  // (the group that is open here)
    }
    const int n = (int)scan.total[0];
    __syncthreads();
    // groups before - 1 .. before + n - 2 are closed; the next goes on
    for (int g = tid; g < n; g += kBooksThreads)
      if (before + g > 0) P.shared_rows[before + g - 1] = least[g] == kBooksMax ? 0 : least[g] * P.ps;
    open = least[n];
    before += n;
    __syncthreads();
  }
  if (tid == 0 && before > 0) P.shared_rows[before - 1] = open == kBooksMax ? 0 : open * P.ps;
  for (int g = before + tid; g <= N; g += kBooksThreads) {
    P.cu_groups[g] = N;
    if (g < N) P.shared_rows[g] = 0;
  }
}

}  // namespace

hipError_t launch_paged_extend(const BooksParams& P, hipStream_t s) {
  const int grid = std::min(std::max((P.T + kBooksThreads - 1) / kBooksThreads, 1), 512);
  hipLaunchKernelGGL(paged_extend_kernel, dim3(grid), dim3(kBooksThreads), 0, s, P);
  return hipGetLastError();
}

hipError_t launch_paged_trim(const BooksParams& P, hipStream_t s) {
  hipLaunchKernelGGL(paged_trim_kernel, dim3(1), dim3(kBooksThreads), 0, s, P);
  return hipGetLastError();
}

hipError_t launch_paged_groups(const BooksParams& P, hipStream_t s) {
  if (P.N > 0) {
    hipLaunchKernelGGL(paged_common_kernel, dim3((P.N + 3) / 4), dim3(256), 0, s, P);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(paged_groups_kernel, dim3(1), dim3(kBooksThreads), 0, s, P);
  return hipGetLastError();
}

}  // namespace fna2
