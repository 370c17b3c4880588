// fna2_paged_rows.hip — the rows of a paged cache: writing a chunk's new rows
// (with QK-RMSNorm and rotation on the way), and eviction.
#include <algorithm>

#include "fna2_kernels.h"
#include "fna2_paged.h"

namespace fna2 {

namespace {

// ── Append ─────────────────────────────────────────────────────────────────
// Token t at position p: x <- x rsqrt(mean(x^2) + eps) w, then for i < D / 2
//     y_i       = x_i cos(a_i) - x_{i+D/2} sin(a_i),   a_i = p inv_freq[i],
//     y_{i+D/2} = x_{i+D/2} cos(a_i) + x_i sin(a_i),
// in fp32 with one rounding at the store.  The angle is formed and reduced in
// fp64: in fp32 it is off by half a unit in its last place, 1e-3 radians at
// position 20,000, as much as a bf16 result's rounding and more than an fp16 one's.
// A wave forms the token's cos and sin once, then walks the token's rows, LPR =
// D / 16 lanes a row, each with 8 values of the first half and the matching 8 of the
// second, two passes of rows in flight.  Many tokens: one to a wave, bound by reading
// and writing every row once (4 chunks of 2048 tokens, 32 heads over 8 KV heads
// of 128, 32 of R_k's 32: 42.5 us, 4.6 TB/s).  Few tokens: the four waves of a
// workgroup share each, which shortens the chain that bounds them, sequence, page,
// rows (64 tokens, 16 heads over 16: 6.6 us).
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));  // (norm weights anywhere)
constexpr int kAppWaves = 4, kAppAhead = 2;
template <int D, bool F16>
__global__ __launch_bounds__(64 * kAppWaves) void paged_append_kernel(const PagedAppendParams A) {
  constexpr int LPR = D / 16, HALF = D / 2, RPP = 64 / LPR;  // rows a pass of a wave
  const PagedParams& P = A.p;
  __shared__ float table[kAppWaves][2 * HALF];
  const int lane = threadIdx.x & 63, wv = uni(threadIdx.x >> 6);
  float* cs = table[wv];
  const int i = lane % LPR, lrow = lane / LPR, col = 8 * i;
  const auto cu = const_space(P.cu);
  const int nv = P.H + P.H_KV, nr = nv + P.H_KV;  // q and k rows; and v rows
  const int share = A.share;                      // waves of a token
  const int sub = wv % share;
  const double inv = A.inv_freq && lane < HALF ? (double)A.inv_freq[lane] : 0.0;
  const int step = gridDim.x * (kAppWaves / share);

  for (int t = blockIdx.x * (kAppWaves / share) + wv / share; t < P.T; t += step) {
    // the token's sequence: the last b with cu[b] <= t
    int lo = -1, hi = P.N;
    if (uni(cu[P.N]) <= t) lo = P.N;
    else
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (uni(cu[mid]) <= t) lo = mid;
        else hi = mid;
      }
    const bool inside = lo >= 0 && lo < P.N;
    int row = -1, pr = 0, shift = 0;
    int64_t page = -1;
    if (inside) {
      const PagedSeq e = paged_seq_uniform(kargs(), lo);
      // (a sequence past its table: its tokens keep their rows, and those that
      // the table does not have are not stored)
      row = max(uni(*const_space(P.lens + lo)), 0) - e.lq + (t - e.q0);
      if (A.shift) shift = uni(*const_space(A.shift + lo));
      if (row >= 0 && row < e.lk) {
        const int pg = page_of(P.ps_mul, P.ps_shift, row);
        pr = row - pg * P.ps;
        const int id = uni(*const_space(P.table + (int64_t)lo * P.tstride + pg));
        if ((uint32_t)id < (uint32_t)P.npages) page = id;
      }
    }
    // Source and destination of row r of the token (q, k, then v rows).
    u32x4 a[kAppAhead], b[kAppAhead];
    uint16_t* dst[kAppAhead];
    auto load = [&](int r0) {
#pragma unroll
      for (int p = 0; p < kAppAhead; ++p) {
        const int r = r0 + p * RPP * share + lrow;
        const bool isq = r < P.H, isk = !isq && r < nv;
        const int h = isq ? r : isk ? r - P.H : r - nv;
        dst[p] = nullptr;
        a[p] = b[p] = u32x4{0, 0, 0, 0};
        if (r >= nr) continue;
        const uint16_t* src;
        if (isq) {
          src = (const uint16_t*)P.q.ptr + (int64_t)t * P.q.ss + (int64_t)h * P.q.sh;
          dst[p] = (uint16_t*)P.o.ptr + (int64_t)t * P.o.ss + (int64_t)h * P.o.sh;
        } else {
          const TView& n = isk ? A.kn : A.vn;
          const TView& d = isk ? P.k : P.v;
          src = (const uint16_t*)n.ptr + (int64_t)t * n.ss + (int64_t)h * n.sh;
          if (page >= 0) dst[p] = (uint16_t*)d.ptr + page * d.sb + (int64_t)h * d.sh + (int64_t)pr * d.ss;
        }
        if (dst[p]) {
          a[p] = ld16(src + col);
          b[p] = ld16(src + HALF + col);
        }
      }
    };
    load(sub * RPP);
    const bool turn = inside && A.inv_freq;
    float co[8], si[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) co[e] = 1.f, si[e] = 0.f;
    if (turn) {
      const int64_t pos = (int64_t)(A.pos ? uni(*const_space(A.pos + t)) : row) + shift;
      if (lane < HALF) {
        // in turns, reduced to half a turn either way
        const double x = (double)pos * inv * 0.15915494309189533577;
        const float ang = (float)((x - __builtin_rint(x)) * 6.28318530717958647693);
        float s, c;
        sincosf(ang, &s, &c);
        cs[lane] = c;
        cs[HALF + lane] = s;
      }
      // (one wave's own LDS: its reads follow its writes in order)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int e = 0; e < 8; ++e) co[e] = cs[col + e], si[e] = cs[HALF + col + e];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    for (int r0 = sub * RPP; r0 < nr; r0 += kAppAhead * RPP * share) {
#pragma unroll
      for (int p = 0; p < kAppAhead; ++p) {
        const int r = r0 + p * RPP * share + lrow;
        const bool isq = r < P.H, isk = !isq && r < nv;
        const float* w = isq ? A.wq : A.wk;
        float x[16];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[2 * e] = elt_lo<F16>(a[p][e]), x[2 * e + 1] = elt_hi<F16>(a[p][e]);
          x[8 + 2 * e] = elt_lo<F16>(b[p][e]), x[8 + 2 * e + 1] = elt_hi<F16>(b[p][e]);
        }
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) ss += x[e] * x[e];
#pragma unroll
        for (int m = 1; m < LPR; m <<= 1) ss += __shfl_xor(ss, m);
        if (!dst[p]) continue;
        if (inside && (isq || isk) && (w || turn)) {
          if (w) {
            const float rs = rsqrtf(ss * (1.f / D) + A.eps);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const f32x4_u w1 = *(const f32x4_u*)(w + col + 4 * e);
              const f32x4_u w2 = *(const f32x4_u*)(w + HALF + col + 4 * e);
#pragma unroll
              for (int k = 0; k < 4; ++k) x[4 * e + k] *= rs * w1[k], x[8 + 4 * e + k] *= rs * w2[k];
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float y[4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float p1 = x[2 * e + k], p2 = x[8 + 2 * e + k], c = co[2 * e + k], s = si[2 * e + k];
              y[k] = turn ? p1 * c - p2 * s : p1;
              y[2 + k] = turn ? p2 * c + p1 * s : p2;
            }
            a[p][e] = pack_e<F16>(y[0], y[1]);
            b[p][e] = pack_e<F16>(y[2], y[3]);
          }
        }
        st16(dst[p] + col, a[p]);
        st16(dst[p] + HALF + col, b[p]);
      }
      if (r0 + kAppAhead * RPP * share < nr) load(r0 + kAppAhead * RPP * share);
    }
    if (P.H_G > 0 && page >= 0) {
      const int cr = P.R / 8, n = P.H_G * cr;
      for (int j = sub * 64 + lane; j < n; j += 64 * share) {
        const int h = j / cr, ch = j - h * cr;
        st16((uint16_t*)P.rk.ptr + page * P.rk.sb + (int64_t)h * P.rk.sh + (int64_t)pr * P.rk.ss + 8 * ch,
             ld16((const uint16_t*)A.rkn.ptr + (int64_t)t * A.rkn.ss + (int64_t)h * A.rkn.sh + 8 * ch));
      }
    }
  }
}

// ── Eviction ───────────────────────────────────────────────────────────────
// Selection, one workgroup per (sequence, KV head): the `top` = budget - first
// - recent rows of largest weight among rows [first, lk - recent).  Weights
// become unsigned keys in their order; three passes of 11, 11 and 10 bits find the
// top-th largest key K, and the rows kept are those above K and, of those equal
// to K, the lowest (top minus the rows above).  Two last passes write
// the kept rows in their order: every wave counts, then writes, a range of its
// own.  Bound by the latency of its passes, not by memory: a wave keeps up to
// 512 weights in registers over all of them (32 sequences of up to 8192 rows, 8 KV
// heads: 16.4 us; 2 of 1201, 4 KV heads: 8.9 us).  With 8 bits a pass the first
// digit of positive weights is their exponent's, a few bins that all lanes count in.
constexpr int kSelAhead = 8;
constexpr int kSelBins = 2048;
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);  // (-0 as 0)
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ int wave_scan(int x, int lane) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int o = __shfl_up(x, m);
    if (lane >= m) x += o;
  }
  return x;
}

// kSelThreads: 1024, or 256 where no sequence holds more rows than those keep in
// registers.
template <int kSelThreads>
__global__ __launch_bounds__(kSelThreads) void paged_select_kernel(const PagedEvictParams E) {
  constexpr int kSelWaves = kSelThreads / 64, kBins = kSelBins / kSelThreads;  // bins a thread
  const PagedParams& P = E.p;
  __shared__ int hist[kSelBins];
  __shared__ int wsum[kSelWaves];
  __shared__ int gt_of[kSelWaves], eq_of[kSelWaves];
  __shared__ int pick[2];
  const int b = blockIdx.x / P.H_KV, kvh = blockIdx.x % P.H_KV, tid = threadIdx.x;
  const int lane = tid & 63, wv = uni(tid >> 6);
  const int lk = min(max(uni(*const_space(P.lens + b)), 0), P.width * P.ps);
  const int keep = min(lk, E.budget);
  if (kvh == 0 && tid == 0) E.new_lens[b] = keep;
  const float* w = E.w + (int64_t)b * E.w_sb + (int64_t)kvh * E.w_sh;
  float* wo = E.w_out + ((int64_t)b * P.H_KV + kvh) * E.cap;
  int* kept = E.kept + ((int64_t)b * P.H_KV + kvh) * E.budget;
  const int cap = E.cap;
  for (int j = keep + tid; j < E.budget; j += kSelThreads) kept[j] = -1;
  for (int j = keep + tid; j < cap; j += kSelThreads) wo[j] = 0.f;
  if (lk <= E.budget) {
    for (int j = tid; j < keep; j += kSelThreads) {
      kept[j] = j;
      if (j < cap) wo[j] = w[j];
    }
    return;
  }
  const int lo = E.first, hi = lk - E.recent, top = E.budget - E.first - E.recent;
  // This wave's rows [j_lo, j_hi), kSelAhead x 64 at a time; up to 8192 rows
  // in all a wave's are one such chunk, loaded once.
  const int span = cdiv(cdiv(lk, kSelWaves), 64) * 64;
  const int j_lo = wv * span, j_hi = min(lk, j_lo + span);
  float x[kSelAhead];
  int loaded = -1;
  auto load = [&](int j0) {
    if (j0 == loaded) return;
    loaded = j0;
#pragma unroll
    for (int i = 0; i < kSelAhead; ++i) {
      const int j = j0 + i * 64 + lane;
      x[i] = j < j_hi && j < cap ? w[j] : 0.f;
    }
  };
  uint32_t prefix = 0, mask = 0;
  int need = top;  // rows still to find among those that match the prefix
  if (top > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digit = pass == 2 ? 1023u : 2047u;
      for (int i = tid; i < kSelBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int j0 = j_lo; j0 < j_hi; j0 += kSelAhead * 64) {
        load(j0);
#pragma unroll
        for (int i = 0; i < kSelAhead; ++i) {
          const int j = j0 + i * 64 + lane;
          const uint32_t k = weight_key(x[i]);
          if (j >= lo && j < hi && j < j_hi && (k & mask) == prefix)
            atomicAdd(&hist[(k >> shift) & digit], 1);
        }
      }
      __syncthreads();
      // The digit d whose rows, with those of larger digits, reach `need`: a
      // thread has kBins bins, from the largest digits down.
      int h[kBins], mine = 0;
#pragma unroll
      for (int i = 0; i < kBins; ++i) mine += h[i] = hist[kSelBins - 1 - kBins * tid - i];
      int s = wave_scan(mine, lane);
      if (lane == 63) wsum[wv] = s;
      __syncthreads();
      for (int i = 0; i < wv; ++i) s += wsum[i];
      int before = s - mine;
#pragma unroll
      for (int i = 0; i < kBins; ++i) {
        if (before < need && before + h[i] >= need) pick[0] = kSelBins - 1 - kBins * tid - i, pick[1] = before;
        before += h[i];
      }
      __syncthreads();
      prefix |= (uint32_t)pick[0] << shift;
      mask |= digit << shift;
      need -= pick[1];
      __syncthreads();
    }
  }
  auto sort_of = [&](int j, float v) {  // 2 kept, 1 equal to the key, 0 not
    if (j >= j_hi) return 0;
    if (j < lo || j >= hi) return 2;
    if (top <= 0) return 0;
    const uint32_t k = weight_key(v);
    return k > prefix ? 2 : k == prefix ? 1 : 0;
  };
  int n_gt = 0, n_eq = 0;
  for (int j0 = j_lo; j0 < j_hi; j0 += kSelAhead * 64) {
    load(j0);
#pragma unroll
    for (int i = 0; i < kSelAhead; ++i) {
      const int k = sort_of(j0 + i * 64 + lane, x[i]);
      n_gt += __builtin_popcountll(__builtin_amdgcn_ballot_w64(k == 2));
      n_eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(k == 1));
    }
  }
  if (lane == 0) gt_of[wv] = n_gt, eq_of[wv] = n_eq;
  __syncthreads();
  int out = 0, left = need;  // where this wave writes; equal rows still to keep
  for (int i = 0; i < wv; ++i) {
    const int q = min(eq_of[i], left);
    out += gt_of[i] + q;
    left -= q;
  }
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  for (int j0 = j_lo; j0 < j_hi; j0 += kSelAhead * 64) {
    load(j0);
#pragma unroll
    for (int i = 0; i < kSelAhead; ++i) {
      const int j = j0 + i * 64 + lane, k = sort_of(j, x[i]);
      const uint64_t eq = __builtin_amdgcn_ballot_w64(k == 1);
      const bool yes = k == 2 || (k == 1 && __builtin_popcountll(eq & below) < left);
      const uint64_t all = __builtin_amdgcn_ballot_w64(yes);
      if (yes) {
        const int at = out + __builtin_popcountll(all & below);
        kept[at] = j;
        if (at < cap) wo[at] = x[i];
      }
      out += __builtin_popcountll(all);
      left -= min(left, (int)__builtin_popcountll(eq));
    }
  }
}

// Compaction in place: row kept[r] becomes row r (kept[r] >= r, increasing).
// A workgroup takes one strip (128 bytes, or less) of the rows of one (sequence,
// head) of K, V or R_k, in rounds of some hundred rows: all of a round's loads, a
// barrier, all of its stores.  Rows stored so lie before every row that is still to
// be loaded, so no other copy is needed.  A round's chain (kept row, its page, the
// row) is as long as for a few rows, so rounds are as large as the registers allow:
// 16 waves of 4 loads of 8 rows, 64 KB in flight, and the next round's rows
// and pages are looked up while this one's are under way.  32 sequences of up to
// 8192 rows to 4096 (8 KV heads of 128, 32 of R_k's 32): 284 us, 4.1 TB/s.  Where few
// strips leave CUs without one they are narrower, and the rounds fewer (2 sequences
// of 1201 rows to 1000, 4 KV heads of 64: 10.6 us become 8.0).
constexpr int kCompactThreads = 1024, kCompactAhead = 4;
__global__ __launch_bounds__(kCompactThreads) void paged_compact_kernel(const PagedEvictParams E) {
  const PagedParams& P = E.p;
  const int width = E.strip;  // 16-byte chunks of a strip, at most
  const int kstrips = P.D / (8 * width), rstrips = P.H_G > 0 ? cdiv(P.R, 8 * width) : 0;
  const int per = 2 * P.H_KV * kstrips + P.H_G * rstrips;  // strips of a sequence
  const int b = blockIdx.x / per;
  int x = blockIdx.x - b * per;
  const int lk = min(max(uni(*const_space(P.lens + b)), 0), P.width * P.ps);
  const int budget = E.budget;
  if (lk <= budget) return;
  int h, kvh, strip, chunks;  // head, its KV head, strip of the row, 16-byte chunks of it
  const int nk = P.H_KV * kstrips;
  const int which = x < nk ? 0 : x < 2 * nk ? 1 : 2;
  if (which < 2) {
    x -= which * nk;
    h = kvh = x / kstrips;
    strip = x - h * kstrips;
    chunks = width;
  } else {
    x -= 2 * nk;
    h = x / rstrips;
    kvh = h / P.group;
    strip = x - h * rstrips;
    chunks = min(P.R / 8 - width * strip, width);
  }
  const TView& t = which == 0 ? P.k : which == 1 ? P.v : P.rk;
  const int64_t sb = t.sb, ss = t.ss;
  const int ps = P.ps, npages = P.npages;
  const int* kept = E.kept + ((int64_t)b * P.H_KV + kvh) * budget;
  const int* trow = P.table + (int64_t)b * P.tstride;
  // lanes a row: the chunks, rounded up to a power of two
  const int lanes = chunks > 8 ? 16 : chunks > 4 ? 8 : chunks > 2 ? 4 : chunks;
  const int c = threadIdx.x & (lanes - 1), row0 = threadIdx.x / lanes, stride = blockDim.x / lanes;
  const int round = stride * kCompactAhead;
  uint16_t* base = (uint16_t*)t.ptr + (int64_t)h * t.sh + 8 * (width * strip + c);
  auto place = [&](int j) -> uint16_t* {
    const int pg = j / ps;
    const int id = trow[pg];
    return (uint32_t)id < (uint32_t)npages ? base + (int64_t)id * sb + (int64_t)(j - pg * ps) * ss
                                           : nullptr;
  };
  const uint16_t* src[kCompactAhead];
  uint16_t* dst[kCompactAhead];
  auto look = [&](int r0) {
    int j[kCompactAhead];
#pragma unroll
    for (int i = 0; i < kCompactAhead; ++i) {
      const int r = r0 + row0 + i * stride;
      j[i] = r < budget && c < chunks ? kept[r] : r;
    }
#pragma unroll
    for (int i = 0; i < kCompactAhead; ++i) {
      const int r = r0 + row0 + i * stride;
      src[i] = nullptr;
      if (j[i] != r) {
        src[i] = place(j[i]);
        dst[i] = place(r);
        if (!dst[i]) src[i] = nullptr;
      }
    }
  };
  look(0);
  for (int r0 = 0; r0 < budget; r0 += round) {
    u32x4 v[kCompactAhead];
    uint16_t* to[kCompactAhead];
#pragma unroll
    for (int i = 0; i < kCompactAhead; ++i) {
      to[i] = src[i] ? dst[i] : nullptr;
      if (src[i]) v[i] = ld16(src[i]);
    }
    if (r0 + round < budget) look(r0 + round);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);  // this wave's loads have their data ...
    __syncthreads();                // ... and every wave's
#pragma unroll
    for (int i = 0; i < kCompactAhead; ++i)
      if (to[i]) st16(to[i], v[i]);
    // (the next round's loads are of rows past every row stored so far)
  }
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendParams& A_, hipStream_t s) {
  PagedAppendParams A = A_;
  const PagedParams& P = A.p;
  if (P.T <= 0) return hipSuccess;
  // Few tokens (a decode step): all four waves of a workgroup on each, which
  // shortens the chain; many: one wave each.
  A.share = P.T <= 2048 ? 4 : 1;
  const int per = kAppWaves / A.share;
  const dim3 grid((uint32_t)std::min((P.T + per - 1) / per, 4096));
  void (*k)(const PagedAppendParams) =
      P.D == 64 ? (P.f16 ? paged_append_kernel<64, true> : paged_append_kernel<64, false>)
                : (P.f16 ? paged_append_kernel<128, true> : paged_append_kernel<128, false>);
  hipLaunchKernelGGL(k, grid, dim3(64 * kAppWaves), 0, s, A);
  return hipGetLastError();
}

hipError_t launch_paged_select(const PagedEvictParams& E, hipStream_t s) {
  const dim3 grid((uint32_t)(E.p.N * E.p.H_KV));
  if ((int64_t)E.p.width * E.p.ps <= 256 * kSelAhead)
    hipLaunchKernelGGL(paged_select_kernel<256>, grid, dim3(256), 0, s, E);
  else
    hipLaunchKernelGGL(paged_select_kernel<1024>, grid, dim3(1024), 0, s, E);
  return hipGetLastError();
}

hipError_t launch_paged_compact(const PagedEvictParams& E_, hipStream_t s) {
  PagedEvictParams E = E_;
  const PagedParams& P = E.p;
  auto strips = [&] {
    return 2 * (int64_t)P.H_KV * (P.D / (8 * E.strip)) + (P.H_G > 0 ? (int64_t)P.H_G * cdiv(P.R, 8 * E.strip) : 0);
  };
  E.strip = 8;
  while (E.strip > 2 && 2 * strips() * P.N <= 512 && E.budget > kCompactAhead * kCompactThreads / E.strip)
    E.strip /= 2;
  // (a small budget is one round of fewer waves)
  const int rows = cdiv(std::min(E.budget, 1 << 20), kCompactAhead);
  const int threads = std::min(kCompactThreads, cdiv(rows * E.strip, 64) * 64);
  hipLaunchKernelGGL(paged_compact_kernel, dim3((uint32_t)(strips() * P.N)), dim3((uint32_t)threads), 0, s, E);
  return hipGetLastError();
}

}  // namespace fna2
