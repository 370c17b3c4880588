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
// A wave takes one token at a time: its lanes form the token's cos and sin
// once, then walk the token's rows, LPR = D / 16 lanes a row, each with 8
// values of the first half and the matching 8 of the second.  Bound by
// reading and writing every row once.
constexpr int kAppWaves = 4;
template <int D, bool F16>
__global__ __launch_bounds__(64 * kAppWaves) void paged_append_kernel(const PagedAppendParams A) {
  constexpr int LPR = D / 16, HALF = D / 2, RPP = 64 / LPR;  // rows a pass
  const PagedParams& P = A.p;
  __shared__ float table[kAppWaves][2 * HALF];
  const int lane = threadIdx.x & 63, wv = uni(threadIdx.x >> 6);
  float* cs = table[wv];
  const int i = lane % LPR, lrow = lane / LPR, col = 8 * i;
  const auto cu = const_space(P.cu);
  const int nv = P.H + P.H_KV, nr = nv + P.H_KV, per = nr + P.H_G;
  float wn[2][16];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    wn[0][e] = A.wq ? A.wq[col + e] : 1.f;
    wn[0][8 + e] = A.wq ? A.wq[HALF + col + e] : 1.f;
    wn[1][e] = A.wk ? A.wk[col + e] : 1.f;
    wn[1][8 + e] = A.wk ? A.wk[HALF + col + e] : 1.f;
  }
  const double inv = A.inv_freq && lane < HALF ? (double)A.inv_freq[lane] : 0.0;

  for (int t = blockIdx.x * kAppWaves + wv; t < P.T; t += gridDim.x * kAppWaves) {
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
    int row = -1;
    int64_t page = -1;
    int pr = 0;
    if (inside) {
      const PagedSeq e = paged_seq_uniform(kargs(), lo);
      row = e.lk - e.lq + (t - e.q0);
      if (row >= 0 && row < e.lk) {
        const int pg = row / P.ps;
        pr = row - pg * P.ps;
        const int id = uni(*const_space(P.table + (int64_t)lo * P.tstride + pg));
        if ((uint32_t)id < (uint32_t)P.npages) page = id;
      }
    }
    const bool turn = inside && A.inv_freq;
    if (turn) {
      const int pos = A.pos ? uni(*const_space(A.pos + t)) : row;
      if (lane < HALF) {
        // in turns, reduced to half a turn either way
        const double x = (double)pos * inv * 0.15915494309189533577;
        const float a = (float)((x - __builtin_rint(x)) * 6.28318530717958647693);
        float s, c;
        sincosf(a, &s, &c);
        cs[lane] = c;
        cs[HALF + lane] = s;
      }
      // (one wave's own LDS: its reads follow its writes in order)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    float co[8], si[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      co[e] = turn ? cs[col + e] : 1.f;
      si[e] = turn ? cs[HALF + col + e] : 0.f;
    }
    if (turn) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    for (int r0 = 0; r0 < nr; r0 += RPP) {
      const int r = r0 + lrow;
      const bool isq = r < P.H, isk = !isq && r < nv, have = r < nr;
      const int h = isq ? r : isk ? r - P.H : r - nv;
      u32x4 a = {0, 0, 0, 0}, b = a;
      uint16_t* dst = nullptr;
      if (have) {
        const uint16_t* src;
        if (isq) {
          src = (const uint16_t*)P.q.ptr + (int64_t)t * P.q.ss + (int64_t)h * P.q.sh;
          dst = (uint16_t*)P.o.ptr + (int64_t)t * P.o.ss + (int64_t)h * P.o.sh;
        } else {
          const TView& n = isk ? A.kn : A.vn;
          const TView& d = isk ? P.k : P.v;
          src = (const uint16_t*)n.ptr + (int64_t)t * n.ss + (int64_t)h * n.sh;
          if (page >= 0) dst = (uint16_t*)d.ptr + page * d.sb + (int64_t)h * d.sh + (int64_t)pr * d.ss;
        }
        if (dst) {
          a = ld16(src + col);
          b = ld16(src + HALF + col);
        }
      }
      const bool norm = isq ? A.wq != nullptr : A.wk != nullptr;
      float x[16];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = elt_lo<F16>(a[e]), x[2 * e + 1] = elt_hi<F16>(a[e]);
        x[8 + 2 * e] = elt_lo<F16>(b[e]), x[8 + 2 * e + 1] = elt_hi<F16>(b[e]);
      }
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) ss += x[e] * x[e];
#pragma unroll
      for (int m = 1; m < LPR; m <<= 1) ss += __shfl_xor(ss, m);
      if (inside && (isq || isk)) {
        if (norm) {
          const float rs = rsqrtf(ss * (1.f / D) + A.eps);
          const float* w = wn[0];
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = x[e] * rs * (isq ? wn[0][e] : wn[1][e]);
          (void)w;
        }
        if (norm || turn) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p0 = x[2 * e], p1 = x[2 * e + 1], q0 = x[8 + 2 * e], q1 = x[8 + 2 * e + 1];
            const float c0 = co[2 * e], c1 = co[2 * e + 1], s0 = si[2 * e], s1 = si[2 * e + 1];
            a[e] = pack_e<F16>(turn ? p0 * c0 - q0 * s0 : p0, turn ? p1 * c1 - q1 * s1 : p1);
            b[e] = pack_e<F16>(turn ? q0 * c0 + p0 * s0 : q0, turn ? q1 * c1 + p1 * s1 : q1);
          }
        }
      }
      if (dst) {
        st16(dst + col, a);
        st16(dst + HALF + col, b);
      }
    }
    if (P.H_G > 0 && page >= 0) {
      const int cr = P.R / 8, n = P.H_G * cr;
      for (int j = lane; j < n; j += 64) {
        const int h = j / cr, ch = j - h * cr;
        st16((uint16_t*)P.rk.ptr + page * P.rk.sb + (int64_t)h * P.rk.sh + (int64_t)pr * P.rk.ss + 8 * ch,
             ld16((const uint16_t*)A.rkn.ptr + (int64_t)t * A.rkn.ss + (int64_t)h * A.rkn.sh + 8 * ch));
      }
    }
    (void)per;
  }
}

// ── Eviction ───────────────────────────────────────────────────────────────
// Selection, one workgroup per (sequence, KV head): the `top` = budget - first
// - recent rows of largest weight among rows [first, lk - recent).  Weights
// become unsigned keys in their order; four passes of 8 bits find the top-th
// largest key K, and the rows kept are those above K and, of those equal
// to K, the lowest (top minus the rows above).  A last pass writes the kept
// rows in their order.
constexpr int kSelThreads = 1024;
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);  // (-0 as 0)
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Sum over the workgroup's threads up to and including this one (exclusive
// of it: minus x); `total` the sum of all.  sh: one int per wave.
__device__ __forceinline__ int block_scan(int x, int* sh, int& total) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int o = __shfl_up(s, m);
    if (lane >= m) s += o;
  }
  __syncthreads();
  if (lane == 63) sh[wv] = s;
  __syncthreads();
  int base = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kSelThreads / 64; ++i) {
    if (i < wv) base += sh[i];
    total += sh[i];
  }
  return base + s;
}

__global__ __launch_bounds__(kSelThreads) void paged_select_kernel(const PagedEvictParams E) {
  const PagedParams& P = E.p;
  __shared__ int hist[256];
  __shared__ int sh[kSelThreads / 64];
  __shared__ int pick[2];
  const int b = blockIdx.x / P.H_KV, kvh = blockIdx.x % P.H_KV, tid = threadIdx.x;
  const int lk = min(max(uni(*const_space(P.lens + b)), 0), P.width * P.ps);
  const int keep = min(lk, E.budget);
  if (kvh == 0 && tid == 0) E.new_lens[b] = keep;
  const float* w = E.w + (int64_t)b * E.w_sb + (int64_t)kvh * E.w_sh;
  float* wo = E.w_out + ((int64_t)b * P.H_KV + kvh) * E.cap;
  int* kept = E.kept + ((int64_t)b * P.H_KV + kvh) * E.budget;
  auto weight = [&](int j) { return j < E.cap ? w[j] : 0.f; };
  for (int j = keep + tid; j < E.budget; j += kSelThreads) kept[j] = -1;
  for (int j = keep + tid; j < E.cap; j += kSelThreads) wo[j] = 0.f;
  if (lk <= E.budget) {
    for (int j = tid; j < keep; j += kSelThreads) {
      kept[j] = j;
      if (j < E.cap) wo[j] = w[j];
    }
    return;
  }
  const int lo = E.first, hi = lk - E.recent, top = E.budget - E.first - E.recent;
  uint32_t prefix = 0, mask = 0;
  int need = top;  // rows still to find among those that match the prefix
  if (top > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int j = lo + tid; j < hi; j += kSelThreads) {
        const uint32_t k = weight_key(weight(j));
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      // the digit d whose rows, with those of larger digits, reach `need`
      int total;
      const int mine = tid < 256 ? hist[255 - tid] : 0;
      const int s = block_scan(mine, sh, total);
      if (tid < 256 && s >= need && s - mine < need) {
        pick[0] = 255 - tid;
        pick[1] = s - mine;
      }
      __syncthreads();
      prefix |= (uint32_t)pick[0] << shift;
      mask |= 255u << shift;
      need -= pick[1];
      __syncthreads();
    }
  }
  // kept rows in order; of the rows equal to the key, the first `need`
  int out = 0, equal = 0;  // rows written, equal rows passed
  for (int j0 = 0; j0 < lk; j0 += kSelThreads) {
    const int j = j0 + tid;
    const bool fixed = j < lk && (j < lo || j >= hi);
    const uint32_t k = j >= lo && j < hi && top > 0 ? weight_key(weight(j)) : 0u;
    const bool cand = j >= lo && j < hi && top > 0;
    const bool eq = cand && k == prefix;
    int eq_all;
    const int eq_at = equal + block_scan(eq ? 1 : 0, sh, eq_all) - 1;
    const bool yes = fixed || (cand && k > prefix) || (eq && eq_at < need);
    int all;
    const int at = out + block_scan(yes ? 1 : 0, sh, all) - 1;
    if (yes) {
      kept[at] = j;
      if (at < E.cap) wo[at] = weight(j);
    }
    out += all;
    equal += eq_all;
  }
}

// Compaction in place: row kept[r] becomes row r (kept[r] >= r, increasing).
// A unit is a wave: a strip of 64 bytes of every row of one (sequence, head)
// of K, V or R_k, walked in order, kAhead x 16 rows at a time: all of their
// loads, then all of their stores.  Rows stored so lie before every row that
// is still to be loaded, so a strip needs no other copy and no barrier.
// Bound by reading and writing the rows that move; the strips of a row are
// neighbouring waves, so that its lines are fetched together.
constexpr int kCompactAhead = 8;
__global__ __launch_bounds__(256) void paged_compact_kernel(const PagedEvictParams E) {
  const PagedParams& P = E.p;
  const int lane = threadIdx.x & 63, wv = uni(threadIdx.x >> 6);
  const int kstrips = P.D / 32, rstrips = P.H_G > 0 ? cdiv(P.R, 32) : 0;
  const int per = 2 * P.H_KV * kstrips + P.H_G * rstrips;  // units of a sequence
  const int64_t unit = (int64_t)blockIdx.x * 4 + wv;
  const int b = uni((int)(unit / per));
  if (b >= P.N) return;
  int x = (int)(unit - (int64_t)b * per);
  const int lk = min(max(uni(*const_space(P.lens + b)), 0), P.width * P.ps);
  if (lk <= E.budget) return;
  TView t;
  int h, kvh, strip, chunks;  // head, its KV head, 64-byte strip, 16-byte chunks of it
  if (x < 2 * P.H_KV * kstrips) {
    t = x < P.H_KV * kstrips ? P.k : P.v;
    x %= P.H_KV * kstrips;
    h = kvh = x / kstrips;
    strip = x % kstrips;
    chunks = 4;
  } else {
    x -= 2 * P.H_KV * kstrips;
    t = P.rk;
    h = x / rstrips;
    kvh = h / P.group;
    strip = x % rstrips;
    chunks = min(P.R / 8 - 4 * strip, 4);
  }
  const int* kept = E.kept + ((int64_t)b * P.H_KV + kvh) * E.budget;
  const int* trow = P.table + (int64_t)b * P.tstride;
  uint16_t* base = (uint16_t*)t.ptr + (int64_t)h * t.sh + 32 * strip + 8 * (lane & 3);
  const bool on = (lane & 3) < chunks;
  auto place = [&](int j) -> uint16_t* {
    const int pg = j / P.ps;
    const int id = trow[pg];
    if ((uint32_t)id >= (uint32_t)P.npages) return nullptr;
    return base + (int64_t)id * t.sb + (int64_t)(j - pg * P.ps) * t.ss;
  };
  for (int r0 = 0; r0 < E.budget; r0 += 16 * kCompactAhead) {
    u32x4 v[kCompactAhead];
    uint16_t* dst[kCompactAhead];
#pragma unroll
    for (int i = 0; i < kCompactAhead; ++i) {
      const int r = r0 + 16 * i + (lane >> 2);
      dst[i] = nullptr;
      if (r < E.budget && on) {
        const int j = kept[r];
        if (j != r) {
          const uint16_t* src = place(j);
          if (src) {
            dst[i] = place(r);
            v[i] = ld16(src);
          }
        }
      }
    }
    __builtin_amdgcn_s_waitcnt(0);  // every load of the group has its data
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kCompactAhead; ++i)
      if (dst[i]) st16(dst[i], v[i]);
  }
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendParams& A, hipStream_t s) {
  const PagedParams& P = A.p;
  if (P.T <= 0) return hipSuccess;
  const dim3 grid((uint32_t)std::min((P.T + kAppWaves - 1) / kAppWaves, 4096));
  void (*k)(const PagedAppendParams) =
      P.D == 64 ? (P.f16 ? paged_append_kernel<64, true> : paged_append_kernel<64, false>)
                : (P.f16 ? paged_append_kernel<128, true> : paged_append_kernel<128, false>);
  hipLaunchKernelGGL(k, grid, dim3(64 * kAppWaves), 0, s, A);
  return hipGetLastError();
}

hipError_t launch_paged_select(const PagedEvictParams& E, hipStream_t s) {
  hipLaunchKernelGGL(paged_select_kernel, dim3((uint32_t)(E.p.N * E.p.H_KV)), dim3(kSelThreads), 0, s, E);
  return hipGetLastError();
}

hipError_t launch_paged_compact(const PagedEvictParams& E, hipStream_t s) {
  const PagedParams& P = E.p;
  const int64_t per = 2 * (int64_t)P.H_KV * (P.D / 32) + (P.H_G > 0 ? (int64_t)P.H_G * ((P.R + 31) / 32) : 0);
  const int64_t units = per * P.N;
  hipLaunchKernelGGL(paged_compact_kernel, dim3((uint32_t)((units + 3) / 4)), dim3(256), 0, s, E);
  return hipGetLastError();
}

}  // namespace fna2
