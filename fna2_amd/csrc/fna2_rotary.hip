// fna2_rotary.hip — rotary positions in either layout, over part of the head,
// scaled, at given positions or those of packed sequences; with the QK norm.
//
// Token at position p, row x of D features, rd of them rotated, f = inv_freq:
//     n = x rsqrt(mean(x^2) + eps) w                   (rows with a norm)
//     (u, v) -> s (u cos a_i - v sin a_i, v cos a_i + u sin a_i),  a_i = p f_i,
// for the pairs i < rd / 2 of features (i, i + rd / 2) or, interleaved, (2i, 2i + 1); features
// from rd on stay n.  The angle is formed and reduced in fp64 (in fp32 it is off by
// 0.06 radians at position 10^6); the rest is fp32 with one rounding, at the store.
// Backward, with g = s R(-a) dy for the rotated features:
//     dx = r (w g - x r^2 mean(x w g)),  dw = sum of g x r,  r = rsqrt(mean(x^2) + eps),
// and dx = g without a norm, which is the forward kernel with the angle's sign
// changed.
//
// Bound by reading and writing every row once.  A lane owns two 16-byte chunks
// of a row that hold whole pairs: the same chunk of both halves, or (interleaved) two
// neighbours; LPR = D / (2 EPL) lanes a row.  Halves that do not begin on a chunk
// (rd / 2 not a multiple of EPL) have their pairs in different lanes: those go
// through LDS.  A wave forms the token's cos and sin once, a lane a pair.
//
// 16384 tokens of 32 + 8 heads of 128 in bf16, no norm, 65 us: 5.2 TB/s; of 16 + 16 with the norm
// 61 forward (4.4 TB/s), 91 backward (4.4), 5 for dw; 64 tokens of 32 + 8 5.6, one launch's latency.
// Halves that begin off a chunk (24 features; 32 of them, which do not, beside it): 16384 tokens of 16 + 16
// heads of 128 in bf16 59 us (43), with the norm 78 (45), backward and dw 116 (92), where the waves are two
// a SIMD and LDS takes the exchange; 5003 of 8 + 4 of 64 in fp32 9.8 (7.9), 11.0 (9.2), 20 (19).
#include <algorithm>

#include "fna2_rope_dev.h"

namespace fna2 {

namespace {

constexpr int kRotHalf = 0, kRotInter = 1, kRotAny = 2;
constexpr int kRotWaves = 4;
constexpr int kRotPasses = 4;  // row passes whose loads are in flight together
constexpr int kRotMaxHalf = 256;

__device__ __forceinline__ void rot_wave_sync() {
  // (one wave's own LDS: its reads follow its writes in order)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Sum over the lpr lanes of a row, every lane of the wave taking part.  Moves between
// lanes' registers up to 16 of them (row_sum's go through LDS).
template <int CTRL>
__device__ __forceinline__ float rot_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                                           0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float rot_row_sum(float v, int lpr) {
  if (lpr >= 2) v = rot_add<0xb1>(v);    // quad_perm 1, 0, 3, 2
  if (lpr >= 4) v = rot_add<0x4e>(v);    // quad_perm 2, 3, 0, 1
  if (lpr >= 8) v = rot_add<0x141>(v);   // row_half_mirror
  if (lpr >= 16) v = rot_add<0x140>(v);  // row_mirror
  if (lpr >= 32) v += __shfl_xor(v, 16);
  if (lpr >= 64) v += __shfl_xor(v, 32);
  return v;
}

// LDS of a wave: the token's cos and sin, and (kRotAny) the rows of a pass.
template <int DT, int MODE>
struct RotShared {
  float cos[kRotMaxHalf], sin[kRotMaxHalf];
  float x[MODE == kRotAny ? 2 * Chunk<DT>::EPL * 64 : 1];
};

// The norm weights (1 for a side without) to LDS.
__device__ __forceinline__ void rot_weights(const RotaryParams& P, float (*wsh)[512]) {
  for (int i = threadIdx.x; i < 2 * P.r.D; i += 64 * kRotWaves) {
    const int side = i >= P.r.D, d = i - side * P.r.D;
    const void* w = side ? P.r.wk : P.r.wq;
    float x = 1.f;
    if (w) {
      const uint16_t h = P.wdt == kRopeF32 ? 0 : ((const uint16_t*)w)[d];
      x = P.wdt == kRopeF32   ? ((const float*)w)[d]
          : P.wdt == kRopeF16 ? (float)__builtin_bit_cast(_Float16, h)
                              : __builtin_bit_cast(float, (uint32_t)h << 16);
    }
    wsh[side][d] = x;
  }
  __syncthreads();
}

template <int DT, int MODE>
struct RotLane {
  static constexpr int EPL = Chunk<DT>::EPL, N = 2 * EPL;
  RotShared<DT, MODE>& sh;
  int lane, lpr, rpw, col, lrow, o1, o2, half;
  float inv;  // of pair `lane` (those from 64 on are read when used)
  float c[MODE == kRotAny ? N : EPL], s[MODE == kRotAny ? N : EPL];
  int off[MODE == kRotAny ? N : 1];

  __device__ __forceinline__ RotLane(const RotaryParams& P, RotShared<DT, MODE>& shared) : sh(shared) {
    lane = threadIdx.x & 63;
    lpr = P.r.D / N;
    rpw = 64 / lpr;
    lrow = lane / lpr;
    col = (lane % lpr) * EPL;  // pairs col .. col + EPL - 1
    half = P.rd / 2;
    o1 = 2 * col, o2 = o1 + EPL;
    if (MODE == kRotHalf) {
      if (col < half) o1 = col, o2 = half + col;
    }
#pragma unroll
    for (int k = 0; k < kRotMaxHalf / 64; ++k) {
      sh.cos[lane + 64 * k] = 1.f;
      sh.sin[lane + 64 * k] = 0.f;
    }
    inv = lane < half ? P.r.inv_freq[lane] : 0.f;
    if constexpr (MODE == kRotAny) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int f = o1 + e, pf = f < half ? f + half : f < P.rd ? f - half : f;
        off[e] = pf % N * 64 + lane - lane % lpr + pf / N;
      }
    }
  }
  // The feature of this lane's value e.
  __device__ __forceinline__ int feature(int e) const { return e < EPL ? o1 + e : o2 + e - EPL; }

  // cos and sin of position p for the lane's pairs.
  __device__ __forceinline__ void at(const RotaryParams& P, int p, float sign) {
#pragma unroll 1
    for (int i = lane; i - lane < half; i += 64) {
      if (i < half) {
        // in turns, reduced to half a turn either way
        const float f = i < 64 ? inv : P.r.inv_freq[i];
        const double x = (double)p * (double)f * 0.15915494309189533577;
        float sv, cv;
        sincospif((float)(2. * (x - __builtin_rint(x))), &sv, &cv);
        sh.cos[i] = cv * P.scale;
        sh.sin[i] = sign * sv * P.scale;
      }
    }
    rot_wave_sync();
    if constexpr (MODE == kRotAny) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int f = o1 + e, i = f < half ? f : f < P.rd ? f - half : 0;
        c[e] = sh.cos[i];
        s[e] = f < half ? -sh.sin[i] : sh.sin[i];
      }
    } else {
#pragma unroll
      for (int e = 0; e < EPL; ++e) c[e] = sh.cos[col + e], s[e] = sh.sin[col + e];
    }
    rot_wave_sync();
  }

  // Rotates the lane's values.  (Every lane of the wave comes here.)
  __device__ __forceinline__ void turn(float (&x)[N]) const {
    if constexpr (MODE == kRotAny) {
#pragma unroll
      for (int e = 0; e < N; ++e) sh.x[64 * e + lane] = x[e];
      rot_wave_sync();
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float y = x[e] * c[e] + sh.x[off[e]] * s[e];
        x[e] = o1 + e < 2 * half ? y : x[e];
      }
      rot_wave_sync();
    } else {
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const int i = MODE == kRotInter ? 2 * e : e, j = MODE == kRotInter ? 2 * e + 1 : EPL + e;
        const float u = x[i], v = x[j];
        const bool in = MODE == kRotInter ? col + e < half : col < half;
        x[i] = in ? u * c[e] - v * s[e] : u;
        x[j] = in ? v * c[e] + u * s[e] : v;
      }
    }
  }
};

// A wave's tokens, and the position of each (inside: it is rotated).
struct RotTokens {
  int t0, n, b;
  __device__ __forceinline__ RotTokens(const RotaryParams& P, int unit) {
    t0 = unit * P.r.tpw;
    n = min(P.r.T - t0, P.r.tpw);
    b = -1;
    if (P.pos || n <= 0) return;
    // Largest b with cu[b] <= t0 (b = -1: before the first sequence).
    const auto cu = const_space(P.r.cu);
    int lo = -1, hi = P.r.nseq;
    if (uni(cu[hi]) <= t0) lo = hi;
    else
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (uni(cu[mid]) <= t0) lo = mid;
        else hi = mid;
      }
    b = lo;
  }
  __device__ __forceinline__ int position(const RotaryParams& P, int t, bool& inside) {
    inside = true;
    if (P.pos) return uni(*const_space(P.pos + t));
    const auto cu = const_space(P.r.cu);
    while (b < P.r.nseq && uni(cu[b + 1]) <= t) ++b;
    inside = b >= 0 && b < P.r.nseq;
    return inside ? t - uni(cu[b]) : 0;
  }
};

template <int DT, int MODE, bool NORM>
__global__ __launch_bounds__(64 * kRotWaves, MODE == kRotAny ? 2 : 4) void rotary_kernel(const RotaryParams P) {
  using Ch = Chunk<DT>;
  constexpr int EPL = Ch::EPL, N = 2 * EPL, ES = DT == kRopeF32 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) RotShared<DT, MODE> shared[kRotWaves];
  __shared__ float wsh[NORM ? 2 : 1][NORM ? 512 : 1];
  const RopeParams& R = P.r;
  const int wv = uni(threadIdx.x >> 6);
  if constexpr (NORM) rot_weights(P, wsh);
  const int unit = blockIdx.x * kRotWaves + wv;
  RotLane<DT, MODE> L(P, shared[wv]);
  RotTokens tokens(P, unit / P.share);
  // Row passes, q's and then k's, of the waves that share the token.
  const int step = L.rpw * P.share, first = unit % P.share * L.rpw + L.lrow, nq = cdiv(R.Hq, step), passes = nq + cdiv(R.Hk, step);
  const int batches = cdiv(passes, kRotPasses), batch = cdiv(passes, max(batches, 1));
  const float inv_d = 1.f / (float)R.D, sign = (float)R.sign;
  const bool in_place = R.q == R.q_out && R.k == R.k_out;

  for (int it = 0; it < tokens.n; ++it) {
    const int t = tokens.t0 + it;
    Raw<DT> x1[kRotPasses], x2[kRotPasses];
    auto load = [&](int j0) {
#pragma unroll
      for (int j = 0; j < kRotPasses; ++j) {
        if (j >= batch || j0 + j >= passes) break;
        const bool k = j0 + j >= nq;  // (the same for every lane)
        const int r = (j0 + j - (k ? nq : 0)) * step + first;
        x1[j].w = x2[j].w = u32x4{0u, 0u, 0u, 0u};
        if (r < (k ? R.Hk : R.Hq)) {
          const char* src = (const char*)(k ? R.k : R.q) + (int64_t)t * ((k ? R.k_ss : R.q_ss) * ES) +
                            (int64_t)r * ((k ? R.k_sh : R.q_sh) * ES);
          x1[j].load(src + L.o1 * ES);
          x2[j].load(src + L.o2 * ES);
        }
      }
    };
    load(0);  // (ahead of the angles, which take as long)
    bool inside;
    const int p = tokens.position(P, t, inside);
    if (inside) L.at(P, p, sign);
    else if (in_place) continue;
#pragma unroll 1
    for (int j0 = 0; j0 < passes; j0 += batch) {
      if (j0 > 0) load(j0);
#pragma unroll
      for (int j = 0; j < kRotPasses; ++j) {
        if (j >= batch || j0 + j >= passes) break;
        const bool k = j0 + j >= nq;
        const int r = (j0 + j - (k ? nq : 0)) * step + first;
        char* dst = (char*)(k ? R.k_out : R.q_out) + (int64_t)t * ((k ? R.ko_ss : R.qo_ss) * ES) +
                    (int64_t)r * ((k ? R.ko_sh : R.qo_sh) * ES);
        const bool live = r < (k ? R.Hk : R.Hq);
        if (inside) {
          float x[N];
#pragma unroll
          for (int e = 0; e < EPL; ++e) x[e] = x1[j].get(e), x[EPL + e] = x2[j].get(e);
          if constexpr (NORM) {
            if ((k ? R.wk : R.wq) != nullptr) {
              float ss = 0.f;
#pragma unroll
              for (int e = 0; e < N; ++e) ss += x[e] * x[e];
              // (a lane past the rows holds zeros; every lane joins the sum)
              const float rs = rsqrtf(rot_row_sum(ss, L.lpr) * inv_d + R.eps);
              const float* w = wsh[k];
#pragma unroll
              for (int e = 0; e < EPL; ++e) {
                x[e] = x[e] * rs * w[L.o1 + e];
                x[EPL + e] = x[EPL + e] * rs * w[L.o2 + e];
              }
            }
          }
          L.turn(x);
          Ch y1, y2;
#pragma unroll
          for (int e = 0; e < EPL; ++e) y1.v[e] = x[e], y2.v[e] = x[EPL + e];
          if (live) {
            y1.store(dst + L.o1 * ES);
            y2.store(dst + L.o2 * ES);
          }
        } else if (live) {
          x1[j].store(dst + L.o1 * ES);
          x2[j].store(dst + L.o2 * ES);
        }
        __builtin_amdgcn_sched_barrier(0);  // (one pass's values at a time: registers)
      }
    }
  }
}

// Backward of the normalised rotation.  Each workgroup writes its part of dw, in a
// fixed order, to part[2][gridDim.x][D].
template <int DT, int MODE>
__global__ __launch_bounds__(64 * kRotWaves, MODE == kRotAny ? 2 : 4) void rotary_norm_bwd_kernel(
    const RotaryParams P) {
  using Ch = Chunk<DT>;
  constexpr int EPL = Ch::EPL, N = 2 * EPL, ES = DT == kRopeF32 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) RotShared<DT, MODE> shared[kRotWaves];
  __shared__ float red[2][kRotWaves][512];
  __shared__ float wsh[2][512];
  const RopeParams& R = P.r;
  const int wv = uni(threadIdx.x >> 6);
  rot_weights(P, wsh);
  RotLane<DT, MODE> L(P, shared[wv]);
  const int unit = blockIdx.x * kRotWaves + wv, step = L.rpw * P.share, first = unit % P.share * L.rpw;
  RotTokens tokens(P, unit / P.share);
  const float inv_d = 1.f / (float)R.D, sign = -(float)R.sign;
  float dw[2][N];
#pragma unroll
  for (int e = 0; e < N; ++e) dw[0][e] = dw[1][e] = 0.f;

  for (int it = 0; it < tokens.n; ++it) {
    const int t = tokens.t0 + it;
    bool inside;
    const int p = tokens.position(P, t, inside);
    if (inside) L.at(P, p, sign);
    auto rows = [&](auto side_, int r0) {
      constexpr int side = decltype(side_)::value;
      const int r = r0 + L.lrow;
      const bool live = r < (side ? R.Hk : R.Hq);
      Raw<DT> x1, x2, g1, g2;
      x1.w = x2.w = g1.w = g2.w = u32x4{0u, 0u, 0u, 0u};
      if (live) {
        const char* x = (const char*)(side ? R.k : R.q) +
                        ((int64_t)t * (side ? R.k_ss : R.q_ss) + (int64_t)r * (side ? R.k_sh : R.q_sh)) * ES;
        const char* g = (const char*)(side ? R.gk : R.gq) +
                        ((int64_t)t * (side ? R.gk_ss : R.gq_ss) + (int64_t)r * (side ? R.gk_sh : R.gq_sh)) * ES;
        x1.load(x + L.o1 * ES);
        x2.load(x + L.o2 * ES);
        g1.load(g + L.o1 * ES);
        g2.load(g + L.o2 * ES);
      }
      char* out = (char*)(side ? R.k_out : R.q_out) +
                  ((int64_t)t * (side ? R.ko_ss : R.qo_ss) + (int64_t)r * (side ? R.ko_sh : R.qo_sh)) * ES;
      if (!inside) {  // (the same for every lane)
        if (live) {
          g1.store(out + L.o1 * ES);
          g2.store(out + L.o2 * ES);
        }
        return;
      }
      float y[N];
#pragma unroll
      for (int e = 0; e < EPL; ++e) y[e] = g1.get(e), y[EPL + e] = g2.get(e);
      L.turn(y);
      if ((side ? R.wk : R.wq) != nullptr) {
        float ss = 0.f, tw = 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float u = e < EPL ? x1.get(e) : x2.get(e - EPL);
          ss += u * u;
          tw += u * wsh[side][L.feature(e)] * y[e];
        }
        // (a lane past the rows holds zeros; every lane joins the sums)
        ss = rot_row_sum(ss, L.lpr);
        tw = rot_row_sum(tw, L.lpr);
        // (fp16, interleaved: the products below stay behind the sums, or 10 registers spill)
        if constexpr (DT == kRopeF16) asm volatile("" : "+v"(ss));
        const float rr = rsqrtf(ss * inv_d + R.eps);
        const float k3 = rr * rr * rr * tw * inv_d;
        if (live) {
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float u = e < EPL ? x1.get(e) : x2.get(e - EPL);
            dw[side][e] += u * rr * y[e];
            y[e] = rr * wsh[side][L.feature(e)] * y[e] - u * k3;
          }
        }
      }
      if (live) {
        Ch y1, y2;
#pragma unroll
        for (int e = 0; e < EPL; ++e) y1.v[e] = y[e], y2.v[e] = y[EPL + e];
        y1.store(out + L.o1 * ES);
        y2.store(out + L.o2 * ES);
      }
    };
    for (int r = first; r < R.Hq; r += step) rows(std::integral_constant<int, 0>{}, r);
    for (int r = first; r < R.Hk; r += step) rows(std::integral_constant<int, 1>{}, r);
  }

  // dw: lanes that share features, then the waves.
#pragma unroll
  for (int e = 0; e < N; ++e)
    for (int m = L.lpr; m < 64; m <<= 1) {
      dw[0][e] += __shfl_xor(dw[0][e], m);
      dw[1][e] += __shfl_xor(dw[1][e], m);
    }
  if (L.lane < L.lpr) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      red[0][wv][L.feature(e)] = dw[0][e];
      red[1][wv][L.feature(e)] = dw[1][e];
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < 2 * R.D; d += 64 * kRotWaves) {
    const int which = d / R.D, dd = d - which * R.D;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kRotWaves; ++w) v += red[which][w][dd];
    R.part[((int64_t)which * gridDim.x + blockIdx.x) * R.D + dd] = v;
  }
}

// dw = the workgroups' parts added up, in 64 bits and a fixed order: workgroup x
// takes 64 of the 2 D columns, its 16 waves every 16th part each.
__global__ __launch_bounds__(1024) void rotary_dw_kernel(const RotaryParams P, int nblocks) {
  __shared__ double acc[16][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, D = P.r.D;
  const int i = blockIdx.x * 64 + lane;
  const bool ok = i < 2 * D;
  const int side = ok && i >= D, d = ok ? i - side * D : 0;
  const float* src = P.r.part + (int64_t)side * nblocks * D + d;
  double v = 0.;
  int b = wv;
  for (; b + 7 * 16 < nblocks; b += 8 * 16) {  // eight loads in flight
    float t[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) t[u] = src[(int64_t)(b + 16 * u) * D];
#pragma unroll
    for (int u = 0; u < 8; ++u) v += t[u];
  }
  for (; b < nblocks; b += 16) v += src[(int64_t)b * D];
  acc[wv][lane] = v;
  __syncthreads();
  if (wv != 0 || !ok) return;
  double sum = 0.;
#pragma unroll
  for (int w = 0; w < 16; ++w) sum += acc[w][lane];
  void* out = side ? P.r.dwk : P.r.dwq;
  if (!out) return;
  const float x = (float)sum;
  if (P.wdt == kRopeF32) ((float*)out)[d] = x;
  else if (P.wdt == kRopeF16) ((_Float16*)out)[d] = (_Float16)x;
  else ((uint16_t*)out)[d] = (uint16_t)pack_bf16(x, 0.f);
}

template <int DT>
void launch_fwd(const RotaryParams& P, int mode, dim3 grid, hipStream_t s) {
  const bool norm = P.r.wq || P.r.wk;
  void (*k)(const RotaryParams) =
      mode == kRotHalf    ? (norm ? rotary_kernel<DT, kRotHalf, true> : rotary_kernel<DT, kRotHalf, false>)
      : mode == kRotInter ? (norm ? rotary_kernel<DT, kRotInter, true> : rotary_kernel<DT, kRotInter, false>)
                          : (norm ? rotary_kernel<DT, kRotAny, true> : rotary_kernel<DT, kRotAny, false>);
  hipLaunchKernelGGL(k, grid, dim3(64 * kRotWaves), 0, s, P);
}
template <int DT>
void launch_bwd(const RotaryParams& P, int mode, dim3 grid, hipStream_t s) {
  void (*k)(const RotaryParams) = mode == kRotHalf    ? rotary_norm_bwd_kernel<DT, kRotHalf>
                                  : mode == kRotInter ? rotary_norm_bwd_kernel<DT, kRotInter>
                                                      : rotary_norm_bwd_kernel<DT, kRotAny>;
  hipLaunchKernelGGL(k, grid, dim3(64 * kRotWaves), 0, s, P);
}

int rot_mode(const RotaryParams& P) {
  const int epl = P.r.dtype == kRopeF32 ? 4 : 8;
  return P.inter ? kRotInter : (P.rd / 2) % epl == 0 ? kRotHalf : kRotAny;
}
// Consecutive tokens per wave, which share its start: one while the waves leave
// the chip with room, or where a token has three passes of rows and more; four once
// short ones fill it.  (us, 1 / 2 / 4 tokens, with norm: 16384 tokens x 32 heads of 128, four passes,
// 52.8 / 53.9 / 54.6; x 12 of 64, one pass, 22.1 / 19.1 / 17.8; 8000 x 12 of 64 in fp32 13.0 / 12.1 /
// 14.0; 2000 x 16 6.4 / 7.2 / 10.8.)  The backward leaves its part of dw as well: 1000 tokens x 40 18.8 /
// 25.4 / 39.0, 8000 x 12 29.2 / 23.7 / 24.1, 16384 x 32 103 / 93 / 92.
int rot_tokens(const RotaryParams& P) {
  const int rpw = 64 * (P.r.dtype == kRopeF32 ? 8 : 16) / P.r.D;
  if (P.r.T <= 256 || cdiv(P.r.Hq, rpw) + cdiv(P.r.Hk, rpw) >= 3) return 1;
  return P.r.T <= 4096 ? 1 : P.r.T <= 12288 ? 2 : 4;
}
int rot_bwd_tokens(int T) { return T <= 1024 ? 1 : T <= 12288 ? 2 : 4; }
// Few tokens with four passes of rows and more: the waves of a workgroup share each (us, one wave a
// token and four: 64 tokens x 64 rows of 128 17.3, 12.3; 256 20.0, 13.0; 500 21.2, 17.1; 1000 x 32 17.6, 19.9;
// 500 x 16 rows of 64, two passes, 13.8, 15.4).
int rot_bwd_share(const RopeParams& R) {
  const int rpw = 64 * (R.dtype == kRopeF32 ? 8 : 16) / R.D;
  return R.T <= 512 && cdiv(R.Hq, rpw) + cdiv(R.Hk, rpw) >= 4 ? kRotWaves : 1;
}

}  // namespace

int rotary_bwd_blocks(const RopeParams& R) {
  const int T = R.T;
  const int64_t waves = ((int64_t)T + rot_bwd_tokens(T) - 1) / rot_bwd_tokens(T) * rot_bwd_share(R);
  return (int)((waves + kRotWaves - 1) / kRotWaves);
}

hipError_t launch_rotary(const RotaryParams& args, hipStream_t s) {
  RotaryParams P = args;
  if (P.r.T <= 0 || P.r.Hq + P.r.Hk <= 0) return hipSuccess;
  P.r.tpw = rot_tokens(P);
  // Few tokens: the waves of a workgroup share each (us, 64 tokens x 40 rows of 128, one
  // wave a token 7.0, four 5.0; 1000 8.5, 8.8; 16384 x 32 53, 83).
  P.share = P.r.T <= 256 ? kRotWaves : 1;
  const int64_t waves = ((int64_t)P.r.T + P.r.tpw - 1) / P.r.tpw * P.share;
  const dim3 grid((uint32_t)((waves + kRotWaves - 1) / kRotWaves));
  switch (P.r.dtype) {
    case kRopeBF16: launch_fwd<kRopeBF16>(P, rot_mode(P), grid, s); break;
    case kRopeF16: launch_fwd<kRopeF16>(P, rot_mode(P), grid, s); break;
    case kRopeF32: launch_fwd<kRopeF32>(P, rot_mode(P), grid, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_rotary_norm_bwd(const RotaryParams& args, hipStream_t s) {
  RotaryParams P = args;
  if (P.r.T <= 0 || P.r.Hq + P.r.Hk <= 0) return hipSuccess;
  P.r.tpw = rot_bwd_tokens(P.r.T);
  P.share = rot_bwd_share(P.r);
  const int nb = rotary_bwd_blocks(P.r);
  const dim3 grid((uint32_t)nb);
  switch (P.r.dtype) {
    case kRopeBF16: launch_bwd<kRopeBF16>(P, rot_mode(P), grid, s); break;
    case kRopeF16: launch_bwd<kRopeF16>(P, rot_mode(P), grid, s); break;
    case kRopeF32: launch_bwd<kRopeF32>(P, rot_mode(P), grid, s); break;
    default: return hipErrorInvalidValue;
  }
  if (hipGetLastError() != hipSuccess) return hipErrorLaunchFailure;
  hipLaunchKernelGGL(rotary_dw_kernel, dim3((2 * P.r.D + 63) / 64), dim3(1024), 0, s, P, nb);
  return hipGetLastError();
}

}  // namespace fna2
