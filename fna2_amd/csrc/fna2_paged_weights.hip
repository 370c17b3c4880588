// fna2_paged_weights.hip — the cached rows' attention weights.
//
//     W_j += sum over the chunk's tokens i and the KV head's query heads h of
//            e^{S_hij - LSE_hi},
// S as in fna2_paged_attn.hip, whose LSE this takes.  Two kernels, for the two of
// the attention; in both keys are the columns of S = Q K^T, so that a lane
// sums its key's weights in registers, in fp32 and in a fixed order, and adds them
// to W once.
//
// Long chunks (weigh kernel): a wave keeps 32 keys (K, and R_k of the head at
// hand) in registers and walks the chunk's row tiles, 32 tokens of one head
// each, which the workgroup's four waves share.  They come through a two-stage LDS
// ring by DMA, two tiles a stage, with each row's -LSE log2(e) (-inf: it sees nothing,
// or is none).  Rows of a tile that no token fills, here and below, repeat the tile's
// first one: e^{S - inf} is then 0 where that row's own weight is a number, while zeros
// times an infinity in K or R_k would be NaN in the key's sum.  Blocks of 128 keys, or of 64
// with the tiles halved between two waves, go round over the workgroups.
// Bound by the blocks' uneven rounds and their starts, not by a pipe: 2 chunks of 509
// tokens over 7001 rows, 16 heads of 64, R = 16, 36 us, 2.1 10^12 weights a second.  A
// tile's 1024 weights take 384 cycles of a SIMD's vector instructions (16 exponentials
// of 16, scale and sum 8 each) and 192 of its products (6 of 32), which over the whole
// chip would be 6.5 10^12 a second; counted, all vector instructions spread evenly
// would take 18 us, the exponentials 8 of them, and the products 6.  But 1360
// blocks for 1024 resident workgroups are two rounds, the second a third full, and a
// block begins with a chain of page id, K row and R_k row for its 11 to 16 tiles.
//
// Short chunks (glance kernel, where the packed kernel runs): usually one row
// tile holds the chunk, so a wave keeps that in registers instead and streams
// keys, 32 at a time in a run of its own, the next ones' K and R_k on their way
// while it works on these.  Bound by reading K (and R_k) once: one token
// of each of 16 sequences of up to 8192 rows, 8 KV heads of 128, 32.6 us (with row
// tiles through LDS 38 us).  Where the attention left its scores, a few columns of
// them, the wave sums over those instead and reads no K: 10.3 us, and 12 us more in
// the attention.
#include <algorithm>

#include "fna2_kernels.h"
#include "fna2_paged_dev.h"

namespace fna2 {

namespace {

template <int D, int RC>
struct WeighCfg {
  static constexpr int KSD = D / 16, KSR = RC / 2;
  static constexpr int QBYTES = 32 * D * 2, RBYTES = 32 * RC * 16;
  static constexpr int NQ = QBYTES / 4096;            // DMA instructions per wave and tile
  static constexpr int NR = (RBYTES / 1024 + 3) / 4;
  static constexpr int U = 2;  // row tiles between two barriers
};

template <int D, int RC, bool F16>
__device__ __forceinline__ void weigh_body(const PagedWeightsParams& W) {
  using C = WeighCfg<D, RC>;
  constexpr int U = C::U, TILE = C::QBYTES + C::RBYTES;
  __shared__ __attribute__((aligned(1024))) uint8_t st0[U * TILE], st1[U * TILE];
  __shared__ __attribute__((aligned(16))) float nl0[32 * U], nl1[32 * U];  // rows' -LSE log2(e)
  __shared__ float half[64];
  KArg P = kargs();
  const int lane = threadIdx.x & 63, wv = uni(threadIdx.x >> 6);
  const int col = lane & 31, hl = lane >> 5;
  // Keys of a workgroup: 32 for each of kw waves; with kw = 2 the waves behind
  // take the second tile of each stage.
  const int kw = W.key_waves, keys = 32 * kw;
  auto units = [&](const PagedSeq& s) { return s.lq > 0 ? (int64_t)P->H_KV * cdiv(s.lk, keys) : 0; };
  SeqWork<decltype(units)> work(P, lane, units);
  const RowLane rdl(lane);
  const int lrow = lane >> 2, lch = (lane & 3) ^ swz4(lane >> 2);
  // DMA slot wv + 4 j of a tile: column group (wv + 4 j) / 2, rows 16 (wv % 2) ..
  const int drow = 16 * (wv & 1) + lrow;  // the row this lane fetches
  const uint32_t qxor = P->qa < 0.f ? 0x80008000u : 0u;
  const uint32_t qand = P->qa == 0.f ? 0u : 0xffffffffu;
  const float c2 = P->c2;

  for (int64_t id = blockIdx.x; id < work.total; id += gridDim.x) {
    P = kargs();
    const PagedAt at = work.seek(P, lane, id);
    const PagedSeq e = at.s;
    const int nkb = cdiv(e.lk, keys);
    const int kvh = uni((int)div64(at.rem, nkb));
    const int kb = keys * (int)(at.rem - (int64_t)kvh * nkb);
    const int k0 = kb + 32 * (wv & (kw - 1)), key = k0 + col, off = e.off;
    const bool causal = P->causal != 0;
    int page = -1, r = 0;
    if (key < e.lk && key < W.cap) {
      const int pg = page_of(P->ps_mul, P->ps_shift, key);
      page = P->table[(int64_t)at.b * P->tstride + pg];
      r = key - pg * P->ps;
      if ((uint32_t)page >= (uint32_t)P->npages) page = -1;
    }
    const bool here = page >= 0;
    const bool any = __builtin_amdgcn_ballot_w64(here) != 0;
    float* wp = W.w + (int64_t)at.b * W.w_sb + (int64_t)kvh * W.w_sh + key;
    const int64_t id64 = here ? page : 0;

    // row tiles: tokens 32 tt .. of query head h of the KV head's
    const int tt0 = causal ? max(kb - off, 0) / 32 : 0;  // earlier tokens see none of the keys
    const int tt1 = cdiv(e.lq, 32), n = P->group * (tt1 - tt0);
    const int hkv0 = kvh * P->group, HG = P->H_G;
    const int crr = P->R / 8;
    const uint32_t qss = (uint32_t)P->q.ss * 2u, rss = (uint32_t)P->rq.ss * 2u;
    const uint8_t* const qbase = (const uint8_t*)P->q.ptr + (int64_t)e.q0 * P->q.ss * 2 + (int64_t)hkv0 * P->q.sh * 2;
    const uint8_t* const rbase = (const uint8_t*)P->rq.ptr + (int64_t)e.q0 * P->rq.ss * 2 + (int64_t)hkv0 * P->rq.sh * 2;
    const float* const lse = (const float*)P->lse.ptr + (int64_t)e.q0 * P->lse.ss + (int64_t)hkv0 * P->lse.sh;
    const int64_t qsh = P->q.sh * 2, rsh = P->rq.sh * 2, lss = P->lse.ss, lsh = P->lse.sh;
    auto issue = [&](int h, int tt, uint8_t* base) {
      const uint32_t row = 32 * tt + drow < e.lq ? drow : 0;
      const uint32_t vo = row * qss + 16u * lch;
      const auto rs = make_rsrc(qbase + (int64_t)(32 * tt) * qss + h * qsh, 0x7ffffff0u);
#pragma unroll
      for (int j = 0; j < C::NQ; ++j) {
        const int slot = wv + 4 * j;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(base + slot * 1024), 16,
                                                 vo + 64u * (slot >> 1), 0, 0, 0);
      }
      if constexpr (RC > 0) {
        const bool g = hkv0 + h < HG;
        const auto rr = make_rsrc(HG > 0 ? rbase + (int64_t)(32 * tt) * rss + h * rsh : qbase, 0x7ffffff0u);
#pragma unroll
        for (int j = 0; j < C::NR; ++j) {
          const int slot = wv + 4 * j;
          if (C::RBYTES / 1024 % 4 == 0 || slot < C::RBYTES / 1024) {
            const int c = 4 * (slot >> 1) + lch;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rr, (lds_void*)(base + C::QBYTES + slot * 1024), 16,
                g && c < crr ? row * rss + 16u * c : kOOB, 0, 0, 0);
          }
        }
      }
    };
    // A stage's U tiles; wave u loads the LSE of the u-th, and put() stores it.
    int fh = 0, ft = tt0, left = n;  // next tile to fetch; tiles not yet fetched
    float lnext = kNegInf;
    auto fill = [&](uint8_t* base) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u >= left) break;
        issue(fh, ft, base + u * TILE);
        if (wv == u) {
          const int tok = 32 * ft + col;
          lnext = tok < e.lq ? lse[(int64_t)tok * lss + fh * lsh] : kNegInf;
        }
        if (++ft == tt1) ft = tt0, ++fh;
      }
      left -= U;
    };
    auto put = [&](float* nl) {
      if (wv < U && hl == 0) nl[32 * wv + col] = lnext == kNegInf ? kNegInf : -lnext * kLog2e;
    };

    ring_barrier<0>();  // the ring's last tiles are read
    fill(st0);
    // K (B of S = Q K^T): lane holds K[key][16 s + 8 hl .. +7]
    bf16x8 kreg[C::KSD];
    {
      const uint16_t* krow = (const uint16_t*)P->k.ptr + id64 * P->k.sb + (int64_t)kvh * P->k.sh + (int64_t)r * P->k.ss;
#pragma unroll
      for (int s = 0; s < C::KSD; ++s) {
        u32x4 w = {0, 0, 0, 0};
        if (here) w = ld16(krow + 16 * s + 8 * hl);
        kreg[s] = as_bf16x8(w);
      }
    }
    float old = 0.f;
    if (here && hl == 0) old = *wp;
    put(nl0);
#pragma unroll
    for (int s = 0; s < C::KSD; ++s) {
      u32x4 w = as_u32x4(kreg[s]);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (w[i] & qand) ^ qxor;
      kreg[s] = as_bf16x8(w);
    }

    bf16x8 rkreg[C::KSR > 0 ? C::KSR : 1];
    float bh = 0.f;
    float sum = 0.f;
    int h = 0, tt = tt0, held = -1;  // the tile at hand; the head whose R_k is held
    auto step = [&](int t, const uint8_t* cur, const float* nl, uint8_t* nxt, float* nl_nxt) {
      ring_barrier<0>();
      const bool more = left > 0;
      if (more) fill(nxt);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (t + u < n && (kw == 4 || u == wv >> 1)) {
          if constexpr (RC > 0) {
            if (h != held) {
              held = h;
              bh = hkv0 + h < HG ? P->gs[hkv0 + h] / P->c : 0.f;
              const uint16_t* rrow = (const uint16_t*)P->rk.ptr + id64 * P->rk.sb + (int64_t)(hkv0 + h) * P->rk.sh + (int64_t)r * P->rk.ss;
#pragma unroll
              for (int s = 0; s < C::KSR; ++s) {
                const int c = 2 * s + hl;
                u32x4 w = {0, 0, 0, 0};
                if (here && hkv0 + h < HG && c < crr) w = ld16(rrow + 8 * c);
                rkreg[s] = as_bf16x8(w);
              }
            }
          }
          if (any && (!causal || k0 <= off + 32 * tt + 31)) {
            f32x16 acc = f32x16{};
            if constexpr (RC > 0) {
#pragma unroll
              for (int s = 0; s < C::KSR; ++s)
                acc = mfma32(row_read<32>(cur + u * TILE + C::QBYTES, rdl, 0, s), rkreg[s], acc);
#pragma unroll
              for (int v = 0; v < 16; ++v) acc[v] *= bh;
            }
#pragma unroll
            for (int s = 0; s < C::KSD; ++s)
              acc = mfma_e<F16>(row_read<32>(cur + u * TILE, rdl, 0, s), kreg[s], acc);
            float part = 0.f;
            if (causal && k0 + 31 > off + 32 * tt) {
              const int first = key - off - 32 * tt;  // the first row that sees the key
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const f32x4_t a = *(const f32x4_t*)(nl + 32 * u + 8 * q + 4 * hl);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[4 * q + i], c2, a[i]));
                  part += 8 * q + 4 * hl + i >= first && a[i] != kNegInf ? p : 0.f;
                }
              }
            } else {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const f32x4_t a = *(const f32x4_t*)(nl + 32 * u + 8 * q + 4 * hl);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  part += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[4 * q + i], c2, a[i]));
              }
            }
            sum += part;
          }
        }
        if (++tt == tt1) tt = tt0, ++h;
      }
      if (more) put(nl_nxt);
    };
    for (int t = 0; t < n; t += 2 * U) {
      step(t, st0, nl0, st1, nl1);
      if (t + U < n) step(t + U, st1, nl1, st0, nl0);
    }
    sum = wave_pair_sum(sum);
    if (kw == 2) {
      // (the next block's first barrier lies between these reads and its writes)
      if (wv >= 2 && hl == 0) half[32 * (wv & 1) + col] = sum;
      __syncthreads();
      if (wv >= 2) continue;
      sum += half[32 * wv + col];
    }
    if (here && hl == 0) *wp = old + sum;
  }
}

// Workgroups of a CU, by the registers that K and R_k take.  (Four at d = 128, R =
// 32 spill: 31 us become 36.)
constexpr int weigh_occ(int D, int rc) { return rc == 0 || (D == 64 && rc <= 4) ? 4 : 3; }

#define FNA2_WEIGH(D, RC)                                                                           \
  __global__ __launch_bounds__(256, weigh_occ(D, RC)) void paged_weigh_d##D##_c##RC(const PagedWeightsParams W) {  \
    weigh_body<D, RC, false>(W);                                                                    \
  }                                                                                                 \
  __global__ __launch_bounds__(256, weigh_occ(D, RC)) void paged_weigh_d##D##_c##RC##_f16(const PagedWeightsParams W) { \
    weigh_body<D, RC, true>(W);                                                                     \
  }
FNA2_WEIGH(64, 0)
FNA2_WEIGH(64, 4)
FNA2_WEIGH(64, 8)
FNA2_WEIGH(128, 0)
FNA2_WEIGH(128, 4)
FNA2_WEIGH(128, 8)
#undef FNA2_WEIGH


template <int D, int RC, bool F16>
__device__ __forceinline__ void glance_body(const PagedWeightsParams& W) {
  constexpr int KSD = D / 16, KSR = RC / 2;
  KArg P = kargs();
  const int lane = threadIdx.x, col = lane & 31, hl = lane >> 5;
  const int gsub = P->gsub, tpt = P->tpt, nsub = P->nsub;
  const int crr = P->R / 8;
  if (P->npages <= 0) return;
  const int tk = small_div(col, gsub), hc = col - tk * gsub;  // the row that this lane loads
  int64_t left;
  int b, kvh, step, steps;
  PagedSeq e;
  auto steps_of = [](const PagedSeq& s) { return s.lq > 0 ? cdiv(s.lk, 32) : 0; };
  {
    auto units = [&](const PagedSeq& s) { return (int64_t)P->H_KV * steps_of(s); };
    SeqWork<decltype(units)> work(P, lane, units);
    const int64_t per = run_units(P, work.total, 1);
    const int64_t u = (int64_t)blockIdx.x * per;
    left = min(work.total - u, per);
    if (left <= 0) return;
    const PagedAt at = work.seek(P, lane, u);
    b = at.b;
    e = at.s;
    steps = steps_of(e);
    kvh = uni((int)div64(at.rem, steps));
    step = uni((int)(at.rem - (int64_t)kvh * steps));
  }
  const uint32_t qxor = P->qa < 0.f ? 0x80008000u : 0u;
  const uint32_t qand = P->qa == 0.f ? 0u : 0xffffffffu;
  while (true) {
    P = kargs();
    const bool causal = P->causal != 0;
    const float c2 = P->c2;
    const int s1 = (int)min((int64_t)steps, step + left);
    const int off = e.off, ps = P->ps, npages = P->npages, HG = P->H_G, group = P->group;
    const int h00 = kvh * group, nct = cdiv(e.lq, tpt), n = nsub * nct;
    const int last = min(32 * s1, e.lk) - 1;
    const int* trow = P->table + (int64_t)b * P->tstride;
    float* const wrow = W.w + (int64_t)b * W.w_sb + (int64_t)kvh * W.w_sh;
    const uint16_t* const kpool = (const uint16_t*)P->k.ptr + (int64_t)kvh * P->k.sh;
    const uint16_t* const rpool = (const uint16_t*)P->rk.ptr;
    const int64_t ksb = P->k.sb, kss = P->k.ss, rsb = P->rk.sb, rss = P->rk.ss, rsh = P->rk.sh;

    // The attention has left the scores: four steps at a time, the columns in
    // turn between the halves of the wave.
    if (P->scores && e.lq <= tpt) {
      const int64_t srows = P->srows;
      for (int s = step; s < s1; s += 4) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f}, old[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int key = 32 * (s + k) + col;
          old[k] = hl == 0 && key <= last && key < W.cap ? wrow[key] : 0.f;
        }
        for (int sub = 0; sub < nsub; ++sub) {
          const float* sc = paged_scores(P, b, kvh * nsub + sub) + 32 * s + col;
          const int nh = min(gsub, group - sub * gsub);
#pragma unroll 2
          for (int c = hl; c < e.lq * gsub; c += 2) {
            const int t = small_div(c, gsub), h = c - t * gsub;
            if (h >= nh) continue;
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = s + k < s1 ? sc[c * srows + 32 * k] : kNegInf;
            const float l = ((const float*)P->lse.ptr)[(int64_t)(e.q0 + t) * P->lse.ss +
                                                       (int64_t)(h00 + sub * gsub + h) * P->lse.sh];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              sum[k] += l == kNegInf ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(x[k], c2, -l * kLog2e));
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int key = 32 * (s + k) + col;
          sum[k] = wave_pair_sum(sum[k]);
          if (hl == 0 && key <= last && key < W.cap) wrow[key] = old[k] + sum[k];
        }
      }
    } else {
      // Row tile i: Q (A of S = Q K^T), and for the rows of this lane's registers
      // -LSE log2(e) and graph scale.
      bf16x8 qreg[KSD + KSR];
      float nl[16], bh[KSR > 0 ? 16 : 1];
      int h0 = h00, gg = 0, lim0 = 0;
      auto rows = [&](int i) {
        const int sub = nsub == 1 ? 0 : i / nct, t0 = (i - sub * nct) * tpt;
        h0 = h00 + sub * gsub;
        gg = KSR > 0 ? min(max(min(HG - h0, group - sub * gsub), 0), gsub) : 0;
        lim0 = off + t0;
        const bool on = tk < tpt && t0 + tk < e.lq && hc < min(gsub, group - sub * gsub);
        const int64_t t = e.q0 + t0 + (on ? tk : 0);
        const int hr = on ? hc : 0, h = h0 + hr;
        const uint16_t* qrow = (const uint16_t*)P->q.ptr + t * P->q.ss + (int64_t)h * P->q.sh + 8 * hl;
#pragma unroll
        for (int s = 0; s < KSD; ++s) {
          u32x4 w = ld16(qrow + 16 * s);
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = (w[k] & qand) ^ qxor;
          qreg[s] = as_bf16x8(w);
        }
        if constexpr (KSR > 0) {
          const uint16_t* rrow = (const uint16_t*)P->rq.ptr + t * P->rq.ss + (int64_t)h * P->rq.sh;
#pragma unroll
          for (int s = 0; s < KSR; ++s) {
            const int c = 2 * s + hl - hr * crr;  // this row's own head's chunks only
            u32x4 w = {0, 0, 0, 0};
            if (hr < gg && c >= 0 && c < crr) w = ld16(rrow + 8 * c);
            qreg[KSD + s] = as_bf16x8(w);
          }
        }
        float l = kNegInf, g = 0.f;
        if (on) l = ((const float*)P->lse.ptr)[t * P->lse.ss + (int64_t)h * P->lse.sh];
        if (KSR > 0 && hr < gg) g = P->gs[h] / P->c;
        l = l == kNegInf ? kNegInf : -l * kLog2e;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int row = 8 * (v >> 2) + 4 * hl + (v & 3);
          nl[v] = __shfl(l, row);
          if constexpr (KSR > 0) bh[v] = __shfl(g, row);
        }
      };
      // The page of this lane's key of step s, and the key's row in it.  A key that is
      // not there reads the pool's first row instead, and its sum is dropped.
      auto find = [&](int s, int& id, int& row) {
        const int key = 32 * s + col;
        id = -1, row = 0;
        if (key <= last && key < W.cap) {
          const int pg = page_of(P->ps_mul, P->ps_shift, key);
          id = trow[pg];
          row = key - pg * ps;
        }
      };
      bf16x8 k[KSD], rk[KSR > 0 ? KSR : 1];
      float old = 0.f;
      bool here = false;
      auto load_k = [&](int s, int id, int row) {
        here = (uint32_t)id < (uint32_t)npages;
        const uint16_t* p = kpool + (here ? (int64_t)id * ksb + (int64_t)row * kss : 0) + 8 * hl;
#pragma unroll
        for (int i = 0; i < KSD; ++i) k[i] = as_bf16x8(ld16(p + 16 * i));
        here = here && hl == 0;
        if (here) old = wrow[32 * s + col];
      };
      auto load_r = [&](int id, int row) {
        if constexpr (KSR > 0) {
          if (gg > 0) {
            const bool in = (uint32_t)id < (uint32_t)npages;
            const uint16_t* p = rpool + (in ? (int64_t)id * rsb + (int64_t)row * rss : 0) + (int64_t)h0 * rsh;
            int cr = crr;
            asm volatile("" : "+s"(cr));  // (offsets found again each time, not kept)
#pragma unroll
            for (int s = 0; s < KSR; ++s) {
              int c = 2 * s + hl;
              c = c < gg * cr ? c : 0;  // (R_q's chunk is zero there)
              const int hh = small_div(c, cr);
              rk[s] = as_bf16x8(ld16(p + (int64_t)hh * rsh + 8 * (c - hh * cr)));
            }
          }
        }
      };

      // The sum of this lane's rows of tile `i` for key 32 s + col, a product at a
      // time: each head meets its own ranks only (in the tile an infinity or a NaN in
      // another head's R_k comes as NaN, times a zero of R_q's).
      auto one_by_one = [&](int s) {
        int id, row;
        find(s, id, row);
        const int key = 32 * s + col, t0 = lim0 - off, hs = min(gsub, group - (h0 - h00));
        float part = 0.f;
        if ((uint32_t)id >= (uint32_t)npages) return part;
        auto dot = [](auto f16, const uint16_t* x, const uint16_t* y, int n) {
          constexpr bool F = decltype(f16)::value;
          float d = 0.f;
#pragma unroll 1
          for (int c = 0; c < n; c += 8) {
            const u32x4 a = ld16(x + c), b = ld16(y + c);
#pragma unroll
            for (int k = 0; k < 4; ++k) d += elt_lo<F>(a[k]) * elt_lo<F>(b[k]) + elt_hi<F>(a[k]) * elt_hi<F>(b[k]);
          }
          return d;
        };
#pragma unroll 1
        for (int v = 0; v < 16; ++v) {
          const int rw = 8 * (v >> 2) + 4 * hl + (v & 3), t = small_div(rw, gsub), h = rw - t * gsub;
          if (t >= tpt || t0 + t >= e.lq || h >= hs || (causal && key > lim0 + t)) continue;
          const int64_t tok = e.q0 + t0 + t;
          const float l = ((const float*)P->lse.ptr)[tok * P->lse.ss + (int64_t)(h0 + h) * P->lse.sh];
          if (l == kNegInf) continue;
          float x = P->qa * dot(std::integral_constant<bool, F16>{}, (const uint16_t*)P->q.ptr + tok * P->q.ss + (int64_t)(h0 + h) * P->q.sh,
                                kpool + (int64_t)id * ksb + (int64_t)row * kss, D);
          if (h < gg)
            x += P->gs[h0 + h] / P->c *
                 dot(std::false_type{}, (const uint16_t*)P->rq.ptr + tok * P->rq.ss + (int64_t)(h0 + h) * P->rq.sh,
                     rpool + (int64_t)id * rsb + (int64_t)row * rss + (int64_t)(h0 + h) * rsh, P->R);
          part += __builtin_amdgcn_exp2f(__builtin_fmaf(x, c2, -l * kLog2e));
        }
        return part;
      };

      int id, row, id1, row1, held = -1;
      find(step, id, row);
      load_k(step, id, row);
      find(step + 1, id1, row1);
      float sum = 0.f;
      for (int s = step, i = 0; s < s1;) {
        if (held != i) {
          rows(i);
          load_r(id, row);
          held = i;
        }
        f32x16 acc = f32x16{};
        if constexpr (KSR > 0) {
          if (gg > 0) {
#pragma unroll
            for (int j = 0; j < KSR; ++j) acc = mfma32(qreg[KSD + j], rk[j], acc);
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[v] *= bh[v];
          }
        }
#pragma unroll
        for (int j = 0; j < KSD; ++j) acc = mfma_e<F16>(qreg[j], k[j], acc);
        // The next step's rows, into the registers that are read.
        const bool put = here;
        const float before = old;
        const int s0 = s;
        const bool turn = i + 1 == n;
        if (turn) {
          ++s, i = 0;
          if (s < s1) {
            id = id1, row = row1;
            load_k(s, id, row);
            if (n == 1) load_r(id, row);
            find(s + 1, id1, row1);
          }
        } else {
          ++i;
        }
        float part = 0.f;
        if (causal && 32 * s0 + 31 > lim0) {
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int rw = 8 * (v >> 2) + 4 * hl + (v & 3);
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[v], c2, nl[v]));
            part += 32 * s0 + col <= lim0 + small_div(rw, gsub) && nl[v] != kNegInf ? p : 0.f;
          }
        } else {
#pragma unroll
          for (int v = 0; v < 16; ++v) part += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[v], c2, nl[v]));
        }
        if constexpr (KSR > 0) {
          if (__builtin_expect(gg > 0 && __builtin_amdgcn_ballot_w64(part != part) != 0, 0))
            if (part != part) part = one_by_one(s0);
        }
        sum += part;
        if (turn) {
          sum = wave_pair_sum(sum);
          if (put) wrow[32 * s0 + col] = before + sum;
          sum = 0.f;
        }
      }
    }
    left -= s1 - step;
    if (left <= 0) return;
    step = 0;
    if (++kvh == P->H_KV) {
      kvh = 0;
      do {
        e = paged_seq_uniform(P, ++b);
        steps = steps_of(e);
      } while (steps == 0 && b + 1 < P->N);
    }
  }
}

// Waves per SIMD, by the registers that a tile of Q, R_q and of K, R_k takes.
constexpr int glance_occ(int D, int rc) {
  return rc > 16 ? 1 : D == 64 ? (rc == 0 ? 4 : rc <= 8 ? 3 : 2) : rc == 0 ? 3 : 2;
}

#define FNA2_GLANCE(D, RC)                                                                              \
  __global__ __launch_bounds__(64, glance_occ(D, RC)) void paged_glance_d##D##_c##RC(const PagedWeightsParams W) { \
    glance_body<D, RC, false>(W);                                                                       \
  }                                                                                                     \
  __global__ __launch_bounds__(64, glance_occ(D, RC)) void paged_glance_d##D##_c##RC##_f16(const PagedWeightsParams W) { \
    glance_body<D, RC, true>(W);                                                                        \
  }
FNA2_GLANCE(64, 0)
FNA2_GLANCE(64, 4)
FNA2_GLANCE(64, 8)
FNA2_GLANCE(64, 16)
FNA2_GLANCE(64, 32)
FNA2_GLANCE(128, 0)
FNA2_GLANCE(128, 4)
FNA2_GLANCE(128, 8)
FNA2_GLANCE(128, 16)
FNA2_GLANCE(128, 32)
#undef FNA2_GLANCE

}  // namespace

int paged_weigh_per_cu(int D, int rc) { return weigh_occ(D, rc); }

hipError_t launch_paged_weights(const PagedWeightsParams& W, int rc, hipStream_t s) {
  const PagedParams& P = W.p;
  void (*k)(const PagedWeightsParams) = nullptr;
#define FNA2_WEIGH_OF(D, RC) (P.f16 ? paged_weigh_d##D##_c##RC##_f16 : paged_weigh_d##D##_c##RC)
  if (P.D == 64)
    k = rc == 0 ? FNA2_WEIGH_OF(64, 0) : rc == 4 ? FNA2_WEIGH_OF(64, 4) : rc == 8 ? FNA2_WEIGH_OF(64, 8) : nullptr;
  if (P.D == 128)
    k = rc == 0 ? FNA2_WEIGH_OF(128, 0) : rc == 4 ? FNA2_WEIGH_OF(128, 4) : rc == 8 ? FNA2_WEIGH_OF(128, 8) : nullptr;
#undef FNA2_WEIGH_OF
  if (!k) return hipErrorInvalidValue;
  hipLaunchKernelGGL(k, dim3((uint32_t)W.grid), dim3(256), 0, s, W);
  return hipGetLastError();
}

int paged_glance_per_cu(int D, int rc) { return 4 * glance_occ(D, rc); }

hipError_t launch_paged_glance(const PagedWeightsParams& W, int rc, hipStream_t s) {
  const PagedParams& P = W.p;
  void (*k)(const PagedWeightsParams) = nullptr;
#define FNA2_GLANCE_OF(D, RC) (P.f16 ? paged_glance_d##D##_c##RC##_f16 : paged_glance_d##D##_c##RC)
  if (P.D == 64)
    k = rc == 0 ? FNA2_GLANCE_OF(64, 0) : rc == 4 ? FNA2_GLANCE_OF(64, 4) : rc == 8 ? FNA2_GLANCE_OF(64, 8)
      : rc == 16 ? FNA2_GLANCE_OF(64, 16) : rc == 32 ? FNA2_GLANCE_OF(64, 32) : nullptr;
  if (P.D == 128)
    k = rc == 0 ? FNA2_GLANCE_OF(128, 0) : rc == 4 ? FNA2_GLANCE_OF(128, 4) : rc == 8 ? FNA2_GLANCE_OF(128, 8)
      : rc == 16 ? FNA2_GLANCE_OF(128, 16) : rc == 32 ? FNA2_GLANCE_OF(128, 32) : nullptr;
#undef FNA2_GLANCE_OF
  if (!k) return hipErrorInvalidValue;
  hipLaunchKernelGGL(k, dim3((uint32_t)W.grid), dim3(64), 0, s, W);
  return hipGetLastError();
}

}  // namespace fna2
