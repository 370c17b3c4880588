// fna2_paged_tile.hip — attention of long chunks of new tokens over a paged cache.
//
// The operator of fna2_paged_attn.hip for chunks whose (token, head) pairs
// fill more than one column tile.  A workgroup is 4 waves that share the K
// and V tiles of one KV head; each wave has 32 tokens of one query head, hw of
// the KV head's in all: (tokens, heads) = (128, 1), (64, 2) or (32, 4).  With
// grouped heads a tile of 4 heads reads K and V once for them all however short the chunk.
// The waves compute as the forward kernel's do: S^T = Ka Qa^T with the rank
// chain first, the lazily rescaled online softmax by column, O^T += V^T P^T with
// P in the element type.
//
// Work and pages as in fna2_paged_attn.hip: the tiles' key steps laid end to
// end, an equal run for each resident workgroup, parts of cut tiles joined by
// a second kernel.  Workgroups whose runs are neighbours share an XCD's L2.  A
// wave DMAs the same 16 rows of every K, V and R_k tile, so it follows one
// page.
//
// Bound by the matrix cores and, between their products, by the exponentials and the
// rounding of P: 1024 tokens over 16,384 rows, 32 heads over 8 KV heads of 128, R = 64,
// 346 to 362 us with the merge of the parts, up to 0.96 10^15 operations a second of the
// 1.23 10^15 of a large matrix product (matrix cores 52% of the cycles, at the 1.85 GHz
// that the power leaves; spread evenly at 2.4 GHz products 132 us, other vector
// instructions 125).  A step of 256 tokens beside 32 decoding sequences over 4096 rows
// is bound by reading K, V and R_k (5.7 TB/s): 123 us and 12 us.  At d = 64, R = 16
// (2 chunks of 509 tokens over 7001 rows, 16 heads) by neither, 48 us and 9: products
// 10 us, vector instructions 19, waves waiting 37% of their time on two workgroups a CU,
// and the ranks padded to 32.  P is rounded once, off by
// half a step (bf16 2^-8) of each p at most, on top of the output's own rounding (1.4 times
// the error of an output alone); in two parts the products with V would double.
#include <algorithm>

#include "fna2_kernels.h"
#include "fna2_paged_dev.h"

namespace fna2 {

namespace {

template <int D, int RPL, int HW>
struct TileCfg {
  // keys per step: 64 at d = 64 while two stages then leave room for three
  // workgroups
  static constexpr int BN = D == 128 || HW * RPL >= 128 ? 32 : 64;
  static constexpr int KSD = D / 16, KSR = RPL / 16;
  static constexpr int KBYTES = BN * D * 2;
  static constexpr int RHEAD = BN * RPL * 2;  // one head's R_k tile
  static constexpr int RBYTES = HW * RHEAD;
  static constexpr int STAGE = 2 * KBYTES + RBYTES;
  static constexpr int G = BN / 16;           // 16-row groups of a tile: a wave loads group wv % G
  static constexpr int NK = KBYTES / 4096;    // DMA instructions of a K tile per wave
  static constexpr int NR = (RBYTES / 1024 + 3) / 4;
  static constexpr bool PIPE = RPL <= 32;
  static constexpr int A1 = PIPE ? 2 : 1, A2 = PIPE ? 2 : 1;  // operand reads ahead of the MFMAs
};

// Workgroup -> run: neighbouring runs on one XCD (workgroups go to the 8 in
// turn).
__device__ __forceinline__ int run_of(int wg, int n) {
  return n % 8 == 0 ? (wg & 7) * (n >> 3) + (wg >> 3) : wg;
}

template <int D, int RPL, int HW, bool F16>
__device__ __forceinline__ void tile_body() {
  KArg P = kargs();
  using C = TileCfg<D, RPL, HW>;
  constexpr int BN = C::BN;
  __shared__ __attribute__((aligned(1024))) uint8_t stage0[C::STAGE];
  __shared__ __attribute__((aligned(1024))) uint8_t stage1[C::STAGE];
  __shared__ volatile int odd_flag;  // a V tile holds infinities or NaN (see fna2_paged_dev.h)
  const int lane = threadIdx.x & 63, wv = uni(threadIdx.x >> 6);
  const int l32 = lane & 31, hl = lane >> 5;
  if (threadIdx.x == 0) odd_flag = 0;  // (read behind a barrier of the first step at the earliest)
  const int hw = RPL > 0 ? HW : P->hw;  // (without ranks a tile's heads do not show in its layout)
  const int TB = 128 / hw;
  const int hblk = cdiv(P->group, hw);  // blocks of heads of a KV head

  const int run = run_of(blockIdx.x, gridDim.x);
  int64_t left, per;  // units of this run still to do, and of a run
  int b, hb, qt, s0;
  PagedSeq e;
  auto cut = [&](int seq, int head, int tile, int parts) {
    if (threadIdx.x == 0) P->cuts[run] = PagedCut{seq, head, tile, parts};
  };
  {
    auto units = [&](const PagedSeq& s) { return TilePlan::units(P, s); };
    SeqWork<decltype(units)> work(P, lane, units);
    per = run_units(P, work.total, P->min_steps);
    const int64_t u = (int64_t)run * per;
    left = min(work.total - u, per);
    if (left <= 0) {
      cut(0, 0, 0, 0);
      return;
    }
    const PagedAt at = work.seek(P, lane, u);
    b = at.b;
    e = at.s;
    const int64_t hu = TilePlan::head_units(P, e);
    hb = uni((int)div64(at.rem, hu));
    int64_t r = at.rem - hb * hu;
    qt = uni(TilePlan::find(P, e, r));
    s0 = uni((int)r);
  }

  const TrLane tl(lane);
  const RowLane rdl(lane);
  const int rg = wv % C::G;  // this wave's row group of a tile
  const uint32_t krb = (uint32_t)P->k.ss * 2u, vrb = (uint32_t)P->v.ss * 2u;
  const int lrow = lane >> 2, lch = (lane & 3) ^ swz4(lane >> 2);
  // K / V DMA instruction j of this wave: slot wv + 4 j = column group * G + rg
  const uint32_t kvo = (uint32_t)lrow * krb + 16u * (lch + 4 * (wv / C::G));
  const uint32_t vvo = (uint32_t)lrow * vrb + 16u * (lch + 4 * (wv / C::G));
  constexpr uint32_t kCol = 64u * (4 / C::G);  // bytes between a wave's instructions

  while (true) {
    P = kargs();
    const bool causal = P->causal != 0;
    const int steps = TilePlan::steps(P, e, qt);
    const int s1 = (int)min((int64_t)steps, s0 + left);
    const int kvh = hb / hblk, h_in = (hb - kvh * hblk) * hw + wv % hw;
    const int h = kvh * P->group + min(h_in, P->group - 1);
    const int off = e.off;
    const int tok0 = qt * TB + 32 * (wv / hw);  // this wave's first token
    const bool idle = tok0 >= e.lq || h_in >= P->group;
    const int tok_last = min(tok0 + 31, e.lq - 1);
    const int tok = tok0 + l32;
    const bool live = !idle && tok < e.lq;
    const bool graph = RPL > 0 && h < P->H_G;
    const float bh = uni_f(graph ? *const_space(P->gs + h) / P->c : 0.f);
    const int k_end = min(32 * s1, e.lk);  // rows of this run's part
    const int lim = min(causal ? off + tok : e.lk - 1, k_end - 1);  // last row this column sees
    const int lim_any = causal ? off + tok_last : e.lk - 1;  // some of them see
    const int* trow = P->table + (int64_t)b * P->tstride;
    const int ps = P->ps, npages = P->npages;
    const float c2 = P->c2;
    const uint16_t* const kpool = (const uint16_t*)P->k.ptr + (int64_t)kvh * P->k.sh;
    const uint16_t* const vpool = (const uint16_t*)P->v.ptr + (int64_t)kvh * P->v.sh;
    const int64_t ksb = P->k.sb, vsb = P->v.sb;
    const uint16_t* const rpool = (const uint16_t*)P->rk.ptr;
    const int64_t rsb = P->rk.sb, rsh = P->rk.sh;
    const uint32_t rrb = (uint32_t)P->rk.ss * 2u;
    const int rchunks = P->R / 8, group = P->group, HG = P->H_G;

    // Page and row within it of this wave's row group of the next tile.
    PageIds ids;
    ids.row = trow;
    ids.last = k_end > 0 ? page_of(P->ps_mul, P->ps_shift, k_end - 1) : -1;
    int row = 32 * s0 + 16 * rg;
    int page = page_of(P->ps_mul, P->ps_shift, row), poff = row - page * ps;
    // Rows of the part in pages that are not there (rare) are masked.
    bool gone = false;
    {
      const int first = page_of(P->ps_mul, P->ps_shift, 32 * s0);
      for (int p = first; p <= ids.last; p += 64) {
        ids.load(lane, p);
        gone |= (uint32_t)ids.ids >= (uint32_t)npages;
      }
      gone = __builtin_amdgcn_ballot_w64(gone) != 0;
      if (ids.last - first >= 64 || ids.last < first) ids.load(lane, first);
    }
    auto issue = [&](uint8_t* base) {
      const int pid = row < k_end ? ids.at(lane, page) : -1;
      const bool in = (uint32_t)pid < (uint32_t)npages;
      const int rows = in ? clamp_rows(k_end - row, 16) : 0;
      const int64_t id = in ? pid : 0;
      const auto rk_ = make_rsrc((const uint8_t*)(kpool + id * ksb) + (uint64_t)(uint32_t)poff * krb,
                                 (uint32_t)rows * krb);
      const auto rv_ = make_rsrc((const uint8_t*)(vpool + id * vsb) + (uint64_t)(uint32_t)poff * vrb,
                                 (uint32_t)rows * vrb);
#pragma unroll
      for (int j = 0; j < C::NK; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rk_, (lds_void*)(base + (wv + 4 * j) * 1024), 16,
                                                 kvo + kCol * j, 0, 0, 0);
      if constexpr (RPL > 0) {
        // slot i = wv + 4 j of the heads' R_k tiles: head i / (slots a head),
        // column group, row group rg
        constexpr int PH = C::RHEAD / 1024;
#pragma unroll
        for (int j = 0; j < C::NR; ++j) {
          const int i = wv + 4 * j;
          if (C::RBYTES / 1024 % 4 == 0 || i < C::RBYTES / 1024) {
            const int hh = i / PH, cg = (i % PH) / C::G;
            const int hq = kvh * group + (hb - kvh * hblk) * HW + hh;
            const bool on = hq < HG && (hb - kvh * hblk) * HW + hh < group;
            const uint8_t* rp = (const uint8_t*)(rpool + id * rsb + (int64_t)(on ? hq : 0) * rsh) +
                                (uint64_t)(uint32_t)poff * rrb;
            const int c = 4 * cg + lch;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                make_rsrc(rp, on ? (uint32_t)rows * rrb : 0u),
                (lds_void*)(base + C::KBYTES + i * 1024), 16,
                c < rchunks ? (uint32_t)lrow * rrb + 16u * c : kOOB, 0, 0, 0);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < C::NK; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rv_, (lds_void*)(base + C::KBYTES + C::RBYTES + (wv + 4 * j) * 1024), 16,
            vvo + kCol * j, 0, 0, 0);
      row += BN;
      poff += BN;
      while (poff >= ps) {
        poff -= ps;
        ++page;
      }
    };

    issue(stage0);
    __builtin_amdgcn_sched_barrier(0);

    // Query operand (B of S^T): lane holds Qa[tok][16 s + 8 hl .. +7].
    bf16x8 qreg[C::KSD + C::KSR];
    {
      const int64_t t = e.q0 + (live ? tok : 0);
      const uint16_t* qrow = (const uint16_t*)P->q.ptr + t * P->q.ss + (int64_t)h * P->q.sh;
      const uint32_t qxor = P->qa < 0.f ? 0x80008000u : 0u;
      const uint32_t qand = P->qa == 0.f ? 0u : 0xffffffffu;
#pragma unroll
      for (int s = 0; s < C::KSD; ++s) {
        u32x4 w = {0, 0, 0, 0};
        if (live) w = ld16(qrow + 16 * s + 8 * hl);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (w[i] & qand) ^ qxor;
        qreg[s] = as_bf16x8(w);
      }
      if constexpr (C::KSR > 0) {
        const uint16_t* rrow = (const uint16_t*)P->rq.ptr + t * P->rq.ss + (int64_t)h * P->rq.sh;
#pragma unroll
        for (int s = 0; s < C::KSR; ++s) {
          u32x4 w = {0, 0, 0, 0};
          if (live && graph && 16 * s + 8 * hl < P->R) w = ld16(rrow + 16 * s + 8 * hl);
          qreg[C::KSD + s] = as_bf16x8(w);
        }
      }
    }

    f32x16 oacc[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) oacc[d] = f32x16{};
    float m_i = kNegInf, l_i = 0.f;

    auto step = [&](auto masks, int kbase, uint8_t* cur, uint8_t* nxt) {
      constexpr bool MASK = decltype(masks)::value;
      ring_barrier<0>();
      if (kbase + BN < k_end) issue(nxt);
      __builtin_amdgcn_sched_barrier(0);
      if (MASK && causal && kbase + BN - 1 > off + qt * TB) {  // (the same for all four waves)
        uint8_t* v = cur + C::KBYTES + C::RBYTES;
        if (tile_odd<C::KBYTES / 4096, F16>(v + wv * (C::KBYTES / 4), lane)) odd_flag = 1;
        ring_barrier<63>();
        if (__builtin_expect(odd_flag, 0)) {
          if (!idle) add_odd<D, BN, F16>(v, kbase, lim, hl, oacc);
          ring_barrier<63>();
          tile_clean<C::KBYTES / 4096, F16>(v + wv * (C::KBYTES / 4), lane);
          odd_flag = 0;
          ring_barrier<63>();
        }
      }
      if (idle || (MASK && kbase > lim_any)) return;
      const uint8_t* kl = cur;
      const uint8_t* rl = kl + C::KBYTES + (HW > 1 ? (wv % HW) * C::RHEAD : 0);
      const uint8_t* vl = kl + C::KBYTES + C::RBYTES;
      f32x16 sacc[BN / 32];
#pragma unroll
      for (int kb2 = 0; kb2 < BN / 32; ++kb2) {
        f32x16 acc = f32x16{};
        bf16x8 kr[C::A1];
        if constexpr (C::PIPE) {
#pragma unroll
          for (int s = 0; s < C::A1; ++s) kr[s] = row_read<BN>(kl, rdl, kb2 * 32, s);
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (C::KSR > 0) {
#pragma unroll
          for (int s = 0; s < C::KSR; ++s)
            acc = mfma32(row_read<BN>(rl, rdl, kb2 * 32, s), qreg[C::KSD + s], acc);
          acc *= here_s(bh);
        }
        if constexpr (C::PIPE) {
#pragma unroll
          for (int s = 0; s < C::KSD; ++s) {
            acc = mfma_e<F16>(kr[s % C::A1], qreg[s], acc);
            if (s + C::A1 < C::KSD) kr[s % C::A1] = row_read<BN>(kl, rdl, kb2 * 32, s + C::A1);
            __builtin_amdgcn_sched_barrier(0);
          }
        } else {
#pragma unroll
          for (int s = 0; s < C::KSD; ++s)
            acc = mfma_e<F16>(row_read<BN>(kl, rdl, kb2 * 32, s), qreg[s], acc);
        }
        sacc[kb2] = acc;
      }
      if constexpr (MASK) {
#pragma unroll
        for (int kb2 = 0; kb2 < BN / 32; ++kb2)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int key = kbase + kb2 * 32 + 8 * (v >> 2) + 4 * hl + (v & 3);
            sacc[kb2][v] = key > lim ? kNegInf : sacc[kb2][v];
          }
        if (gone) {
          for (int g = 0; g < C::G; ++g) {
            const int r = kbase + 16 * g;
            if (r >= k_end || (uint32_t)uni(*const_space(trow + page_of(kargs()->ps_mul, kargs()->ps_shift, r))) < (uint32_t)npages) continue;
#pragma unroll
            for (int kb2 = 0; kb2 < BN / 32; ++kb2)
#pragma unroll
              for (int v = 0; v < 16; ++v)
                if (2 * kb2 + (v >> 3) == g) sacc[kb2][v] = kNegInf;
          }
        }
      }
      float mx = kNegInf;
#pragma unroll
      for (int kb2 = 0; kb2 < BN / 32; ++kb2)
#pragma unroll
        for (int v = 0; v < 16; ++v) mx = fmaxf(mx, sacc[kb2][v]);
      mx = wave_pair_max(mx);
      // lazy rescale, as in the forward kernel
      if (__builtin_amdgcn_ballot_w64((mx - m_i) * c2 > 8.f) != 0) {
        const float m_new = fmaxf(m_i, mx);
        const float alpha = weight2((m_i - ((m_new == kNegInf) ? 0.f : m_new)) * c2);
        l_i *= alpha;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) oacc[d] *= alpha;
        m_i = m_new;
      }
      const float nm = -((m_i == kNegInf) ? 0.f : m_i) * c2;
      float ls = 0.f;
      bf16x8 pb[BN / 16];
      u32x4 pk[BN / 16];
      auto exps = [&](int q, int i0, int i1) {
#pragma unroll
        for (int i = i0; i < i1; ++i) {
          const int v0 = 8 * (q & 1) + 2 * i;
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[q >> 1][v0], c2, nm));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[q >> 1][v0 + 1], c2, nm));
          ls += p0 + p1;
          pk[q][i] = pack_e<F16>(p0, p1);
        }
        if (i1 == 4) pb[q] = as_bf16x8(pk[q]);
      };
      constexpr int NS = BN / 16, N = NS * (D / 32), PPM = 4 / (D / 32);
      exps(0, 0, 4);
      bf16x8 vr[C::A2];
#pragma unroll
      for (int i = 0; i < C::A2; ++i)
        vr[i] = tr_operand<BN>(vl, tl, 16 * (i / (D / 32)), 32 * (i % (D / 32)));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int s = i / (D / 32), d = i % (D / 32);
        oacc[d] = mfma_e<F16>(vr[i % C::A2], pb[s], oacc[d]);
        if (i + C::A2 < N)
          vr[i % C::A2] = tr_operand<BN>(vl, tl, 16 * ((i + C::A2) / (D / 32)), 32 * ((i + C::A2) % (D / 32)));
        __builtin_amdgcn_sched_barrier(0);
        if (s + 1 < NS) exps(s + 1, PPM * d, PPM * d + PPM);
        __builtin_amdgcn_sched_barrier(0);
      }
      l_i += ls;
    };

    // The steps whose rows all tokens see, in pairs (the ring's two stages),
    // without the masks and their registers; then the others.
    int k = 32 * s0;
    if (!gone) {
      const int k_fast = min(causal ? off + qt * TB + 1 : k_end, k_end);
      for (; k + 2 * BN <= k_fast; k += 2 * BN) {
        step(std::false_type{}, k, stage0, stage1);
        step(std::false_type{}, k + BN, stage1, stage0);
      }
    }
    for (; k < k_end; k += 2 * BN) {
      step(std::true_type{}, k, stage0, stage1);
      if (k + BN < k_end) step(std::true_type{}, k + BN, stage1, stage0);
    }
    // (every wave has left the ring, and no DMA is under way, before the next
    // part's goes out)
    ring_barrier<0>();

    P = kargs();
    const float l_tot = wave_pair_sum(l_i);
    if (s0 == 0 && s1 == steps) {
      if (live) {
        const float inv = 1.f / (l_tot + 1e-6f);
        uint16_t* orow = (uint16_t*)P->o.ptr + (int64_t)(e.q0 + tok) * P->o.ss + (int64_t)h * P->o.sh;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            u32x2 val;
            val[0] = pack_e<F16>(oacc[d][4 * g] * inv, oacc[d][4 * g + 1] * inv);
            val[1] = pack_e<F16>(oacc[d][4 * g + 2] * inv, oacc[d][4 * g + 3] * inv);
            *(u32x2*)(orow + d * 32 + 8 * g + 4 * hl) = val;
          }
        if (hl == 0 && P->lse.ptr)
          ((float*)P->lse.ptr)[(int64_t)(e.q0 + tok) * P->lse.ss + (int64_t)h * P->lse.sh] =
              m_i == kNegInf ? kNegInf : m_i * P->c + __builtin_amdgcn_logf(l_tot + 1e-6f) * kLn2;
      }
    } else if (live) {
      // As the registers lie: [slot][wave][d][4][lane] of 16 bytes.
      const int64_t slot = (2 * (int64_t)run + (s0 == 0 ? 1 : 0)) * 4 + wv;
      float* arow = P->part + slot * 32 * D + 4 * lane;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f32x4_t val = {oacc[d][4 * g], oacc[d][4 * g + 1], oacc[d][4 * g + 2], oacc[d][4 * g + 3]};
          *(f32x4_t*)(arow + (d * 4 + g) * 256) = val;
        }
      if (hl == 0) *(f32x2*)(P->ml + 2 * (slot * 32 + l32)) = f32x2{m_i, l_tot};
    }

    left -= s1 - s0;
    if (left <= 0) {
      const int rest = steps - s1;
      cut(b, hb, qt, s0 == 0 && rest > 0 ? 1 + (int)div64(rest + per - 1, per) : 0);
      return;
    }
    s0 = 0;
    if (++qt * TB >= e.lq) {
      qt = 0;
      if (++hb == P->H_KV * hblk) {
        hb = 0;
        do e = paged_seq_uniform(P, ++b); while (e.lq == 0 && b + 1 < P->N);
      }
    }
  }
}

// Joins the parts of a tile that runs cut: workgroup (i, y) takes 32 features
// of the tile that run i's end cuts, four parts at a time.  A wave takes the tokens
// of one wave of the tile; where a tile has many parts (by_part) the
// workgroup does, its waves every fourth group of parts each, joined in LDS.  The
// order of the sums goes by the parts alone.
template <int D, bool F16>
__global__ __launch_bounds__(256) void paged_tile_merge_kernel(const PagedParams) {
  KArg P = kargs();
  __shared__ f32x4_t part[4][4][64];
  __shared__ float stat[4][2][32];
  const int lane = threadIdx.x & 63, own = uni(threadIdx.x >> 6);
  const bool by_part = P->merge_by_part != 0;
  const int d = blockIdx.y % (D / 32), wv = by_part ? blockIdx.y / (D / 32) : own;
  const int l32 = lane & 31, hl = lane >> 5;
  const int i0 = blockIdx.x;
  const auto rec = const_space(P->cuts + i0);
  const int n = uni(rec->parts);
  if (blockIdx.y == 0) clear_loose_tokens(P, blockIdx.x, gridDim.x);
  if (n <= 0) return;
  const int hb = uni(rec->head), qt = uni(rec->tile);
  const PagedSeq e = paged_seq_uniform(P, rec->b);
  const int hblk = cdiv(P->group, P->hw), kvh = hb / hblk, h_in = (hb - kvh * hblk) * P->hw + wv % P->hw;
  const int tok = qt * TilePlan::tokens(P) + 32 * (wv / P->hw) + l32;
  const bool live = tok < e.lq && h_in < P->group;
  const int h = kvh * P->group + h_in;
  const float c2 = P->c2;
  float M = kNegInf, L = 0.f;
  f32x4_t o[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) o[g] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;  // parts in flight
  if (live) {
    for (int j0 = by_part ? U * own : 0; j0 < n; j0 += by_part ? 4 * U : U) {
      f32x4_t x[U][4];
      f32x2 ml[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int j = min(j0 + k, n - 1);  // (past the last: not added below)
        const int64_t slot = (int64_t)(j == 0 ? 2 * i0 + 1 : 2 * (i0 + j)) * 4 + wv;
        const float* src = P->part + slot * 32 * D + d * 1024 + 4 * lane;
        ml[k] = *(const f32x2*)(P->ml + 2 * (slot * 32 + l32));
#pragma unroll
        for (int g = 0; g < 4; ++g) x[k][g] = *(const f32x4_t*)(src + g * 256);
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
        if (j0 + k >= n) break;  // (uniform)
        const float wb = weight2((ml[k][0] - ref) * c2);
        L += ml[k][1] * wb;
#pragma unroll
        for (int g = 0; g < 4; ++g) o[g] += x[k][g] * wb;
      }
      M = m;
    }
  }
  if (by_part) {
#pragma unroll
    for (int g = 0; g < 4; ++g) part[own][g][lane] = o[g];
    if (hl == 0) stat[own][0][l32] = M, stat[own][1][l32] = L;
    __syncthreads();
    if (own != 0) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float mw = stat[w][0][l32], m = fmaxf(M, mw);
      const float ref = m == kNegInf ? 0.f : m;
      const float wa = weight2((M - ref) * c2), wb = weight2((mw - ref) * c2);
      L = L * wa + stat[w][1][l32] * wb;
#pragma unroll
      for (int g = 0; g < 4; ++g) o[g] = o[g] * wa + part[w][g][lane] * wb;
      M = m;
    }
  }
  if (!live) return;
  const float inv = 1.f / (L + 1e-6f);
  uint16_t* orow = (uint16_t*)P->o.ptr + (int64_t)(e.q0 + tok) * P->o.ss + (int64_t)h * P->o.sh;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    u32x2 val;
    val[0] = pack_e<F16>(o[g][0] * inv, o[g][1] * inv);
    val[1] = pack_e<F16>(o[g][2] * inv, o[g][3] * inv);
    *(u32x2*)(orow + d * 32 + 8 * g + 4 * hl) = val;
  }
  if (d == 0 && hl == 0 && P->lse.ptr)
    ((float*)P->lse.ptr)[(int64_t)(e.q0 + tok) * P->lse.ss + (int64_t)h * P->lse.sh] =
        M == kNegInf ? kNegInf : M * P->c + __builtin_amdgcn_logf(L + 1e-6f) * kLn2;
}

// Waves per SIMD that the register budget is cut for, and workgroups of a CU.
// Three where one head's ranks or none come with d = 128: such tiles are long,
// bound by the matrix cores, and a third workgroup fills the others' waits
// (1024-token piece, rank 64, in turn: 346 us, two 351).  Two for the others: the third
// costs spilled registers (mixed step, 4 heads of rank 32: 146 us, two 133; d =
// 64, rank 16, 509-token pieces with their weights: 103, 97).  A third ring
// stage in the room that leaves: 136 and 99.
constexpr int tile_occ(int D, int RPL, int HW) { return D == 128 && (RPL == 0 || HW == 1) ? 3 : 2; }

#define FNA2_TILE(D, RPL, HW)                                                               \
  __global__ __launch_bounds__(256, tile_occ(D, RPL, HW)) void paged_tile_d##D##_r##RPL##_h##HW( \
      const PagedParams) {                                                                \
    tile_body<D, RPL, HW, false>();                                                         \
  }                                                                                         \
  __global__ __launch_bounds__(256, tile_occ(D, RPL, HW)) void                              \
      paged_tile_d##D##_r##RPL##_h##HW##_f16(const PagedParams) {                         \
    tile_body<D, RPL, HW, true>();                                                          \
  }
FNA2_TILE(64, 0, 1)
FNA2_TILE(64, 32, 1)
FNA2_TILE(64, 32, 2)
FNA2_TILE(64, 32, 4)
FNA2_TILE(64, 64, 1)
FNA2_TILE(64, 64, 2)
FNA2_TILE(64, 64, 4)
FNA2_TILE(128, 0, 1)
FNA2_TILE(128, 32, 1)
FNA2_TILE(128, 32, 2)
FNA2_TILE(128, 32, 4)
FNA2_TILE(128, 64, 1)
FNA2_TILE(128, 64, 2)
FNA2_TILE(128, 64, 4)
#undef FNA2_TILE

}  // namespace

int paged_tile_per_cu(int D, int rpl, int hw) { return tile_occ(D, rpl, hw); }

size_t paged_tile_slot(int D) { return (size_t)128 * D * 4; }

hipError_t launch_paged_tile(const PagedParams& P, int rpl, hipStream_t s) {
  void (*k)(const PagedParams) = nullptr;
#define FNA2_TILE_OF(D, RPL, HW) \
  (P.f16 ? paged_tile_d##D##_r##RPL##_h##HW##_f16 : paged_tile_d##D##_r##RPL##_h##HW)
#define FNA2_TILE_HW(D, RPL)                             \
  (P.hw == 1   ? FNA2_TILE_OF(D, RPL, 1)                 \
   : P.hw == 2 ? FNA2_TILE_OF(D, RPL, 2)                 \
   : P.hw == 4 ? FNA2_TILE_OF(D, RPL, 4)                 \
               : nullptr)
  if (P.D == 64)
    k = rpl == 0 ? FNA2_TILE_OF(64, 0, 1) : rpl == 32 ? FNA2_TILE_HW(64, 32) : FNA2_TILE_HW(64, 64);
  if (P.D == 128)
    k = rpl == 0 ? FNA2_TILE_OF(128, 0, 1) : rpl == 32 ? FNA2_TILE_HW(128, 32) : FNA2_TILE_HW(128, 64);
#undef FNA2_TILE_HW
#undef FNA2_TILE_OF
  if (!k) return hipErrorInvalidValue;
  hipLaunchKernelGGL(k, dim3((uint32_t)P.waves), dim3(256), 0, s, P);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid((uint32_t)P.waves, (uint32_t)(P.D / 32 * (P.merge_by_part ? 4 : 1)));
  void (*m)(const PagedParams) =
      P.D == 64 ? (P.f16 ? paged_tile_merge_kernel<64, true> : paged_tile_merge_kernel<64, false>)
                : (P.f16 ? paged_tile_merge_kernel<128, true> : paged_tile_merge_kernel<128, false>);
  hipLaunchKernelGGL(m, grid, dim3(256), 0, s, P);
  return hipGetLastError();
}

}  // namespace fna2
