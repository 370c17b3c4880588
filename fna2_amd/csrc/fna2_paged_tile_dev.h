// fna2_paged_tile_dev.h — the body of the tile kernels: attention of tiles of
// 128 (token, head) columns over a paged cache (fna2_paged_tile.hip), and over
// one whose groups of sequences share rows (fna2_paged_shared.hip).
#pragma once

#include "fna2_kernels.h"
#include "fna2_paged_dev.h"
#include "fna2_paged_shared.h"

namespace fna2 {

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

// SHARED: the sequences are those of a plan (PagedSharedParams), in which a
// sequence may begin behind rows that its group shares; a tile leaves its
// output for the join of the two.  TWO: P in two parts, as the packed kernel has it.
template <int D, int RPL, int HW, bool F16, bool SHARED, bool TWO = false>
__device__ __forceinline__ void tile_body() {
  KArg P = kargs();
  using C = TileCfg<D, RPL, HW>;
  constexpr int BN = C::BN;
  __shared__ __attribute__((aligned(1024))) uint8_t stage0[C::STAGE];
  __shared__ __attribute__((aligned(1024))) uint8_t stage1[C::STAGE];
  __shared__ typename std::conditional<SHARED, SharedSmallPlan, int>::type small;  // (SHARED) the plan
  __shared__ volatile int odd_flag;  // a V tile holds infinities or NaN (see fna2_paged_dev.h)
  const int lane = threadIdx.x & 63, wv = uni(threadIdx.x >> 6);
  const int l32 = lane & 31, hl = lane >> 5;
  if (threadIdx.x == 0) odd_flag = 0;  // (read behind a barrier of the first step at the earliest)
  const int hw = RPL > 0 ? HW : P->hw;  // (without ranks a tile's heads do not show in its layout)
  const int TB = 128 / hw;
  const int hblk = cdiv(P->group, hw);  // blocks of heads of a KV head

  int run = run_of(blockIdx.x, gridDim.x);
  bool full = false;  // (SHARED) a chunk of a tile of shared rows, the run's all
  int64_t left, per;  // units of this run still to do, and of a run
  int b, hb, qt, s0;
  PagedSeq e;
  SharedSeq v{};  // (SHARED) the rest of the sequence's record
  SharedPlanRef plan{};
  auto cut = [&](int seq, int head, int tile, int parts) {
    if (threadIdx.x == 0) P->cuts[run] = PagedCut{seq, head, tile, parts};
  };
  if constexpr (SHARED) {
    SArg S = sargs();
    plan = SharedPlanRef{S->meta, S->groups, S->group_ends, S->seqs, S->ends};
    if (S->small) {
      plan = SharedPlanRef{&small.meta, small.groups, small.group_ends, small.seqs, small.ends};
      if (wv == 0) shared_plan_small(S, small, lane);
      __syncthreads();
    }
    per = uni64(plan.meta->per);
    const int nfull = (int)uni64(plan.meta->full);
    const int64_t units = uni64(plan.meta->units);
    // Every XCD has its share of the full runs, first, and of the others.
    const int x = blockIdx.x & 7, j = blockIdx.x >> 3;
    const int lo = nfull * x / 8, mine = nfull * (x + 1) / 8 - lo;
    full = j < mine;
    if (full) {
      run = lo + j;
      int64_t at;
      const SharedGroup& g = plan.groups[shared_seek(plan.group_ends, S->G, lane, run, at)];
      e = PagedSeq{uni(g.s.q0), uni(g.s.lq), uni(g.s.lk), uni(g.s.off)};
      v.table = uni(g.table);
      const int tiles = uni(g.tiles);
      const int c = (int)at / (tiles * TilePlan::blocks(P)), rest = (int)at - c * (tiles * TilePlan::blocks(P));
      b = 0;
      hb = uni(rest / tiles);
      qt = uni(rest - hb * tiles);
      left = per;
      s0 = uni((int)(c * left));
    } else {
      run = nfull + x * (int)(gridDim.x >> 3) - lo + (j - mine);
      const int64_t u = (int64_t)(run - nfull) * per;
      left = min(units - u, per);
      if (left <= 0) return;
      int64_t rem;
      b = shared_seek(plan.ends, S->V, lane, u, rem);
      v = shared_seq_uniform(plan.seqs, b);
      e = v.s;
      const int64_t hu = SharedUnits::head_units(S, e);
      hb = uni((int)div64(rem, hu));
      int64_t r = rem - hb * hu;
      qt = uni(SharedUnits::find(S, e, r));
      // (a run that ends in a tile's start leaves the tile to the next one)
      s0 = uni((int)max(r - S->start, (int64_t)0));
      left -= max(S->start - r, (int64_t)0);
      if (left <= 0) return;
    }
  } else {
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
    const int row0 = SHARED ? v.row0 : 0;  // of the cache: the sequence's row 0 here
    const int* trow = P->table + (int64_t)(SHARED ? v.table : b) * P->tstride;
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
    ids.last = k_end > 0 ? page_of(P->ps_mul, P->ps_shift, k_end - 1 + row0) : -1;
    int row = 32 * s0 + 16 * rg;
    int page = page_of(P->ps_mul, P->ps_shift, row + row0), poff = row + row0 - page * ps;
    // Rows of the part in pages that are not there (rare) are masked.
    bool gone = false;
    {
      const int first = page_of(P->ps_mul, P->ps_shift, 32 * s0 + row0);
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
            if (r >= k_end || (uint32_t)uni(*const_space(trow + page_of(kargs()->ps_mul, kargs()->ps_shift, r + row0))) < (uint32_t)npages) continue;
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
      bf16x8 pb[BN / 16], pe[BN / 16];
      u32x4 pk[BN / 16], ek[BN / 16];  // (ek, pe: TWO)
      auto exps = [&](int q, int i0, int i1) {
#pragma unroll
        for (int i = i0; i < i1; ++i) {
          const int v0 = 8 * (q & 1) + 2 * i;
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[q >> 1][v0], c2, nm));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[q >> 1][v0 + 1], c2, nm));
          ls += p0 + p1;
          if constexpr (TWO) {
            split_p<F16>(p0, p1, pk[q], ek[q], i);
          } else {
            pk[q][i] = pack_e<F16>(p0, p1);
          }
        }
        if (i1 == 4) {
          pb[q] = as_bf16x8(pk[q]);
          if constexpr (TWO) pe[q] = as_bf16x8(ek[q]);
        }
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
        if constexpr (TWO) oacc[d] = mfma_e<F16>(vr[i % C::A2], pe[s], oacc[d]);
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
    const bool whole = s0 == 0 && s1 == steps && !full;
    if (whole && (!SHARED || v.kind == kSharedAlone)) {
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
    } else if (SHARED && whole) {
      if (live) {
        SArg S = sargs();
        const int64_t r = ((int64_t)(v.kind == kSharedPrefix) * P->T + e.q0 + tok) * P->H + h;
        float* arow = S->whole + r * D + 4 * hl;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            f32x4_t val = {oacc[d][4 * g], oacc[d][4 * g + 1], oacc[d][4 * g + 2], oacc[d][4 * g + 3]};
            *(f32x4_t*)(arow + d * 32 + 8 * g) = val;
          }
        if (hl == 0) *(f32x2*)(S->whole_ml + 2 * r) = f32x2{m_i, l_tot};
      }
    } else if (live) {
      // As the registers lie: [slot][wave][d][4][lane] of 16 bytes.
      const int64_t slot = (2 * (int64_t)run + (s0 == 0 || full ? 1 : 0)) * 4 + wv;
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

    if constexpr (SHARED) {
      if (full) return;
      // The run in which a tile begins says where its parts lie.
      if (s0 == 0 && wv % hw == 0 && live && hl == 0) {
        SArg S = sargs();
        const int rest = steps - s1;
        SharedRec rec{};
        rec.at = run | (tok - qt * TB) << 16;
        rec.parts = rest > 0 ? 1 + (int)div64(rest + per - 1, per) : v.kind == kSharedAlone ? -1 : 0;
        if (v.kind == kSharedOwn) {
          const SharedGroup g = plan.groups[v.group];
          const int t = e.q0 + tok - g.s.q0;
          rec.at |= kSharedHas | (g.full * per * 32 < g.s.lk ? kSharedRest : 0);
          rec.run0 = (int)g.run0 + hb * g.tiles + t / TB;
          rec.stride = g.tiles * TilePlan::blocks(P);
          rec.full = (int)g.full;
          rec.at0 = t % TB;
        }
        S->recs[((int64_t)(v.kind == kSharedPrefix) * (P->H_KV * hblk) + hb) * P->T + e.q0 + tok] = rec;
      }
    }
    left -= s1 - s0;
    if constexpr (SHARED) left -= sargs()->start;  // of the next tile
    if (SHARED && left <= 0) return;
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
        if constexpr (SHARED) {
          SArg S = sargs();
          do v = shared_seq_uniform(plan.seqs, ++b); while (v.s.lq == 0 && b + 1 < S->V);
          e = v.s;
        } else {
          do e = paged_seq_uniform(P, ++b); while (e.lq == 0 && b + 1 < P->N);
        }
      }
    }
  }
}

// Waves per SIMD that the register budget is cut for, and workgroups of a CU.
// Three where one head's ranks or none come with d = 128: such tiles are long,
// bound by the matrix cores, and a third workgroup fills the others' waits
// (1024-token piece, rank 64, in turn: 346 us, two 351).  Two for the others: the third
// costs spilled registers (mixed step, 4 heads of rank 32: 146 us, two 133; d =
// 64, rank 16, 509-token pieces with their weights: 103, 97).  A third ring
// stage in the room that leaves: 136 and 99.  Two for P in two parts with ranks too,
// where a third spills 19 to 106 registers (32 sequences of a token over 8192 shared and 512 own
// rows, 16 heads, rank 32 85 us, two 74; rank 64 103, 83).
constexpr int tile_occ(int D, int RPL, int HW, bool TWO = false) {
  return D == 128 && (RPL == 0 || (HW == 1 && !TWO)) ? 3 : 2;
}

}  // namespace fna2
