// fna2_paged_attn.hip — attention of chunks of new tokens over a paged cache.
//
// Token i of a sequence's chunk of lq tokens sits at row off + i of the cache,
// off = lk - lq, and sees the rows up to its own (all lk, not causal):
//     S_j = softmax_scale <q, K_j> + [h < H_G] graph_scale[h] <rq, Rk_j>,
//     O = sum_j e^{S_j - m} V_j / (l + 1e-6),  LSE = m + log(l + 1e-6).
//
// Packed kernel.  The columns of a 32-wide MFMA tile are (token, query head)
// pairs: the gsub query heads that share a KV head (and whose ranks fit one
// tile) times as many tokens as fit.  One token and a few drafted ones so
// read K and V once per KV head.  A wave works alone: per 32-row step it
// forms S^T = Ka Qa^T by one MFMA chain over the head dim and the
// concatenated ranks of its heads (Rq block diagonal), the online softmax by
// column, and O^T += V^T P^T with V^T read transposed from LDS.
//
// Work.  The column tiles' key steps are laid end to end over all sequences
// and every wave takes an equal run of them, so that the chip is evenly busy
// however ragged the lengths are; the lengths stay on the device, where every
// wave finds its run from them.  A run that covers a tile writes its output;
// a tile cut by runs leaves unnormalised parts that the merge kernel joins in
// the order of the runs.
//
// Pages.  A step's rows come as two groups of 16, each within one page
// (page_size is a multiple of 16), DMA'd to LDS through descriptors of their
// own that end with the sequence: what lies behind its last row, or in a
// page that is not there, is never read and comes as zeros.  64 page ids at a time
// lie in the lanes of a register.
//
// Bound by reading K, V and R_k once: 64 sequences of 4096 rows, one token each, 16
// heads over 16 KV heads of 128, R = 32, 410 us, 5.9 TB/s (a large copy, read and written, 5.1 TB/s).
// Few sequences are bound by the latency of the chain lengths, page ids, first
// rows, parts, merge: 2 of 500 rows, 8 heads of 64, 7.7 us and 4.6 us for the merge.
// A few drafted tokens (5 for 16 ragged sequences of up to 2500 rows, 16 heads over 4,
// R = 24) are as well: 25.6 and 7.8 us, 2.8 TB/s from three waves a CU.
// A ring of three stages gained nothing over two: the other waves cover the loads.
#include <algorithm>

#include "fna2_kernels.h"
#include "fna2_paged_dev.h"

namespace fna2 {

namespace {

constexpr int kPagBN = 32;  // keys per step

template <int N>
__device__ __forceinline__ void paged_wait() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));  // lgkmcnt(0)
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

template <int D, int RC>
struct PackCfg {
  static constexpr int CD = D / 8;
  static constexpr int KSD = D / 16;
  static constexpr int KSR = RC / 2;
  static constexpr int KBYTES = kPagBN * D * 2;
  static constexpr int RBYTES = kPagBN * RC * 16;
  static constexpr int STAGE = 2 * KBYTES + RBYTES;
  static constexpr int NG = CD / 4;      // column groups of a K / V tile
  static constexpr int NR = RC / 4;      // ... of an Rk tile
};

template <int D, int RC, bool F16>
__device__ __forceinline__ void packed_body() {
  KArg P = kargs();
  using C = PackCfg<D, RC>;
  __shared__ __attribute__((aligned(1024))) uint8_t st0[C::STAGE];
  __shared__ __attribute__((aligned(1024))) uint8_t st1[C::STAGE];
  const int lane = threadIdx.x;
  const int col = lane & 31, hl = lane >> 5;
  const int tk = small_div(col, P->gsub), hc = col - tk * P->gsub;  // token of the tile, head of the group
  const int cols = P->gsub * P->tpt;
  const int HB = P->H_KV * P->nsub;
  auto cut = [&](int b, int head, int tile, int parts) {
    if (lane == 0) P->cuts[blockIdx.x] = PagedCut{b, head, tile, parts};
  };
  int64_t left, per;  // units of this run still to do, and of a run
  int b, ct, sg, s0, steps;
  PagedSeq e;
  {
    auto units = [&](const PagedSeq& s) { return PackedPlan::units(P, s); };
    SeqWork<decltype(units)> work(P, lane, units);
    // One step a run while the parts are few, else two.  (us, one step, two,
    // four: 128 steps x 2 columns 10.6, 11.8, 14.9; 640 x 4 13.9, 15.0, 19.9;
    // 1024 x 4 16.6, 14.5, 15.3; 512 x 24 20.8, 17.6, 21.5)
    per = run_units(P, work.total, work.total * cols <= 3000 ? 1 : 2);
    const int64_t u = (int64_t)blockIdx.x * per;
    left = min(work.total - u, per);
    if (left <= 0) {
      cut(0, 0, 0, 0);
      return;
    }
    const PagedAt at = work.seek(P, lane, u);
    b = at.b;
    e = at.s;
    steps = PackedPlan::steps(e);
    const int64_t tile = div64(at.rem, steps);
    s0 = uni((int)(at.rem - tile * steps));
    ct = uni((int)div64(tile, HB));
    sg = uni((int)(tile - (int64_t)ct * HB));
  }

  const TrLane tl(lane);
  const RowLane rdl(lane);
  const int crr = P->R / 8;
  const uint32_t krb = (uint32_t)P->k.ss * 2u, vrb = (uint32_t)P->v.ss * 2u;
  // lane offsets within a 16-row group: row lane / 4, chunk 4 g + (lane % 4)
  // swizzled (row bits 1..3 only, so both groups of a tile agree)
  const int lrow = lane >> 2, lch = (lane & 3) ^ swz4(lane >> 2);
  const uint32_t kvo = (uint32_t)lrow * krb + 16u * lch, vvo = (uint32_t)lrow * vrb + 16u * lch;

  while (true) {
    P = kargs();
    const bool causal = P->causal != 0;
    const int ps = P->ps, npages = P->npages;
    const float c2 = P->c2;
    const int s1 = (int)min((int64_t)steps, s0 + left);
    const int kvh = P->nsub == 1 ? sg : sg / P->nsub, h_in = (sg - kvh * P->nsub) * P->gsub;
    const int nh = min(P->gsub, P->group - h_in);  // heads of this group
    const int h0 = kvh * P->group + h_in;
    const int gg = RC > 0 ? min(max(P->H_G - h0, 0), nh) : 0;  // graph heads
    const int rch = gg * crr, nrs = cdiv(rch, 2);
    const int tok = ct * P->tpt + tk;
    const bool live = tk < P->tpt && tok < e.lq && hc < nh;
    const int off = e.off;
    // last key that this column, and that every column, sees
    const int lim = min(causal ? off + tok : e.lk, e.lk - 1);
    const int lim_all = causal ? min(off + ct * P->tpt, e.lk - 1) : e.lk - 1;
    const int lim_any = causal ? off + ct * P->tpt + P->tpt - 1 : e.lk - 1;  // ... that any sees
    const int* trow = P->table + (int64_t)b * P->tstride;
    const uint16_t* const kpool = (const uint16_t*)P->k.ptr + (int64_t)kvh * P->k.sh;
    const uint16_t* const vpool = (const uint16_t*)P->v.ptr + (int64_t)kvh * P->v.sh;
    const uint16_t* const rpool = RC > 0 ? (const uint16_t*)P->rk.ptr + (int64_t)h0 * P->rk.sh : nullptr;
    const int64_t ksb = P->k.sb, vsb = P->v.sb, rsb = P->rk.sb;
    const uint32_t rrb = (uint32_t)P->rk.ss * 2u;

    uint32_t roff[RC > 0 ? C::NR : 1];
    if constexpr (RC > 0) {
      const uint32_t hs = (uint32_t)P->rk.sh * 2u, rs = (uint32_t)P->rk.ss * 2u;
#pragma unroll
      for (int i = 0; i < C::NR; ++i) {
        const int c = 4 * i + lch, hh = small_div(c, max(crr, 1));
        roff[i] = c < rch ? (uint32_t)hh * hs + (uint32_t)lrow * rs + (uint32_t)(c - hh * crr) * 16u
                          : kOOB;
      }
    }
    // Page and row within it of the next row group to be issued.
    PageIds ids;
    ids.row = trow;
    ids.last = e.lk > 0 ? page_of(P->ps_mul, P->ps_shift, e.lk - 1) : -1;
    int page = page_of(P->ps_mul, P->ps_shift, 32 * s0), poff = 32 * s0 - page * ps;
    ids.load(lane, page);
    // Tile t into `base`; returns the row groups that are not there although
    // below lk (bit g).
    auto issue = [&](int t, uint8_t* base) {
      int gone = 0;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int row = 32 * t + 16 * g;
        const bool in = row < e.lk && t < s1;
        int id = in ? ids.at(lane, page) : 0;
        const int r = poff;
        poff += 16;
        if (poff >= ps) poff = 0, ++page;
        if ((uint32_t)id >= (uint32_t)npages) {
          id = -1;
          if (in) gone |= 1 << g;
        }
        const int rows = in && id >= 0 ? clamp_rows(e.lk - row, 16) : 0;
        id = max(id, 0);
        const auto rk_ = make_rsrc((const uint8_t*)(kpool + (int64_t)id * ksb) + (uint64_t)(uint32_t)r * krb,
                                   (uint32_t)rows * krb);
        const auto rv_ = make_rsrc((const uint8_t*)(vpool + (int64_t)id * vsb) + (uint64_t)(uint32_t)r * vrb,
                                   (uint32_t)rows * vrb);
#pragma unroll
        for (int i = 0; i < C::NG; ++i) {
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rk_, (lds_void*)(base + (2 * i + g) * 1024), 16,
                                                   kvo + 64u * i, 0, 0, 0);
          __builtin_amdgcn_raw_ptr_buffer_load_lds(
              rv_, (lds_void*)(base + C::KBYTES + C::RBYTES + (2 * i + g) * 1024), 16,
              vvo + 64u * i, 0, 0, 0);
        }
        if constexpr (RC > 0) {
          const auto rr = make_rsrc((const uint8_t*)(rpool + (int64_t)id * rsb) + (uint64_t)(uint32_t)r * rrb,
                                    rows > 0 && gg > 0 ? 0x7ffffff0u : 0u);
#pragma unroll
          for (int i = 0; i < C::NR; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rr, (lds_void*)(base + C::KBYTES + (2 * i + g) * 1024), 16,
                lrow < rows ? roff[i] : kOOB, 0, 0, 0);
        }
      }
      return gone;
    };

    // Query operand (B of S^T): lane holds Qa[col][16 s + 8 hl .. +7].  Loaded
    // behind the page ids and ahead of the first tile, whose waits it shares.
    bf16x8 qreg[C::KSD + (RC > 0 ? C::KSR : 0)];
    float bh = 0.f;
    {
      const int64_t t = (int64_t)(e.q0 + (live ? tok : 0));
      const uint16_t* qrow = (const uint16_t*)P->q.ptr + t * P->q.ss + (int64_t)(h0 + hc) * P->q.sh;
#pragma unroll
      for (int s = 0; s < C::KSD; ++s) {
        u32x4 w = {0, 0, 0, 0};
        if (live) w = ld16(qrow + 16 * s + 8 * hl);
        qreg[s] = as_bf16x8(w);
      }
      if constexpr (RC > 0) {
        const bool g = live && hc < gg;
        const uint16_t* rrow = (const uint16_t*)P->rq.ptr + t * P->rq.ss + (int64_t)(h0 + hc) * P->rq.sh;
        bh = g ? P->gs[h0 + hc] / P->c : 0.f;
#pragma unroll
        for (int s = 0; s < C::KSR; ++s) {
          const int c = 2 * s + hl - hc * crr;  // this head's chunk of the lane
          u32x4 w = {0, 0, 0, 0};
          if (g && c >= 0 && c < crr) w = ld16(rrow + 8 * c);
          qreg[C::KSD + s] = as_bf16x8(w);
        }
      }
    }
    int gone = issue(s0, st0);
    __builtin_amdgcn_sched_barrier(0);
    {
      const uint32_t qxor = P->qa < 0.f ? 0x80008000u : 0u;
      const uint32_t qand = P->qa == 0.f ? 0u : 0xffffffffu;
#pragma unroll
      for (int s = 0; s < C::KSD; ++s) {
        u32x4 w = as_u32x4(qreg[s]);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (w[i] & qand) ^ qxor;
        qreg[s] = as_bf16x8(w);
      }
    }

    // Scores kept for the rows' weights.
    const bool keep = P->scores && e.lq <= P->tpt;
    float* const srow = keep ? paged_scores(P, b, sg) + (int64_t)min(col, cols - 1) * P->srows + 4 * hl : nullptr;
    bool stored = false;  // the newest four memory instructions are a step's scores

    f32x16 oacc[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) oacc[d] = f32x16{};
    float m_i = kNegInf, l_i = 0.f;

    auto step = [&](auto apart, int t, uint8_t* cur_st, uint8_t* nxt_st) {
      constexpr bool APART = decltype(apart)::value;
      // (loads and stores end in order: those before the scores have)
      if (stored) paged_wait<4>();
      else paged_wait<0>();
      stored = false;
      const int gone_now = gone;
      gone = issue(t + 1, nxt_st);  // (past the run: zeros, from no memory)
      __builtin_amdgcn_sched_barrier(0);
      if (32 * t > lim_any) return;  // no column sees these rows
      if (causal && 32 * t + 31 > lim_all) {
        uint8_t* v = cur_st + C::KBYTES + C::RBYTES;
        if (__builtin_expect(tile_odd<C::KBYTES / 1024, F16>(v, lane), 0)) {
          add_odd<D, kPagBN, F16>(v, 32 * t, lim, hl, oacc);
          tile_clean<C::KBYTES / 1024, F16>(v, lane);
        }
      }
      const uint8_t* kl = cur_st;
      const uint8_t* rl = kl + C::KBYTES;
      const uint8_t* vl = rl + C::RBYTES;
      f32x16 acc = f32x16{};
      if constexpr (RC > 0 && !APART) {
#pragma unroll
        for (int s = 0; s < C::KSR; ++s)
          if (s < nrs) acc = mfma32(row_read<kPagBN>(rl, rdl, 0, s), qreg[C::KSD + s], acc);
        acc *= bh;
      }
      if constexpr (APART) {  // a chain for each head, without the others' ranks
        const int cr = uni(kargs()->R / 8);
#pragma unroll 1
        for (int hh = 0; hh * cr < uni(rch); ++hh) {
          f32x16 own = f32x16{};
#pragma unroll
          for (int s = 0; s < C::KSR; ++s) {
            const int c = 2 * s + hl - hh * cr;
            u32x4 w = as_u32x4(row_read<kPagBN>(rl, rdl, 0, s));
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = c >= 0 && c < cr ? w[i] : 0u;
            own = mfma32(as_bf16x8(w), qreg[C::KSD + s], own);
          }
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[v] = hc == hh ? own[v] * bh : acc[v];
        }
      }
#pragma unroll
      for (int s = 0; s < C::KSD; ++s)
        acc = mfma_e<F16>(row_read<kPagBN>(kl, rdl, 0, s), qreg[s], acc);
      const int kbase = 32 * t;
      const bool masked = kbase + 31 > lim_all || gone_now;
      if (masked) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int key = kbase + 8 * (v >> 2) + 4 * hl + (v & 3);
          const bool dead = key > lim || ((gone_now >> (v >> 3)) & 1);
          acc[v] = dead ? kNegInf : acc[v];
        }
      }
      if (keep) {
        if (col < cols) {  // (column 0 always is: four stores)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *(f32x4_t*)(srow + kbase + 8 * g) = f32x4_t{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
        }
        stored = true;
      }
      float mx = kNegInf;
#pragma unroll
      for (int v = 0; v < 16; ++v) mx = fmaxf(mx, acc[v]);
      mx = wave_pair_max(mx);
      const float m_new = fmaxf(m_i, mx);
      const float m_use = (m_new == kNegInf) ? 0.f : m_new;
      const float nm = -m_use * c2;
      float ls = 0.f;
      bf16x8 pb[2], pe[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        u32x4 pk, ek;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int v0 = 8 * half + 2 * i;
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[v0], c2, nm));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[v0 + 1], c2, nm));
          ls += p0 + p1;
          split_p<F16>(p0, p1, pk, ek, i);
        }
        pb[half] = as_bf16x8(pk);
        pe[half] = as_bf16x8(ek);
      }
      if (__builtin_amdgcn_ballot_w64(m_new != m_i) != 0) {
        const float alpha = weight2((m_i - m_use) * c2);
        l_i *= alpha;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) oacc[d] *= alpha;
      }
      l_i += ls;
      m_i = m_new;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
          const bf16x8 vt = tr_operand<kPagBN>(vl, tl, 16 * s, 32 * d);
          oacc[d] = mfma_e<F16>(vt, pb[s], oacc[d]);
          oacc[d] = mfma_e<F16>(vt, pe[s], oacc[d]);
        }
    };

    for (int t = s0; t < s1; t += 2) {
      step(std::false_type{}, t, st0, st1);
      if (t + 1 < s1) step(std::false_type{}, t + 1, st1, st0);
    }
    paged_wait<0>();  // no DMA may still write when the ring is used again, or the wave ends
    // R_q's zeros keep the heads of a tile apart, but not from an infinity or a NaN in
    // another's R_k row, which times zero is NaN.  Where a sum is NaN the part is done
    // again, a rank chain for each head (in the step itself: 50 scalar registers more
    // spilled).
    if constexpr (RC > 0) {
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(live && l_i != l_i) != 0 && rch > 0, 0)) {
        KArg p = kargs();
        page = page_of(p->ps_mul, p->ps_shift, 32 * s0), poff = 32 * s0 - page * ps;
        ids.load(lane, page);
#pragma unroll
        for (int d = 0; d < D / 32; ++d) oacc[d] = f32x16{};
        m_i = kNegInf, l_i = 0.f;
        stored = false;
        gone = issue(s0, st0);
        uint8_t *cur = st0, *nxt = st1;
#pragma unroll 1
        for (int t = s0; t < s1; ++t) {
          step(std::true_type{}, t, cur, nxt);
          uint8_t* const was = cur;
          cur = nxt, nxt = was;
        }
        paged_wait<0>();
      }
    }

    P = kargs();
    const float l_tot = wave_pair_sum(l_i);
    if (s0 == 0 && s1 == steps) {
      if (live) {
        const float inv = 1.f / (l_tot + 1e-6f);
        uint16_t* orow = (uint16_t*)P->o.ptr + (int64_t)(e.q0 + tok) * P->o.ss + (int64_t)(h0 + hc) * P->o.sh;
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
          ((float*)P->lse.ptr)[(int64_t)(e.q0 + tok) * P->lse.ss + (int64_t)(h0 + hc) * P->lse.sh] =
              m_i == kNegInf ? kNegInf : m_i * P->c + __builtin_amdgcn_logf(l_tot + 1e-6f) * kLn2;
      }
    } else if (col < cols) {
      // slot 2 w: wave w's run ends or lies in a tile begun before it; 2 w + 1:
      // it begins the tile
      const int64_t slot = 2 * (int64_t)blockIdx.x + (s0 == 0 ? 1 : 0);
      float* arow = P->part + (slot * cols + col) * D;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f32x4_t val = {oacc[d][4 * g], oacc[d][4 * g + 1], oacc[d][4 * g + 2], oacc[d][4 * g + 3]};
          *(f32x4_t*)(arow + d * 32 + 8 * g + 4 * hl) = val;
        }
      if (hl == 0) *(f32x2*)(P->ml + 2 * (slot * cols + col)) = f32x2{m_i, l_tot};
    }

    left -= s1 - s0;
    if (left <= 0) {
      const int rest = steps - s1;
      cut(b, sg, ct, s0 == 0 && rest > 0 ? 1 + (int)div64(rest + per - 1, per) : 0);
      return;
    }
    s0 = 0;
    if (++sg == HB) {
      sg = 0;
      if ((++ct) * P->tpt >= e.lq) {
        ct = 0;
        do e = paged_seq_uniform(P, ++b); while (e.lq == 0 && b + 1 < P->N);
        steps = PackedPlan::steps(e);
      }
    }
  }
}

// Joins the parts of the tiles that runs cut: workgroup (x, y) those of runs
// x merge_runs .. + merge_runs - 1 (of which most cut no tile, or not first, where a
// tile has many parts), columns y, y + gridDim.y, ...  D / 4 lanes hold a row,
// so the workgroup NG rows at once: with a workgroup for every column NG parts of it,
// four deep; else NG columns, each of whose lanes walk its parts.  The order of the
// sums goes by the parts alone.
constexpr int kMergeParts = 2048;  // at most one part for each resident wave
template <int D, bool F16>
__global__ __launch_bounds__(256) void paged_merge_kernel(const PagedParams) {
  KArg P = kargs();
  constexpr int LPR = D / 4, NG = 256 / LPR;
  __shared__ float wt[kMergeParts];
  __shared__ float part[NG][D];
  __shared__ float red[4], red2[4];
  if (blockIdx.y == 0) clear_loose_tokens(P, blockIdx.x, gridDim.x);
  const int mr = P->merge_runs, r0 = blockIdx.x * mr + (threadIdx.x & 63);
  uint64_t todo = __builtin_amdgcn_ballot_w64(
      (int)(threadIdx.x & 63) < mr && r0 < P->waves && P->cuts[min(r0, P->waves - 1)].parts > 0);
  while (todo) {
    const int i0 = blockIdx.x * mr + uni(__builtin_ctzll(todo));
    todo &= todo - 1;
    const auto rec = const_space(P->cuts + i0);
    const int n = uni(rec->parts);
    const int ct = uni(rec->tile), sg = uni(rec->head);
    const PagedSeq e = paged_seq_uniform(P, rec->b);
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int kvh = sg / P->nsub, h_in = (sg - kvh * P->nsub) * P->gsub;
    const int nh = min(P->gsub, P->group - h_in), h0 = kvh * P->group + h_in;
    const int cols = P->gsub * P->tpt;
    const int grp = threadIdx.x / LPR, f = 4 * (threadIdx.x % LPR);
    const float c2 = P->c2;
    auto slot = [&](int j) { return (int64_t)(j == 0 ? 2 * i0 + 1 : 2 * (i0 + j)); };
    if (n <= LPR && (int)gridDim.y < cols) {
      const int c = blockIdx.y + gridDim.y * grp;  // (gridDim.y * NG >= cols)
      const int l = threadIdx.x % LPR;
      const int tk = c / P->gsub, hc = c - tk * P->gsub, tok = ct * P->tpt + tk;
      const bool on = c < cols && tok < e.lq && hc < nh;
      f32x2 ml = {kNegInf, 0.f};
      if (on && l < n) ml = *(const f32x2*)(P->ml + 2 * (slot(l) * cols + c));
      const float* src = P->part + (int64_t)(on ? c : 0) * D + f;
      float m = ml[0];
#pragma unroll
      for (int k = LPR / 2; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
      const float ref = m == kNegInf ? 0.f : m;
      const float w = weight2((ml[0] - ref) * c2);
      float sum = ml[1] * w;
#pragma unroll
      for (int k = LPR / 2; k > 0; k >>= 1) sum += __shfl_xor(sum, k);
      f32x4_t o = {0.f, 0.f, 0.f, 0.f};
      for (int j0 = 0; j0 < n; j0 += 4) {
        f32x4_t x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
          if (on && j0 + k < n) x[k] = *(const f32x4_t*)(src + slot(j0 + k) * cols * D);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float wj = __shfl(w, min(j0 + k, n - 1), LPR);
          if (j0 + k < n) o += wj * x[k];
        }
      }
      if (!on) continue;
      const float inv = 1.f / (sum + 1e-6f);
      uint16_t* orow = (uint16_t*)P->o.ptr + (int64_t)(e.q0 + tok) * P->o.ss + (int64_t)(h0 + hc) * P->o.sh;
      u32x2 val;
      val[0] = pack_e<F16>(o[0] * inv, o[1] * inv);
      val[1] = pack_e<F16>(o[2] * inv, o[3] * inv);
      *(u32x2*)(orow + f) = val;
      if (l == 0 && P->lse.ptr)
        ((float*)P->lse.ptr)[(int64_t)(e.q0 + tok) * P->lse.ss + (int64_t)(h0 + hc) * P->lse.sh] =
            m == kNegInf ? kNegInf : m * P->c + __builtin_amdgcn_logf(sum + 1e-6f) * kLn2;
      continue;
    }
    for (int c = blockIdx.y; c < cols; c += gridDim.y) {
      const int tk = c / P->gsub, hc = c - tk * P->gsub, tok = ct * P->tpt + tk;
      if (tok >= e.lq || hc >= nh) continue;  // (uniform)
      const float* src = P->part + (int64_t)c * D + f;
      f32x4_t x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = grp + k * NG;
        if (j < n) x[k] = *(const f32x4_t*)(src + slot(j) * cols * D);
      }
      float m = kNegInf;
      for (int j = threadIdx.x; j < n; j += 256) m = fmaxf(m, P->ml[2 * (slot(j) * cols + c)]);
#pragma unroll
      for (int k = 32; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
      if (lane == 0) red[wv] = m;
      __syncthreads();
      m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
      const float ref = m == kNegInf ? 0.f : m;
      float l = 0.f;
      for (int j = threadIdx.x; j < n; j += 256) {
        const f32x2 ml = *(const f32x2*)(P->ml + 2 * (slot(j) * cols + c));
        const float w = weight2((ml[0] - ref) * c2);
        wt[j] = w;
        l += ml[1] * w;
      }
#pragma unroll
      for (int k = 32; k > 0; k >>= 1) l += __shfl_xor(l, k);
      if (lane == 0) red2[wv] = l;
      __syncthreads();
      l = (red2[0] + red2[1]) + (red2[2] + red2[3]);
      f32x4_t o = {0.f, 0.f, 0.f, 0.f};
      for (int base = 0; base < n; base += 4 * NG) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = base + grp + k * NG;
          if (j < n) o += wt[j] * x[k];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = base + grp + (4 + k) * NG;
          if (j < n) x[k] = *(const f32x4_t*)(src + slot(j) * cols * D);
        }
      }
      *(f32x4_t*)(&part[grp][f]) = o;
      __syncthreads();
      const float inv = 1.f / (l + 1e-6f);
      if (threadIdx.x < D / 2) {
        const int d = 2 * threadIdx.x;
        float y0 = 0.f, y1 = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) y0 += part[g][d], y1 += part[g][d + 1];
        uint16_t* orow = (uint16_t*)P->o.ptr + (int64_t)(e.q0 + tok) * P->o.ss + (int64_t)(h0 + hc) * P->o.sh;
        *(uint32_t*)(orow + d) = pack_e<F16>(y0 * inv, y1 * inv);
        if (d == 0 && P->lse.ptr)
          ((float*)P->lse.ptr)[(int64_t)(e.q0 + tok) * P->lse.ss + (int64_t)(h0 + hc) * P->lse.sh] =
              m == kNegInf ? kNegInf : m * P->c + __builtin_amdgcn_logf(l + 1e-6f) * kLn2;
      }
      __syncthreads();
    }
  }
}

// Waves per SIMD that the register budget is cut for.  Two (256 registers): the
// accumulators then stay in ordinary registers, where with one wave's budget
// the compiler keeps them in the other half of the file and copies them to
// and fro in every step.
constexpr int packed_occ(int D, int RC) { return D == 128 && RC > 16 ? 1 : 2; }

#define FNA2_PACKED(D, RC)                                                                     \
  __global__ __launch_bounds__(64, packed_occ(D, RC)) void paged_packed_d##D##_c##RC(const PagedParams) {    \
    packed_body<D, RC, false>();                                                               \
  }                                                                                            \
  __global__ __launch_bounds__(64, packed_occ(D, RC)) void paged_packed_d##D##_c##RC##_f16(const PagedParams) { \
    packed_body<D, RC, true>();                                                                \
  }
FNA2_PACKED(64, 0)
FNA2_PACKED(64, 4)
FNA2_PACKED(64, 8)
FNA2_PACKED(64, 16)
FNA2_PACKED(64, 32)
FNA2_PACKED(128, 0)
FNA2_PACKED(128, 4)
FNA2_PACKED(128, 8)
FNA2_PACKED(128, 16)
FNA2_PACKED(128, 32)
#undef FNA2_PACKED

}  // namespace

int paged_rank_chunks(int rch) {
  return rch <= 0 ? 0 : rch <= 4 ? 4 : rch <= 8 ? 8 : rch <= 16 ? 16 : rch <= 32 ? 32 : -1;
}

int paged_waves_per_cu(int D, int rc) {
  const int ring = 2 * kPagBN * (2 * D * 2 + rc * 16);
  return std::max(1, std::min(8, (160 * 1024 - 1) / ring));
}

hipError_t launch_paged_packed(const PagedParams& P, int rc, hipStream_t s) {
  void (*k)(const PagedParams) = nullptr;
#define FNA2_PACKED_OF(D, RC) (P.f16 ? paged_packed_d##D##_c##RC##_f16 : paged_packed_d##D##_c##RC)
  if (P.D == 64)
    k = rc == 0 ? FNA2_PACKED_OF(64, 0) : rc == 4 ? FNA2_PACKED_OF(64, 4) : rc == 8 ? FNA2_PACKED_OF(64, 8)
      : rc == 16 ? FNA2_PACKED_OF(64, 16) : rc == 32 ? FNA2_PACKED_OF(64, 32) : nullptr;
  if (P.D == 128)
    k = rc == 0 ? FNA2_PACKED_OF(128, 0) : rc == 4 ? FNA2_PACKED_OF(128, 4) : rc == 8 ? FNA2_PACKED_OF(128, 8)
      : rc == 16 ? FNA2_PACKED_OF(128, 16) : rc == 32 ? FNA2_PACKED_OF(128, 32) : nullptr;
#undef FNA2_PACKED_OF
  if (!k) return hipErrorInvalidValue;
  hipLaunchKernelGGL(k, dim3((uint32_t)P.waves), dim3(64), 0, s, P);
  return hipGetLastError();
}

hipError_t launch_paged_merge(const PagedParams& P, hipStream_t s) {
  const int cols = P.gsub * P.tpt, rows = 256 / (P.D / 4);
  const dim3 grid((uint32_t)((P.waves + P.merge_runs - 1) / P.merge_runs),
                  (uint32_t)(P.merge_by_part ? cols : (cols + rows - 1) / rows));
  if (P.D == 64)
    hipLaunchKernelGGL(P.f16 ? (paged_merge_kernel<64, true>) : (paged_merge_kernel<64, false>), grid, dim3(256), 0, s, P);
  else
    hipLaunchKernelGGL(P.f16 ? (paged_merge_kernel<128, true>) : (paged_merge_kernel<128, false>), grid, dim3(256), 0, s, P);
  return hipGetLastError();
}

}  // namespace fna2
