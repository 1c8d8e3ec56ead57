// Attention backward (include/ifd_ops.h): the probabilities are recomputed from q, k and the forward's log-sum-exp.
//   p = 2^(c s - lse2), dp = dout v^T, ds = p (dp - delta), delta = rowsum(dout out)
//   dq = scale ds k, dk = scale ds^T q, dv = p^T dout
// Two passes, each owning its outputs, so that nothing is added atomically and the result does not depend on timing:
// attn_bwd_q_kernel (a wave owns 32 query rows; three products per score tile) also leaves each row's lse2 and delta for
// attn_bwd_kv_kernel (a wave owns 32 keys; four products). Seven products against the five of one pass with atomics on dq.
// Short calls run both side by side in one launch (attn_bwd_both_kernel). Where there are few workgroups each pass deals its
// walk out in shares (q_split, kv_split), whose fp32 sums attn_bwd_join_kernel adds in order.
// Bound by the matrix units: 2 x 16|4 heads x 4096 x 128 bf16 causal 491 us, 980 TFLOP/s over the seven products (traced, at
// lower clocks: row pass 223, key pass 292, join 23), matrix units busy in 57 and 55 % of the cycles; 16 x 4 x 1024 x 64 fp32
// 487 us, 123 TFLOP/s (traced: 228, 307), busy in 83 and 81 %.
#include "attn_dev.h"

namespace ifd {

// (waves and tiles as in the forward kernel)
template <typename T, int DP, int BK, int AHEAD, bool STATS>
__device__ __forceinline__ void attn_bwd_q(const AttnK& p, lds_c* sm, int wg) {
  typedef AttnTile<T, DP> TL;
  typedef typename TL::frag frag;
  constexpr int NW = 4, KT = BK / 32, TB = BK * TL::ROWB;
  const int nblk = (p.Tq + NW * 32 - 1) / (NW * 32);
  const int blk = wg / p.nsplit_q, sp = wg - blk * p.nsplit_q;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int BH = p.B * p.Hq;
  int bh, qblk;
  if (p.causal) {
    const int r = blk % BH;
    qblk = nblk - 1 - blk / BH;
    bh = (BH & 7) ? r : (r & 7) * (BH >> 3) + (r >> 3);
  } else {
    const int id = xcd_order(blk, BH * nblk);
    bh = id / nblk;
    qblk = id - bh * nblk;
  }
  const int b = bh / p.Hq, hq = bh - b * p.Hq, hk = hq / p.G;
  const int len = seq_len(p, b), qs = q_first(p, b);
  const int q0 = qblk * (NW * 32) + w * 32;
  const int i = q0 + l32;
  const bool ok = i < p.Tq;
  const int lim = ok ? row_limit(p, qs, len, i) : 0;

  frag qf[TL::KS], gf[TL::KS];
  float delta = 0.f;
  {
    const char* rq = p.q + b * p.qb + hq * p.qh + (int64_t)i * p.qt;
    const char* rg = p.dout + b * p.gb + hq * p.gh + (int64_t)i * p.gt;
    const char* ro = p.out + b * p.ob + hq * p.oh + (int64_t)i * p.ot;
#pragma unroll
    for (int ks = 0; ks < TL::KS; ++ks) {
      qf[ks] = TL::gload(rq, ok, ks, h, p.D);
      gf[ks] = TL::gload(rg, ok, ks, h, p.D);
      const frag of = TL::gload(ro, ok, ks, h, p.D);
#pragma unroll
      for (int j = 0; j < TL::CE; ++j) delta = fmaf((float)gf[ks][j], (float)of[j], delta);
    }
    delta += xhalf(delta);
  }
  float lse2 = INFINITY;  // a row that sees no key: every p is 0
  const int64_t srow = ((int64_t)b * p.Hq + hq) * p.Tq + i;
  if (ok) {
    const float l = p.lse[srow];
    if (l != -INFINITY) lse2 = l * 1.4426950408889634f;
    if (lim == 0) delta = 0.f;
    if (STATS && h == 0 && sp == 0) {
      p.ws[srow] = lse2;
      p.ws[(int64_t)p.B * p.Hq * p.Tq + srow] = delta;
    }
  }
  f32x16 acc[TL::DT];
#pragma unroll
  for (int d = 0; d < TL::DT; ++d)
#pragma unroll
    for (int x = 0; x < 16; ++x) acc[d][x] = 0.f;

  const int last = min(p.Tq, (qblk + 1) * (NW * 32)) - 1;
  const int wg_end = row_limit(p, qs, len, last);
  const int w_last = min(p.Tq, q0 + 32) - 1;
  const int w_end = __builtin_amdgcn_readfirstlane(w_last < q0 ? 0 : row_limit(p, qs, len, w_last));
  const int w_all = __builtin_amdgcn_readfirstlane(w_last < q0 ? 0 : row_limit(p, qs, len, q0));
  const int tiles = (wg_end + BK - 1) / BK, per = (tiles + p.nsplit_q - 1) / p.nsplit_q;
  const int tb = sp * per, nt = min(tiles, tb + per);  // this workgroup's tiles: [tb, nt)
  AttnStage<T, DP, BK, NW> sg;
  sg.init(w, lane, p.D);
  const char* kp = p.k + b * p.kb + hk * p.kh;
  const char* vp = p.v + b * p.vb + hk * p.vh;
  auto stage = [&](int t) {
    const int k0 = t * BK, n = min(BK, wg_end - k0);
    lds_c* d = sm + ((t - tb) & 1) * (2 * TB);
    sg.load(kp + (int64_t)k0 * p.kt, p.kt, n, d, w);
    sg.load(vp + (int64_t)k0 * p.vt, p.vt, n, d + TB, w);
  };
  if (tb < nt) {
    stage(tb);
    dma_wait();
    __syncthreads();
  }
  for (int t = tb; t < nt; ++t) {
    if (t + 1 < nt) stage(t + 1);
    const lds_c* kb = sm + ((t - tb) & 1) * (2 * TB);
    const lds_c* vb = kb + TB;
    const int k0 = t * BK;
    if (k0 < w_end) {
      const bool mask = k0 + BK > w_all;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        f32x16 s, dp;
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] = dp[x] = 0.f;
#pragma unroll
        for (int k1 = 0; k1 < TL::KS; k1 += AHEAD) {  // operands are read ahead of the products that take them
          frag ka[AHEAD], va[AHEAD];
#pragma unroll
          for (int x = 0; x < AHEAD; ++x) {
            ka[x] = TL::row(kb, kt * 32, k1 + x, l32, h);
            va[x] = TL::row(vb, kt * 32, k1 + x, l32, h);
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int x = 0; x < AHEAD; ++x)
#pragma unroll
            for (int j = 0; j < TL::A::MS; ++j) {
              s = TL::A::mma(ka[x], qf[k1 + x], j, s);
              dp = TL::A::mma(va[x], gf[k1 + x], j, dp);
            }
        }
        if (mask) {
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (k0 + kt * 32 + 8 * (x >> 2) + 4 * h + (x & 3) >= lim) s[x] = -INFINITY;
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], p.c, -lse2)) * (dp[x] - delta);
        if constexpr (TL::ES == 4) {
          // the products of 32 keys are added up by themselves first, as in the forward kernel (200 rows x 16000 keys x 64:
          // error of dq 8.6e-7 instead of 2.4e-6; 1024 x 1024: 4.8e-7, 7.3e-7)
#pragma unroll
          for (int d = 0; d < TL::DT; ++d) {
            f32x16 z;
#pragma unroll
            for (int x = 0; x < 16; ++x) z[x] = 0.f;
#pragma unroll
            for (int ps = 0; ps < TL::PS; ++ps) {
              const frag f = TL::pack(s, ps), a = TL::col(kb, kt * 32, ps, d, lane);
#pragma unroll
              for (int j = 0; j < TL::A::MS; ++j) z = TL::A::mma(a, f, j, z);
            }
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[d][x] += z[x];
          }
        } else {
#pragma unroll
          for (int ps = 0; ps < TL::PS; ++ps) {
            const frag f = TL::pack(s, ps);
            frag a[TL::DT];
#pragma unroll
            for (int d = 0; d < TL::DT; ++d) a[d] = TL::col(kb, kt * 32, ps, d, lane);
#pragma unroll
            for (int j = 0; j < TL::A::MS; ++j)
#pragma unroll
              for (int d = 0; d < TL::DT; ++d) acc[d] = TL::A::mma(a[d], f, j, acc[d]);
          }
        }
      }
    }
    dma_wait();
    __syncthreads();
  }
  if (!ok) return;
  if (p.nsplit_q > 1) {
    float* po = p.ws_q + ((((int64_t)b * p.Hq + hq) * p.nsplit_q + sp) * p.Tq + i) * DP;
#pragma unroll
    for (int d = 0; d < TL::DT; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = lim ? acc[d][4 * j + e] : 0.f;
        *reinterpret_cast<f32x4*>(po + d * 32 + 8 * j + 4 * h) = v;
      }
    return;
  }
  T* op = reinterpret_cast<T*>(p.dq + b * p.dqb + hq * p.dqh + (int64_t)i * p.dqt);
#pragma unroll
  for (int d = 0; d < TL::DT; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int ch = d * 32 + 8 * j + 4 * h;
      if (ch >= p.D) continue;
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = lim ? acc[d][4 * j + e] * p.scale : 0.f;  // (no key seen: 0, whatever dout holds)
      *reinterpret_cast<typename TL::A::quad*>(op + ch) = __builtin_convertvector(v, typename TL::A::quad);
    }
}

// A workgroup owns NW * 32 keys of one key-value head and walks over the (query head, row tile) pairs of its share:
// with nsplit > 1 the pairs are dealt to nsplit workgroups, whose fp32 sums attn_bwd_join_kernel adds in order.
// FUSED: lse2 and delta of the share's rows are found here, ahead of the walk, instead of read from the row pass.
template <typename T, int DP, int NW, int BQ, bool VL, bool FUSED>
__device__ __forceinline__ void attn_bwd_kv(const AttnK& p, lds_c* sm, int blk) {
  typedef AttnTile<T, DP> TL;
  typedef typename TL::frag frag;
  constexpr int QT = BQ / 32, TB = BQ * TL::ROWB, BUF = 2 * TB + (FUSED ? 0 : 1024);  // Q, dout, lse2[BQ], delta[BQ]
  const int nblk = (p.Tk + NW * 32 - 1) / (NW * 32);
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  // causal: the first key blocks see most rows and go first, a head's on one XCD; else head by head on each XCD
  int sp, kblk, bh;
  if (p.causal) {
    const int n = p.B * p.Hk * p.nsplit;
    const int r = blk % n, x = (n & 7) ? r : (r & 7) * (n >> 3) + (r >> 3);
    kblk = blk / n;
    bh = x / p.nsplit;
    sp = x - bh * p.nsplit;
  } else {
    const int id = xcd_order(blk, nblk * p.B * p.Hk * p.nsplit);
    sp = id % p.nsplit;
    kblk = (id / p.nsplit) % nblk;
    bh = id / p.nsplit / nblk;
  }
  const int b = bh / p.Hk, hk = bh - b * p.Hk;
  const int qs = q_first(p, b), len = row_limit(p, qs, seq_len(p, b), p.Tq - 1);  // keys that some row sees
  const int kb0 = kblk * (NW * 32), key = kb0 + w * 32 + l32;
  const bool ok = key < len;
  // rows [lo, Tq) see this lane's key, [wg_lo, Tq) some key of the workgroup
  auto first_row = [&](int k) {
    const int64_t n = p.causal ? (int64_t)k - qs : 0;
    return n < 0 ? 0 : (n > p.Tq ? p.Tq : (int)n);
  };
  const int lo = first_row(key), wg_lo = first_row(kb0);
  const int row0 = first_row(0);  // row tiles begin here: rows that see no key are not read
  const int w_lo = __builtin_amdgcn_readfirstlane(first_row(kb0 + w * 32));
  const int w_hi = __builtin_amdgcn_readfirstlane(first_row(kb0 + w * 32 + 31));

  frag kf[TL::KS], vf[VL ? 1 : TL::KS];
  const lds_c* vt = sm + 2 * BUF;  // VL: the workgroup's V rows stay in LDS, for want of registers
  lds_c* tab = sm + 2 * BUF + (VL ? NW * 32 * TL::ROWB : 0);  // FUSED: lse2[32], delta[32] of each 32 rows of the share
  {
    const char* rk = p.k + b * p.kb + hk * p.kh + (int64_t)key * p.kt;
    const char* rv = p.v + b * p.vb + hk * p.vh + (int64_t)key * p.vt;
#pragma unroll
    for (int ks = 0; ks < TL::KS; ++ks) {
      kf[ks] = TL::gload(rk, ok, ks, h, p.D);
      if (!VL) vf[VL ? 0 : ks] = TL::gload(rv, ok, ks, h, p.D);
    }
  }
  f32x16 dk[TL::DT], dv[TL::DT];
#pragma unroll
  for (int d = 0; d < TL::DT; ++d)
#pragma unroll
    for (int x = 0; x < 16; ++x) dk[d][x] = dv[d][x] = 0.f;

  const int tq0 = (wg_lo - row0) / BQ, ntq = kb0 < len && wg_lo < p.Tq ? (p.Tq - row0 + BQ - 1) / BQ - tq0 : 0;
  const int64_t all = (int64_t)ntq * p.G;
  const int it0 = (int)(all * sp / p.nsplit), it1 = (int)(all * (sp + 1) / p.nsplit);
  AttnStage<T, DP, BQ, NW> sg;
  sg.init(w, lane, p.D);
  // the next pair to stage: (head of the group, row tile)
  int sg_h = 0, sg_t = 0;
  if (it0 < it1) {
    sg_h = it0 / ntq;
    sg_t = it0 - sg_h * ntq;
  }
  auto stage = [&](int buf) {
    const int hq = hk * p.G + sg_h, r0 = row0 + (tq0 + sg_t) * BQ, n = min(BQ, p.Tq - r0);
    if (++sg_t == ntq) {
      sg_t = 0;
      ++sg_h;
    }
    lds_c* d = sm + buf * BUF;
    sg.load(p.q + b * p.qb + hq * p.qh + (int64_t)r0 * p.qt, p.qt, n, d, w);
    sg.load(p.dout + b * p.gb + hq * p.gh + (int64_t)r0 * p.gt, p.gt, n, d + TB, w);
    if (!FUSED && w < 2) {  // lse2 by wave 0, delta by wave 1
      const float* st = p.ws + (w ? (int64_t)p.B * p.Hq * p.Tq : 0) + ((int64_t)b * p.Hq + hq) * p.Tq + r0;
      dma_word(st, 4 * min(lane, n - 1), d + 2 * TB + w * 512);
    }
  };
  if (it0 < it1) {
    if (VL) {
      AttnStage<T, DP, NW * 32, NW> sv;
      sv.init(w, lane, p.D);
      sv.load(p.v + b * p.vb + hk * p.vh + (int64_t)kb0 * p.vt, p.vt, min(NW * 32, len - kb0), sm + 2 * BUF, w);
    }
    const int h0 = sg_h, t0 = sg_t;
    stage(0);
    if (FUSED) {
      int hq = hk * p.G + h0, tt = t0, qt = w;  // this wave's 32 rows: row tile tt, part qt
      for (int x = w; x < (it1 - it0) * QT; x += NW, qt += NW) {
        for (; qt >= QT; qt -= QT)
          if (++tt == ntq) {
            tt = 0;
            ++hq;
          }
        const int i = row0 + (tq0 + tt) * BQ + qt * 32 + l32;
        const bool in = i < p.Tq;
        const char* rg = p.dout + b * p.gb + hq * p.gh + (int64_t)i * p.gt;
        const char* ro = p.out + b * p.ob + hq * p.oh + (int64_t)i * p.ot;
        float delta = 0.f;
#pragma unroll
        for (int ks = 0; ks < TL::KS; ++ks) {
          const frag gf = TL::gload(rg, in, ks, h, p.D), of = TL::gload(ro, in, ks, h, p.D);
#pragma unroll
          for (int j = 0; j < TL::CE; ++j) delta = fmaf((float)gf[j], (float)of[j], delta);
        }
        delta += xhalf(delta);
        if (h == 0) {
          const float l = in ? p.lse[((int64_t)b * p.Hq + hq) * p.Tq + i] : -INFINITY;
          auto* st = (__attribute__((address_space(3))) float*)(tab + x * 256) + l32;
          st[0] = l == -INFINITY ? INFINITY : l * 1.4426950408889634f;
          st[32] = delta;
        }
      }
    }
    dma_wait();
    if (VL && p.D < DP) {
      // both factors of dp come from LDS here: V's channels past D must be zeros
      __syncthreads();
      const int c0 = p.D / TL::CE, nz = TL::NCH - c0;
      for (int x = tid; x < NW * 32 * nz; x += NW * 64) {
        const int r = x / nz, c = c0 + x - r * nz;
        lds_zero(sm + 2 * BUF + r * TL::ROWB + ((c ^ TL::swz(r)) << 4));
      }
    }
    __syncthreads();
  }
  int buf = 0, t = it0 < it1 ? sg_t - 1 : 0;  // this round's row tile
  if (t < 0) t = ntq - 1;
  for (int it = it0; it < it1; ++it, buf ^= 1, t = t + 1 == ntq ? 0 : t + 1) {
    if (it + 1 < it1) stage(buf ^ 1);
    const lds_c* qb = sm + buf * BUF;
    const lds_c* gb = qb + TB;
    const int r0 = row0 + (tq0 + t) * BQ;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int rr = r0 + qt * 32;
      if (rr + 32 <= w_lo || rr >= p.Tq) continue;
      f32x16 s, dp;
#pragma unroll
      for (int x = 0; x < 16; ++x) s[x] = dp[x] = 0.f;
#pragma unroll
      for (int ks = 0; ks < TL::KS; ++ks) {
        const frag qa = TL::row(qb, qt * 32, ks, l32, h), ga = TL::row(gb, qt * 32, ks, l32, h);
        const frag vb = VL ? TL::row(vt, w * 32, ks, l32, h) : vf[VL ? 0 : ks];
#pragma unroll
        for (int j = 0; j < TL::A::MS; ++j) {
          s = TL::A::mma(qa, kf[ks], j, s);
          dp = TL::A::mma(ga, vb, j, dp);
        }
      }
      if (rr < w_hi || rr + 32 > p.Tq) {  // rows before the key's first, or past the last (copies of it): p = ds = 0
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const int r = rr + 8 * (x >> 2) + 4 * h + (x & 3);
          if (r < lo || r >= p.Tq) s[x] = -INFINITY;
        }
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const lds_c* st = FUSED ? tab + ((it - it0) * QT + qt) * 256 : qb + 2 * TB + 4 * (qt * 32);
        const f32x4 ls = lds_quad(st + 4 * (8 * y + 4 * h));
        const f32x4 de = lds_quad(st + (FUSED ? 128 : 512) + 4 * (8 * y + 4 * h));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int x = 4 * y + e;
          s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], p.c, -ls[e]));
          dp[x] = s[x] * (dp[x] - de[e]);
        }
      }
      if constexpr (TL::ES == 4) {  // the products of 32 rows are added up by themselves first
#pragma unroll
        for (int d = 0; d < TL::DT; ++d) {
          f32x16 zv, zk;
#pragma unroll
          for (int x = 0; x < 16; ++x) zv[x] = zk[x] = 0.f;
#pragma unroll
          for (int ps = 0; ps < TL::PS; ++ps) {
            const frag fp = TL::pack(s, ps), fd = TL::pack(dp, ps);
            const frag ga = TL::col(gb, qt * 32, ps, d, lane), qa = TL::col(qb, qt * 32, ps, d, lane);
#pragma unroll
            for (int j = 0; j < TL::A::MS; ++j) {
              zv = TL::A::mma(ga, fp, j, zv);
              zk = TL::A::mma(qa, fd, j, zk);
            }
          }
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            dv[d][x] += zv[x];
            dk[d][x] += zk[x];
          }
        }
      } else {
#pragma unroll
        for (int ps = 0; ps < TL::PS; ++ps) {
          const frag fp = TL::pack(s, ps), fd = TL::pack(dp, ps);
#pragma unroll
          for (int d = 0; d < TL::DT; ++d) {
            const frag ga = TL::col(gb, qt * 32, ps, d, lane), qa = TL::col(qb, qt * 32, ps, d, lane);
#pragma unroll
            for (int j = 0; j < TL::A::MS; ++j) {
              dv[d] = TL::A::mma(ga, fp, j, dv[d]);
              dk[d] = TL::A::mma(qa, fd, j, dk[d]);
            }
          }
        }
      }
    }
    dma_wait();
    __syncthreads();
  }
  if (key >= p.Tk) return;
  if (p.nsplit > 1) {
    if (!ok) return;
    float* po = p.ws_kv + ((((int64_t)b * p.Hk + hk) * p.nsplit + sp) * p.Tk + key) * (2 * DP);
#pragma unroll
    for (int d = 0; d < TL::DT; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int ch = d * 32 + 8 * j + 4 * h;
        f32x4 a, c;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] = dk[d][4 * j + e];
          c[e] = dv[d][4 * j + e];
        }
        *reinterpret_cast<f32x4*>(po + ch) = a;
        *reinterpret_cast<f32x4*>(po + DP + ch) = c;
      }
    return;
  }
  T* ok_ = reinterpret_cast<T*>(p.dk + b * p.dkb + hk * p.dkh + (int64_t)key * p.dkt);
  T* ov_ = reinterpret_cast<T*>(p.dv + b * p.dvb + hk * p.dvh + (int64_t)key * p.dvt);
#pragma unroll
  for (int d = 0; d < TL::DT; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int ch = d * 32 + 8 * j + 4 * h;
      if (ch >= p.D) continue;
      f32x4 a, c;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = ok ? dk[d][4 * j + e] * p.scale : 0.f;
        c[e] = ok ? dv[d][4 * j + e] : 0.f;
      }
      *reinterpret_cast<typename TL::A::quad*>(ok_ + ch) = __builtin_convertvector(a, typename TL::A::quad);
      *reinterpret_cast<typename TL::A::quad*>(ov_ + ch) = __builtin_convertvector(c, typename TL::A::quad);
    }
}

template <typename T, int DP, int BK, int AHEAD, int OCC>
__global__ __launch_bounds__(256, OCC) void attn_bwd_q_kernel(AttnK p) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  attn_bwd_q<T, DP, BK, AHEAD, true>(p, (lds_c*)smem, blockIdx.x);
}
template <typename T, int DP, int NW, int BQ, bool VL, int OCC>
__global__ __launch_bounds__(NW * 64, OCC) void attn_bwd_kv_kernel(AttnK p) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  attn_bwd_kv<T, DP, NW, BQ, VL, false>(p, (lds_c*)smem, blockIdx.x);
}
// Both passes side by side: the first nq workgroups take rows, the others keys.
template <typename T, int DP, int BK, int AHEAD, int BQ, bool VL, int OCC>
__global__ __launch_bounds__(256, OCC) void attn_bwd_both_kernel(AttnK p, int nq) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  if ((int)blockIdx.x < nq)
    attn_bwd_q<T, DP, BK, AHEAD, false>(p, (lds_c*)smem, blockIdx.x);
  else
    attn_bwd_kv<T, DP, 4, BQ, VL, true>(p, (lds_c*)smem, blockIdx.x - nq);
}

// dk, dv = the shares' sums in order; one thread per four channels of a (key, dk | dv) row. The workgroups from nkv on: dq.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_bwd_join_kernel(AttnK p, int nkv) {
  typedef typename AttnT<T>::quad quad;
  if ((int)blockIdx.x >= nkv) {
    const int64_t g = (int64_t)(blockIdx.x - nkv) * 256 + threadIdx.x, row = g / (DP / 4);
    const int ch = 4 * (int)(g - row * (DP / 4));
    if (row >= (int64_t)p.B * p.Hq * p.Tq || ch >= p.D) return;
    const int64_t bh = row / p.Tq;
    const int i = (int)(row - bh * p.Tq), b = (int)(bh / p.Hq), hq = (int)(bh - (int64_t)b * p.Hq);
    const float* w = p.ws_q + (bh * p.nsplit_q * p.Tq + i) * DP + ch;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.nsplit_q; ++s) v += *reinterpret_cast<const f32x4*>(w + (int64_t)s * p.Tq * DP);
    v *= p.scale;
    *reinterpret_cast<quad*>(reinterpret_cast<T*>(p.dq + b * p.dqb + hq * p.dqh + (int64_t)i * p.dqt) + ch) =
        __builtin_convertvector(v, quad);
    return;
  }
  constexpr int C4 = 2 * DP / 4;
  const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = g / C4;
  if (row >= (int64_t)p.B * p.Hk * p.Tk) return;
  const int c4 = (int)(g - row * C4), isv = c4 >= DP / 4, ch = 4 * (c4 - isv * (DP / 4));
  if (ch >= p.D) return;
  const int64_t bh = row / p.Tk;
  const int key = (int)(row - bh * p.Tk), b = (int)(bh / p.Hk), hk = (int)(bh - (int64_t)b * p.Hk);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (key < row_limit(p, q_first(p, b), seq_len(p, b), p.Tq - 1)) {
    const float* w = p.ws_kv + (bh * p.nsplit * p.Tk + key) * (2 * DP) + isv * DP + ch;
    for (int s = 0; s < p.nsplit; ++s) v += *reinterpret_cast<const f32x4*>(w + (int64_t)s * p.Tk * (2 * DP));
    if (!isv) v *= p.scale;
  }
  T* o = isv ? reinterpret_cast<T*>(p.dv + b * p.dvb + hk * p.dvh + (int64_t)key * p.dvt)
             : reinterpret_cast<T*>(p.dk + b * p.dkb + hk * p.dkh + (int64_t)key * p.dkt);
  *reinterpret_cast<quad*>(o + ch) = __builtin_convertvector(v, quad);
}

// Shares of the row pass, whose workgroups else walk over all keys one after the other: where they are few, up to 128 of them
// with 128 keys in fp32 and 256 in 16 bits, up to 192 with twice as many (us, in one share and so: 2 x 3 heads x
// 1000 x 64 fp32 114, 79; 3 x 4 x 500 x 128 fp32 causal 126, 80; 1 x 4 x 2048 x 64 bf16 causal 48, 35; 1 x 8 x 1024 x 128 bf16
// causal 46, 39, 45 with 256 workgroups; 8 x 4|2 x 300 x 40 fp32 causal 49, 65 with 192 of one or two tiles).
static int q_split(const ifd_attention_args& a) {
  const int64_t nq = (int64_t)a.B * a.Hq * cdiv(a.Tq, 128), tiles = cdiv(a.Tk, 64), few = a.dtype == IFD_F32 ? 2 : 4;
  if (!nq || nq > 128) return 1;
  const int64_t n = std::max(std::min(128 / nq, tiles / few), std::min(192 / nq, tiles / (2 * few)));
  return (int)std::min<int64_t>(std::max<int64_t>(n, 1), 16);
}

// Shares of the key pass: workgroups of 128 keys (two per CU at a time) deal their walk out among each other. With a causal
// mask, whose workgroups are unlike, until they fill the chip twice (2 x 4 heads x 4096 keys x 128: 518 us at 512
// workgroups, 343 at 1024, 362 at 2048); without one only until they fill it once together with the row pass, more would
// only add sums to join (8 x 8 x 512 x 64: 32 us in one share, 46 in two; 1 x 2 x 4096 x 64: 85 us in eight, 108 in four).
// At least four row tiles each; fp32, whose products take eight times as long, two while every workgroup has a CU to
// itself (2 x 4 x 130 x 64: 32 us against 47; past that, 2 x 3 x 1000 x 64, 142 against 121). (Row pass in one share.)
static int kv_split(const ifd_attention_args& a) {
  const int64_t base = std::max<int64_t>((int64_t)a.B * a.Hk * cdiv(a.Tk, 128), 1);
  const int64_t nq = (int64_t)a.B * a.Hq * cdiv(a.Tq, 128) * q_split(a);
  const int64_t tiles = (int64_t)(a.Hq / a.Hk) * cdiv(a.Tq, 64);
  int64_t n = std::min(a.causal ? cdiv(1024, base) : (640 - nq) / base, tiles / 4);
  if (a.dtype == IFD_F32) n = std::max(n, std::min((256 - nq) / base, tiles / 2));
  return (int)std::min<int64_t>(std::max<int64_t>(n, 1), 16);
}

// Short calls run both passes in one launch. Each pass alone leaves most of the chip waiting for its longest workgroups;
// side by side they fill it, for the price of finding lse2 and delta twice (us as two launches, as one: 2 x 8|2 heads x 512
// x 128 bf16 causal 48, 33; 4 x 8 x 256 x 64 fp32 75, 49; 1 x 1 x 16 x 64 22, 5; 16 x 8 x 256 x 128, 1024 workgroups, 39,
// 34). FUSE_ROWS: rows of a share (their lse2 and delta stay in 4 KB of LDS); FUSE_WGS: workgroups of both.
constexpr int FUSE_ROWS = 512, FUSE_WGS = 1024;

template <typename T, int DP>
static int run_bwd(const AttnK& p, hipStream_t s) {
  typedef AttnTile<T, DP> TL;
  constexpr int ROWB = TL::ROWB, BK = ROWB >= 512 ? 32 : 64, OCC = ROWB >= 512 ? 1 : 2;
  constexpr int AHEAD = sizeof(T) == 4 && DP == 64 ? 1 : TL::KS % 4 ? 3 : 4;  // (fp32 has no registers to read ahead into)
  // V in LDS where K, V and both results together pass the registers (the whole backward, in registers and so: 16-bit 2 x
  // 16|4 heads x 4096 x 128 causal 583, 553 us traced; fp32 16 x 4 x 1024 x 64 502, 485 untraced)
  constexpr bool VL = sizeof(T) == 2 ? DP == 128 : DP == 64;
  constexpr int BQ = VL ? 32 : BK;
  constexpr int lds_q = 4 * BK * ROWB, lds_kv = 4 * BQ * ROWB + (VL ? 128 * ROWB : 0);  // (without lse2 and delta)
  const int64_t nq = cdiv(p.Tq, 128) * p.B * p.Hq * p.nsplit_q, nkv = cdiv(p.Tk, 128) * p.B * p.Hk * p.nsplit;
  if (nq && nkv && nq + nkv <= FUSE_WGS && cdiv(cdiv(p.Tq, BQ) * p.G, p.nsplit) * BQ <= FUSE_ROWS) {
    constexpr int lds = std::max(lds_q, lds_kv + FUSE_ROWS * 8);
    static bool attr[kMaxDevices] = {};
    auto kern = attn_bwd_both_kernel<T, DP, BK, AHEAD, BQ, VL, OCC>;
    if (set_lds_attr_once(attr, reinterpret_cast<const void*>(kern), lds) != hipSuccess) return IFD_LAUNCH_STATUS();
    hipLaunchKernelGGL(kern, dim3((unsigned)(nq + nkv)), dim3(256), lds, s, p, (int)nq);
    if (int e = IFD_LAUNCH_STATUS()) return e;
  } else {
    if (nq) {
      static bool attr[kMaxDevices] = {};
      auto kern = attn_bwd_q_kernel<T, DP, BK, AHEAD, OCC>;
      if (set_lds_attr_once(attr, reinterpret_cast<const void*>(kern), lds_q) != hipSuccess) return IFD_LAUNCH_STATUS();
      hipLaunchKernelGGL(kern, dim3((unsigned)nq), dim3(256), lds_q, s, p);
      if (int e = IFD_LAUNCH_STATUS()) return e;
    }
    if (nkv) {
      constexpr int lds = lds_kv + 2048;
      static bool attr[kMaxDevices] = {};
      auto kern = attn_bwd_kv_kernel<T, DP, 4, BQ, VL, OCC>;
      if (set_lds_attr_once(attr, reinterpret_cast<const void*>(kern), lds) != hipSuccess) return IFD_LAUNCH_STATUS();
      hipLaunchKernelGGL(kern, dim3((unsigned)nkv), dim3(256), lds, s, p);
      if (int e = IFD_LAUNCH_STATUS()) return e;
    }
  }
  const int64_t jkv = p.nsplit > 1 ? cdiv((int64_t)p.B * p.Hk * p.Tk * (DP / 2), 256) : 0;
  const int64_t jq = p.nsplit_q > 1 ? cdiv((int64_t)p.B * p.Hq * p.Tq * (DP / 4), 256) : 0;
  if (jkv + jq == 0) return 0;
  auto join = attn_bwd_join_kernel<T, DP>;
  hipLaunchKernelGGL(join, dim3((unsigned)(jkv + jq)), dim3(256), 0, s, p, (int)jkv);
  return IFD_LAUNCH_STATUS();
}

template <typename T>
static int run_bwd_d(const AttnK& p, hipStream_t s) {
  return p.D <= 64 ? run_bwd<T, 64>(p, s) : p.D <= 96 ? run_bwd<T, 96>(p, s) : run_bwd<T, 128>(p, s);
}

}  // namespace ifd

using namespace ifd;
extern "C" {

// floats of workspace up to where the key pass' shares begin (behind lse2 and delta, on 16 bytes), the row pass', and the end
static void bwd_ws(const ifd_attention_args& a, int64_t& kv, int64_t& q, int64_t& all) {
  const int64_t dp = a.D <= 64 ? 64 : a.D <= 96 ? 96 : 128, n = kv_split(a), nq = q_split(a), rows = (int64_t)a.B * a.Hq * a.Tq;
  kv = (2 * rows + 3) & ~(int64_t)3;
  q = kv + (n > 1 ? (int64_t)a.B * a.Hk * n * a.Tk * 2 * dp : 0);
  all = q + (nq > 1 ? rows * nq * dp : 0);
}

int64_t ifd_op_attention_bwd_ws_bytes(const ifd_attention_args* a) {
  if (!a || attention_check(*a) || !a->B) return 0;
  int64_t kv, q, all;
  bwd_ws(*a, kv, q, all);
  return all * 4;
}

int ifd_op_attention_bwd(const ifd_attention_args* a, void* ws, int64_t ws_bytes, void* stream) {
  IFD_OP_REQUIRE(a != nullptr, "null arguments");
  const char* why = attention_check(*a);
  IFD_OP_REQUIRE(!why, why);
  if (!a->B || (!a->Tq && !a->Tk)) return 0;
  if (a->Tq && ((why = attention_tensor_check(*a, a->q, a->q_s)) || (why = attention_tensor_check(*a, a->out, a->out_s)) ||
                (why = attention_tensor_check(*a, a->dout, a->dout_s)) ||
                (why = attention_tensor_check(*a, a->dq, a->dq_s))))
    IFD_OP_REQUIRE(false, why);
  if (a->Tk && ((why = attention_tensor_check(*a, a->k, a->k_s)) || (why = attention_tensor_check(*a, a->v, a->v_s)) ||
                (why = attention_tensor_check(*a, a->dk, a->dk_s)) ||
                (why = attention_tensor_check(*a, a->dv, a->dv_s))))
    IFD_OP_REQUIRE(false, why);
  IFD_OP_REQUIRE(a->lse != nullptr || !a->Tq, "a null lse");
  const int64_t need = ifd_op_attention_bwd_ws_bytes(a);
  IFD_OP_REQUIRE(ws_bytes >= need && (ws || !need) && !((uintptr_t)ws & 15), "workspace too small or not aligned to 16 bytes");
  const int n = kv_split(*a), nq = q_split(*a);
  IFD_OP_REQUIRE(cdiv(a->Tk, 128) * a->B * a->Hk * n < 0x7fffffff && cdiv(a->Tq, 128) * a->B * a->Hq * nq < 0x7fffffff &&
                     (int64_t)a->B * a->Hk * a->Tk < (int64_t)1 << 31,
                 "sizes beyond one launch");
  AttnK p = attention_kernel_args(*a);
  int64_t kv, q, all;
  bwd_ws(*a, kv, q, all);
  p.ws = (float*)ws;
  p.ws_kv = p.ws + kv;
  p.ws_q = p.ws + q;
  p.nsplit = n;
  p.nsplit_q = nq;
  hipStream_t s = (hipStream_t)stream;
  return a->dtype == IFD_F32 ? run_bwd_d<float>(p, s)
                             : a->dtype == IFD_BF16 ? run_bwd_d<__bf16>(p, s) : run_bwd_d<_Float16>(p, s);
}

}  // extern "C"
