// Attention forward: out = softmax(scale q k^T) v and the rows' log-sum-exp (include/ifd_ops.h), one pass over the keys
// with a running maximum and sum.
#include <type_traits>
#include "attn_dev.h"
#include "kernels.h"

namespace ifd {

// The running softmax of 32 query rows (column l32 of the score tile) and their output accumulators.
// Scores are kept in units of log2: p = 2^(c s - m). The reference point m need not be the maximum: a tile's p are first
// taken with the m there is, and only when a lane's sum of them passes LIMIT (or is not a number: the first tile, whose m
// is -inf) are the tile's maxima found, m moved there and O rescaled. The usual tile so needs no maximum, no exchange
// between lanes and no rescaling; p <= LIMIT is exact in fp32 and inside fp16's range.
constexpr float ATTN_LIMIT = 4096.f;

template <typename T, int DP, int KT>
struct AttnRows {
  typedef AttnTile<T, DP> TL;
  typedef typename TL::frag frag;
  f32x16 o[TL::DT];
  float m, l, lo;  // l: this lane's keys only; the two halves are added at the end

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int d = 0; d < TL::DT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    m = -INFINITY;
    l = lo = 0.f;
  }
  static __device__ __forceinline__ float probs(const f32x16 (&s)[KT], float c, float ms, frag (&pf)[KT][TL::PS]) {
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      f32x16 e;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        e[i] = __builtin_amdgcn_exp2f(fmaf(s[kt][i], c, -ms));
        sum[i & 1] += e[i];
      }
#pragma unroll
      for (int ps = 0; ps < TL::PS; ++ps) pf[kt][ps] = TL::pack(e, ps);
    }
    return sum[0] + sum[1];
  }
  // scores -> probabilities as operands. lim: keys [0, lim) of this tile are seen by the row (mask != 0)
  __device__ __forceinline__ void soft(f32x16 (&s)[KT], float c, bool mask, int lim, int h, frag (&pf)[KT][TL::PS]) {
    if (mask) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (kt * 32 + 8 * (i >> 2) + 4 * h + (i & 3) >= lim) s[kt][i] = -INFINITY;
    }
    float sum = probs(s, c, m, pf);
    if (__any(!(sum < ATTN_LIMIT))) {
      float mx = s[0][0];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int i = kt ? 0 : 1; i < 16; ++i) mx = fmaxf(mx, s[kt][i]);
      mx = fmaxf(mx, xhalf(mx)) * c;
      const float mn = fmaxf(m, mx);
      const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= a;
      lo *= a;
#pragma unroll
      for (int d = 0; d < TL::DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= a;
      sum = probs(s, c, m == -INFINITY ? 0.f : m, pf);  // no key seen yet: every p is 2^-inf = 0
    }
    if constexpr (TL::ES == 4) {  // compensated: one rounding less per tile
      const float y = sum - lo, t = l + y;
      lo = (t - l) - y;
      l = t;
    } else {
      l += sum;
    }
  }
  // O^T += V^T P^T. fp32 adds a tile's products up by themselves first: a long row of keys then rounds once per tile and
  // not once per product (300 rows x 3000 keys x 64: error 3.6e-7 instead of 1.0e-6, plain products 5.3e-7, for 0 to 10 %
  // of the time; in the 16-bit types P's own rounding is far larger).
  __device__ __forceinline__ void values(const lds_c* vb, const frag (&pf)[KT][TL::PS], int lane) {
    if constexpr (TL::ES == 4) {
#pragma unroll
      for (int d = 0; d < TL::DT; ++d) {
        f32x16 z;
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = 0.f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int ps = 0; ps < TL::PS; ++ps) {
            const frag a = TL::col(vb, kt * 32, ps, d, lane);
#pragma unroll
            for (int j = 0; j < TL::A::MS; ++j) z = TL::A::mma(a, pf[kt][ps], j, z);
          }
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] += z[i];
      }
    } else {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int ps = 0; ps < TL::PS; ++ps) {
          frag a[TL::DT];
#pragma unroll
          for (int d = 0; d < TL::DT; ++d) a[d] = TL::col(vb, kt * 32, ps, d, lane);
#pragma unroll
          for (int j = 0; j < TL::A::MS; ++j)
#pragma unroll
            for (int d = 0; d < TL::DT; ++d) o[d] = TL::A::mma(a[d], pf[kt][ps], j, o[d]);
        }
    }
  }
};

// Partial results of a row (r = token * G + head of the group) and split: O [DP], reference point, sum, two unused.
template <int DP>
__device__ __forceinline__ float* part_row(const AttnK& p, int b, int hk, int r, int sp) {
  return p.ws + ((((int64_t)b * p.Hk + hk) * p.Tq * p.G + r) * p.nsplit + sp) * (DP + 4);
}

// Many rows. A workgroup's four waves take 32 rows each of one (sequence, head) and share the K and V tiles (BK keys, two
// buffers, the next tile's DMA in flight during this one's products). Per wave and tile: S^T = K Q^T with Q in registers,
// softmax down the registers of each lane (a lane holds one row's scores of half the keys), O^T += V^T P^T.
// SPLIT: the keys are dealt to nsplit workgroups, whose results attn_join_kernel joins.
// Bound by the matrix units, in the 16-bit types with the exponentials beside them (a wave's tile of 64 keys at 64 channels:
// 16 products of 32 cycles, 576 cycles of exponentials, scaling, sums and conversions): 4 x 8 heads x 4096 x 4096 x 64 bf16
// 154 us, 890 TFLOP/s, matrix units busy in 45 % of the cycles (four waves a SIMD, OCC, for four registers spilled: in one
// traced run 179, 189 with three, 202 with two; traced runs of it vary from 162 to 187). fp32 32 x 8 x 256 x 256 x 64 43 us, 101
// TFLOP/s, busy in 70 %: a workgroup has four tiles, and nothing covers its first loads and its last stores.
template <typename T, int DP, int BK, int OCC, bool SPLIT>
__global__ __launch_bounds__(256, OCC) void attn_fwd_kernel(AttnK p) {
  typedef AttnTile<T, DP> TL;
  typedef typename TL::frag frag;
  constexpr int NW = 4, KT = BK / 32, TB = BK * TL::ROWB;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  lds_c* sm = (lds_c*)smem;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  // causal: longest blocks first, a head's blocks on one XCD; else head by head on each XCD
  const int BH = p.B * p.Hq, nblk = (p.Tq + NW * 32 - 1) / (NW * 32);
  const int blk = SPLIT ? blockIdx.x / p.nsplit : blockIdx.x, sp = SPLIT ? blockIdx.x - blk * p.nsplit : 0;
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
  const int lim = i < p.Tq ? row_limit(p, qs, len, i) : 0;

  frag qf[TL::KS];
  {
    const char* rp = p.q + b * p.qb + hq * p.qh + (int64_t)i * p.qt;
#pragma unroll
    for (int ks = 0; ks < TL::KS; ++ks) qf[ks] = TL::gload(rp, i < p.Tq, ks, h, p.D);
  }
  AttnRows<T, DP, KT> st;
  st.init();

  // keys that any row of the workgroup sees, of the wave; and those that all its rows see
  const int last = min(p.Tq, (qblk + 1) * (NW * 32)) - 1;
  const int wg_end = row_limit(p, qs, len, last);
  const int w_last = min(p.Tq, q0 + 32) - 1;
  const int w_end = __builtin_amdgcn_readfirstlane(w_last < q0 ? 0 : row_limit(p, qs, len, w_last));
  const int w_all = __builtin_amdgcn_readfirstlane(w_last < q0 ? 0 : row_limit(p, qs, len, q0));
  int tb = 0, nt = (wg_end + BK - 1) / BK;  // this workgroup's tiles: [tb, nt)
  if (SPLIT) {
    const int per = (nt + p.nsplit - 1) / p.nsplit;
    tb = sp * per;
    nt = min(nt, tb + per);
  }

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
    const int k0 = t * BK;
    if (k0 < w_end) {
      const lds_c* kb = sm + ((t - tb) & 1) * (2 * TB);
      const lds_c* vb = kb + TB;
      f32x16 s[KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int x = 0; x < 16; ++x) s[kt][x] = 0.f;
      // KB steps' operands are read ahead of the products that take them
      constexpr int KB = TL::ROWB == 128 ? 2 : TL::KS % 4 ? 3 : 4;
#pragma unroll
      for (int k1 = 0; k1 < TL::KS; k1 += KB) {
        frag a[KB][KT];
#pragma unroll
        for (int x = 0; x < KB; ++x)
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) a[x][kt] = TL::row(kb, kt * 32, k1 + x, l32, h);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < KB; ++x)
#pragma unroll
          for (int j = 0; j < TL::A::MS; ++j)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) s[kt] = TL::A::mma(a[x][kt], qf[k1 + x], j, s[kt]);
      }
      frag pf[KT][TL::PS];
      st.soft(s, p.c, k0 + BK > w_all, lim - k0, h, pf);
      st.values(vb, pf, lane);
    }
    dma_wait();
    __syncthreads();
  }
  const float l = st.l + xhalf(st.l);
  if (i >= p.Tq) return;
  if (SPLIT) {
    float* po = part_row<DP>(p, b, hk, i * p.G + hq - hk * p.G, sp);
#pragma unroll
    for (int d = 0; d < TL::DT; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = st.o[d][4 * j + e];
        *reinterpret_cast<f32x4*>(po + d * 32 + 8 * j + 4 * h) = v;
      }
    if (h == 0) {
      po[DP] = st.m;
      po[DP + 1] = l;
    }
    return;
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  if (h == 0 && p.lse)
    p.lse[((int64_t)b * p.Hq + hq) * p.Tq + i] =
        l == 0.f ? -INFINITY : (st.m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
  T* op = reinterpret_cast<T*>(p.out + b * p.ob + hq * p.oh + (int64_t)i * p.ot);
#pragma unroll
  for (int d = 0; d < TL::DT; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int ch = d * 32 + 8 * j + 4 * h;
      if (ch >= p.D) continue;
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = st.o[d][4 * j + e] * inv;
      *reinterpret_cast<typename TL::A::quad*>(op + ch) = __builtin_convertvector(v, typename TL::A::quad);
    }
}

// Few rows against many keys. The rows of all query heads of one key-value head (row r = token r / G, head r % G) fill
// one 32-row tile, every key is read once, and the keys are split over the NW waves of a workgroup (each streams its own
// tiles through its own LDS, no barriers) and over `nsplit` workgroups. The waves' results are joined in LDS, the
// workgroups' by attn_join_kernel: O = sum_s 2^(m_s - m) O_s, l likewise.
// Bound by reading the keys: one token against 8 x 4 heads x up to 16384 x 128 bf16, 144 MB, 34 us, 4.3 TB/s, and 5 to join.
template <typename T, int DP, int NW, int BK>
__global__ __launch_bounds__(NW * 64) void attn_split_kernel(AttnK p) {
  typedef AttnTile<T, DP> TL;
  typedef typename TL::frag frag;
  constexpr int KT = BK / 32, TB = BK * TL::ROWB, WB = 4 * TB;  // per wave: two buffers of K and V
  static_assert(32 * DP * 4 + 256 <= WB, "a wave's result fits its tiles' LDS");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  lds_c* sm = (lds_c*)smem + w * WB;
  const int id = xcd_order(blockIdx.x, gridDim.x);
  const int sp = id % p.nsplit;
  int r_ = id / p.nsplit;
  const int rb = r_ % p.nblk;
  r_ /= p.nblk;
  const int hk = r_ % p.Hk, b = r_ / p.Hk;
  const int len = seq_len(p, b), qs = q_first(p, b);
  const int rows = p.Tq * p.G;
  const int r = rb * 32 + l32;
  const bool ok = r < rows;
  const int i = ok ? r / p.G : 0, hq = hk * p.G + (ok ? r - i * p.G : 0);
  const int lim = ok ? row_limit(p, qs, len, i) : 0;
  const int r1 = min(rows, rb * 32 + 32) - 1;  // the last row sees most
  const int end = __builtin_amdgcn_readfirstlane(row_limit(p, qs, len, r1 / p.G));
  const int all = __builtin_amdgcn_readfirstlane(row_limit(p, qs, len, rb * 32 / p.G));
  frag qf[TL::KS];
  {
    const char* rp = p.q + b * p.qb + hq * p.qh + (int64_t)i * p.qt;
#pragma unroll
    for (int ks = 0; ks < TL::KS; ++ks) qf[ks] = TL::gload(rp, ok, ks, h, p.D);
  }
  AttnRows<T, DP, KT> st;
  st.init();
  // this workgroup's tiles: [t0, t1), wave w takes t0 + w, t0 + w + NW, ...
  const int nt = (end + BK - 1) / BK;
  const int per = (nt + p.nsplit - 1) / p.nsplit;
  const int t0 = sp * per, t1 = min(nt, t0 + per);
  AttnStage<T, DP, BK, 1> sg;
  sg.init(0, lane, p.D);
  const char* kp = p.k + b * p.kb + hk * p.kh;
  const char* vp = p.v + b * p.vb + hk * p.vh;
  auto stage = [&](int t, int buf) {
    const int k0 = t * BK, n = min(BK, end - k0);
    lds_c* d = sm + buf * (2 * TB);
    sg.load(kp + (int64_t)k0 * p.kt, p.kt, n, d, 0);
    sg.load(vp + (int64_t)k0 * p.vt, p.vt, n, d + TB, 0);
  };
  int buf = 0;
  if (t0 + w < t1) stage(t0 + w, 0);
  for (int t = t0 + w; t < t1; t += NW) {
    // this tile's DMA is complete once at most the next tile's is outstanding
    if (t + NW < t1) {
      stage(t + NW, buf ^ 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * AttnStage<T, DP, BK, 1>::NI) : "memory");
    } else {
      dma_wait();
    }
    const lds_c* kb = sm + buf * (2 * TB);
    const lds_c* vb = kb + TB;
    const int k0 = t * BK;
    f32x16 s[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
      for (int i2 = 0; i2 < 16; ++i2) s[kt][i2] = 0.f;
#pragma unroll
      for (int ks = 0; ks < TL::KS; ++ks) {
        const frag a = TL::row(kb, kt * 32, ks, l32, h);
#pragma unroll
        for (int j = 0; j < TL::A::MS; ++j) s[kt] = TL::A::mma(a, qf[ks], j, s[kt]);
      }
    }
    frag pf[KT][TL::PS];
    st.soft(s, p.c, k0 + BK > all, lim - k0, h, pf);
    st.values(vb, pf, lane);
    // the reads above are complete before the next round's DMA overwrites this buffer
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    buf ^= 1;
  }
  // the waves' results: m, l of each row, then O [DP][32 rows] in the wave's own (now idle) LDS
  const float l = st.l + xhalf(st.l);
  float* wf = reinterpret_cast<float*>(smem + w * WB);
  __syncthreads();
  if (h == 0) {
    wf[l32] = st.m;
    wf[32 + l32] = l;
  }
#pragma unroll
  for (int d = 0; d < TL::DT; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) wf[64 + (d * 32 + 8 * (j >> 2) + 4 * h + (j & 3)) * 32 + l32] = st.o[d][j];
  __syncthreads();
  float m = -INFINITY;
#pragma unroll
  for (int x = 0; x < NW; ++x) m = fmaxf(m, reinterpret_cast<const float*>(smem + x * WB)[l32]);
  float f[NW], lt = 0.f;
#pragma unroll
  for (int x = 0; x < NW; ++x) {
    const float* xf = reinterpret_cast<const float*>(smem + x * WB);
    f[x] = xf[l32] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(xf[l32] - m);
    lt += f[x] * xf[32 + l32];
  }
  // thread (row l32, group tid / 32): channels group, group + 2 NW, ...
  float* po = p.nsplit > 1 ? part_row<DP>(p, b, hk, r, sp) : nullptr;
  const float inv = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt);
  T* op = reinterpret_cast<T*>(p.out + b * p.ob + hq * p.oh + (int64_t)i * p.ot);
  for (int g = tid >> 5; g < DP / 4; g += 2 * NW) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float* xf = reinterpret_cast<const float*>(smem + x * WB) + 64 + (4 * g) * 32 + l32;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += f[x] * xf[e * 32];
    }
    if (!ok) continue;
    if (po) {
      *reinterpret_cast<f32x4*>(po + 4 * g) = v;
    } else if (4 * g < p.D) {
      v *= inv;
      *reinterpret_cast<typename TL::A::quad*>(op + 4 * g) = __builtin_convertvector(v, typename TL::A::quad);
    }
  }
  if (tid < 32 && ok) {
    if (po) {
      po[DP] = m;
      po[DP + 1] = lt;
    } else {
      p.lse[((int64_t)b * p.Hq + hq) * p.Tq + i] =
          lt == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(lt)) * 0.69314718055994531f;
    }
  }
}

// The splits' partial results in order: W lanes per row, four channels each; the splits' statistics are spread over the
// lanes, so that no load waits for another.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnK p) {
  constexpr int W = DP == 64 ? 16 : 32, U = 64 / W;  // at most 64 splits
  const int li = threadIdx.x & (W - 1), first = threadIdx.x & 63 & ~(W - 1), ch = 4 * li;
  const int64_t row = (int64_t)blockIdx.x * (256 / W) + threadIdx.x / W;
  const int rows = p.Tq * p.G;
  if (row >= (int64_t)p.B * p.Hk * rows) return;
  const int bk = (int)(row / rows), r = (int)(row - (int64_t)bk * rows);
  const int b = bk / p.Hk, hk = bk - b * p.Hk, i = r / p.G, hq = hk * p.G + (r - i * p.G);
  const float* w = part_row<DP>(p, b, hk, r, 0);
  float f[U], ls[U], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int s = u * W + li;
    f[u] = s < p.nsplit ? w[s * (DP + 4) + DP] : -INFINITY;
    ls[u] = s < p.nsplit ? w[s * (DP + 4) + DP + 1] : 0.f;
    m = fmaxf(m, f[u]);
  }
#pragma unroll
  for (int o = W / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
#pragma unroll
  for (int u = 0; u < U; ++u) {
    f[u] = f[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(f[u] - m);
    l += f[u] * ls[u];
  }
#pragma unroll
  for (int o = W / 2; o; o >>= 1) l += __shfl_xor(l, o);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int n = min(p.nsplit - u * W, W);
    auto some = [&](int s0, auto k) {  // (loads past the last split read it again, with a factor of 0)
      f32x4 x[k.value];
#pragma unroll
      for (int e = 0; e < k.value; ++e)
        if (ch < DP) x[e] = *reinterpret_cast<const f32x4*>(w + (u * W + min(s0 + e, n - 1)) * (DP + 4) + ch);
#pragma unroll
      for (int e = 0; e < k.value; ++e) {
        const float fs = __shfl(f[u], first + min(s0 + e, n - 1));
        if (ch < DP && s0 + e < n) v += fs * x[e];
      }
    };
    if (n <= 4) {
      if (n > 0) some(0, std::integral_constant<int, 4>{});
    } else {
      for (int s = 0; s < n; s += 16) some(s, std::integral_constant<int, 16>{});
    }
  }
  v *= l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  if (ch < p.D)
    *reinterpret_cast<typename AttnT<T>::quad*>(reinterpret_cast<T*>(p.out + b * p.ob + hq * p.oh + (int64_t)i * p.ot) + ch) =
        __builtin_convertvector(v, typename AttnT<T>::quad);
  if (li == 0)
    p.lse[((int64_t)b * p.Hq + hq) * p.Tq + i] =
        l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f;
}

// ---------------------------------------------------------------------------------------------- host side
const char* attention_check(const ifd_attention_args& a) {
  if (!dtype_ok(a.dtype)) return "dtype";
  if (a.B < 0 || a.Tq < 0 || a.Tk < 0 || a.Hq < 1 || a.Hk < 1 || a.D < 1) return "negative or zero sizes";
  if (a.Hq % a.Hk) return "the query heads are not a multiple of the key-value heads";
  const int es = (int)dtype_bytes(a.dtype), ce = 16 / es;
  if (a.D > 128 || a.D % ce) return "head width: at most 128, a multiple of 8 (16-bit) or 4 (fp32)";
  if (!(a.scale > 0.f) || !(a.scale < 3e38f)) return "scale must be positive and finite";
  if (a.Tk > 0x3fffffff || (int64_t)a.Tq * (a.Hq / a.Hk) > 0x3fffffff || (int64_t)a.B * a.Hq > 0x3fffffff)
    return "sizes beyond 2^30 rows";
  if (!on(a.lse, 4) || !on(a.kv_len, 4) || !on(a.q_start, 4)) return "lse, kv_len or q_start: an address off its elements";
  return nullptr;
}

const char* attention_tensor_check(const ifd_attention_args& a, const void* p, const int64_t (&s)[3]) {
  const int es = (int)dtype_bytes(a.dtype);
  if (!p) return "a null tensor";
  if ((uintptr_t)p & 15) return "tensors must be aligned to 16 bytes";
  for (int j = 0; j < 3; ++j)
    if ((s[j] * es) & 15) return "strides must be multiples of 16 bytes";
  if (s[1] < 0 || s[1] * es >= (int64_t)1 << 24) return "token stride negative or 16 MiB and more";
  return nullptr;
}

struct FwdPlan {
  bool few;  // attn_split_kernel, else attn_fwd_kernel
  int dp, nsplit;
  int64_t wgs;
};

// Keys of a tile of attn_fwd_kernel
constexpr int rows_tile(int dp, int es) { return attn_row_bytes(dp, es) >= 512 ? 32 : 64; }

// Which kernel, and into how many shares of the keys. attn_split_kernel reads every key once for all heads of a group, but
// its waves share no tiles: it is taken for up to 32 rows a head, or 128 rows a group of narrow heads (us, it against
// attn_fwd_kernel: 2 x 8|4 heads x 24 x 3000 x 96 bf16 13, 18; 8 x 8|4 x 64 x 700 x 64 fp32 19, 36; the other way round
// 4 x 8|2 x 100 x 4096 x 128 bf16 39, 27; 2 x 4|1 x 120 x 16000 x 64 fp16 30, 22). attn_fwd_kernel shares the keys out while
// its workgroups would fill half the chip's CUs at most: to two a CU (in one share and in this many: 4 x 8 x 200 x 8192 x 64
// bf16 103, 36; 3 x 6|3 x 500 x 3000 x 80 fp32 348, 131; 2 x 8 x 1024 x 4096 x 64 fp16 58, 38; with 256 workgroups in one
// share already, 4 x 8 x 1024 x 1024 x 64, two take 29 instead of 21), of eight tiles at least, four in fp32, whose tiles
// take longer to multiply (4 x 8|2 x 100 x 4096 x 128 bf16 27 in shares of eight tiles, 30 of four; 2 x 4 x 700 x 128 fp32
// causal 62 and 37). fp32 heads of 65 to 96 channels, whose tiles multiply faster for as much to join, take four only up to
// one workgroup a CU (2 x 4 x 700 x 80 causal 51 in shares of eight tiles, 32 of four; 1 x 2 x 2000 x 80 47 as 256 workgroups,
// 52 as 480; but 3 x 3 x 500 x 3000 x 80 77 and 64).
// attn_split_kernel's shares: 256 workgroups or the next multiple above (a workgroup's LDS lets one into a CU at a time, so
// that group counts which do not divide 256 run a second, partly filled round; not measured), eight tiles each at least.
static FwdPlan fwd_plan(const ifd_attention_args& a) {
  const int G = a.Hq / a.Hk, es = (int)dtype_bytes(a.dtype);
  FwdPlan r;
  const int64_t rows = (int64_t)a.Tq * G;
  r.few = a.Tq <= 32 || rows <= (a.D <= 64 ? 128 : 32);
  if (!r.few) {
    r.dp = a.D <= 64 ? 64 : a.D <= 96 ? 96 : 128;
    r.wgs = cdiv(a.Tq, 128) * a.B * a.Hq;
    const int64_t tiles = cdiv(a.Tk, rows_tile(r.dp, es));
    int64_t n = es == 4 ? tiles / 4 : tiles / 8;
    if (es == 4 && r.dp == 96 && r.wgs <= 128) n = std::max(tiles / 8, std::min(n, 256 / r.wgs));
    r.nsplit = r.wgs > 128 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>({512 / r.wgs, n, 64}));
  } else {
    r.dp = a.D <= 64 ? 64 : 128;
    r.wgs = cdiv(rows, 32) * a.B * a.Hk;
    const int64_t tiles = cdiv(a.Tk, r.dp * es == 128 ? 64 : 32);
    r.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({cdiv(256, r.wgs), cdiv(tiles, 8), 64}));
  }
  r.wgs *= r.nsplit;
  return r;
}

AttnK attention_kernel_args(const ifd_attention_args& a) {
  const int es = (int)dtype_bytes(a.dtype);
  AttnK p = {};
  p.q = (const char*)a.q; p.k = (const char*)a.k; p.v = (const char*)a.v;
  p.out = (char*)a.out; p.lse = a.lse; p.kv_len = a.kv_len; p.q_start = a.q_start;
  p.qb = a.q_s[0] * es; p.qt = (int)(a.q_s[1] * es); p.qh = a.q_s[2] * es;
  p.kb = a.k_s[0] * es; p.kt = (int)(a.k_s[1] * es); p.kh = a.k_s[2] * es;
  p.vb = a.v_s[0] * es; p.vt = (int)(a.v_s[1] * es); p.vh = a.v_s[2] * es;
  p.ob = a.out_s[0] * es; p.ot = (int)(a.out_s[1] * es); p.oh = a.out_s[2] * es;
  p.dout = (const char*)a.dout; p.dq = (char*)a.dq; p.dk = (char*)a.dk; p.dv = (char*)a.dv;
  p.gb = a.dout_s[0] * es; p.gt = (int)(a.dout_s[1] * es); p.gh = a.dout_s[2] * es;
  p.dqb = a.dq_s[0] * es; p.dqt = (int)(a.dq_s[1] * es); p.dqh = a.dq_s[2] * es;
  p.dkb = a.dk_s[0] * es; p.dkt = (int)(a.dk_s[1] * es); p.dkh = a.dk_s[2] * es;
  p.dvb = a.dv_s[0] * es; p.dvt = (int)(a.dv_s[1] * es); p.dvh = a.dv_s[2] * es;
  p.B = a.B; p.Tq = a.Tq; p.Tk = a.Tk; p.Hq = a.Hq; p.Hk = a.Hk; p.D = a.D; p.G = a.Hq / a.Hk;
  p.causal = a.causal != 0;
  p.scale = a.scale;
  p.c = a.scale * 1.4426950408889634f;
  return p;
}

template <typename T, int DP, bool SPLIT>
static int run_rows(const AttnK& p, int64_t wgs, hipStream_t s) {
  constexpr int ROWB = AttnTile<T, DP>::ROWB, BK = rows_tile(DP, sizeof(T)), OCC = ROWB == 128 ? 4 : ROWB == 256 ? 2 : 1;
  constexpr int lds = 4 * BK * ROWB;
  static bool attr[kMaxDevices] = {};
  auto kern = attn_fwd_kernel<T, DP, BK, OCC, SPLIT>;
  if (set_lds_attr_once(attr, reinterpret_cast<const void*>(kern), lds) != hipSuccess) return IFD_LAUNCH_STATUS();
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(256), lds, s, p);
  return IFD_LAUNCH_STATUS();
}

template <typename T, int DP>
static int run_few(const AttnK& p, int64_t wgs, hipStream_t s) {
  constexpr int ROWB = DP * (int)sizeof(T);
  constexpr int BK = ROWB == 128 ? 64 : 32, NW = ROWB >= 512 ? 2 : 4;
  constexpr int lds = NW * 4 * BK * ROWB;
  static bool attr[kMaxDevices] = {};
  auto kern = attn_split_kernel<T, DP, NW, BK>;
  if (set_lds_attr_once(attr, reinterpret_cast<const void*>(kern), lds) != hipSuccess) return IFD_LAUNCH_STATUS();
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(NW * 64), lds, s, p);
  return IFD_LAUNCH_STATUS();
}

template <typename T, int DP>
static int run_fwd_d(const FwdPlan& pl, const AttnK& p, hipStream_t s) {
  int e;
  if constexpr (DP == 96)
    e = pl.nsplit > 1 ? run_rows<T, DP, true>(p, pl.wgs, s) : run_rows<T, DP, false>(p, pl.wgs, s);
  else
    e = pl.few ? run_few<T, DP>(p, pl.wgs, s)
               : pl.nsplit > 1 ? run_rows<T, DP, true>(p, pl.wgs, s) : run_rows<T, DP, false>(p, pl.wgs, s);
  if (e || pl.nsplit == 1) return e;
  auto join = attn_join_kernel<T, DP>;
  hipLaunchKernelGGL(join, dim3((unsigned)cdiv((int64_t)p.B * p.Hq * p.Tq, DP == 64 ? 16 : 8)), dim3(256), 0, s, p);
  return IFD_LAUNCH_STATUS();
}

template <typename T>
static int run_fwd(const FwdPlan& pl, AttnK p, hipStream_t s) {
  p.nblk = (int)cdiv((int64_t)p.Tq * p.G, 32);  // (attn_split_kernel's row tiles)
  p.nsplit = pl.nsplit;
  return pl.dp == 64 ? run_fwd_d<T, 64>(pl, p, s) : pl.dp == 96 ? run_fwd_d<T, 96>(pl, p, s) : run_fwd_d<T, 128>(pl, p, s);
}

// The UNet's QKVAttention (code/nn.py:222-235) on qkv [N][T][3C]: heads of 64 channels at offsets 0, C, 2C; queries and keys
// carry `scale` each. In one share however few the workgroups: an image's result then does not depend on the batch it is in,
// and the call needs no workspace (what shares would gain at batch 1 is not measured).
int launch_attention_rows(const float* qkv, int N, int T, int C, float scale, float* out, hipStream_t s) {
  AttnK p = {};
  p.q = (const char*)qkv; p.k = (const char*)(qkv + C); p.v = (const char*)(qkv + 2 * C);
  p.out = (char*)out;
  p.qb = p.kb = p.vb = (int64_t)T * 3 * C * 4; p.ob = (int64_t)T * C * 4;
  p.qt = p.kt = p.vt = 3 * C * 4; p.ot = C * 4;
  p.qh = p.kh = p.vh = p.oh = 64 * 4;
  p.B = N; p.Tq = p.Tk = T; p.Hq = p.Hk = C / 64; p.D = 64; p.G = 1;
  p.scale = scale * scale;
  p.c = p.scale * 1.4426950408889634f;
  return run_rows<float, 64, false>(p, cdiv(T, 128) * N * (C / 64), s);
}

}  // namespace ifd

using namespace ifd;
extern "C" {

int64_t ifd_op_attention_ws_bytes(const ifd_attention_args* a) {
  if (!a || attention_check(*a) || !a->B || !a->Tq) return 0;
  const FwdPlan pl = fwd_plan(*a);
  return pl.nsplit == 1 ? 0 : (int64_t)a->B * a->Hq * a->Tq * pl.nsplit * (pl.dp + 4) * 4;
}

int ifd_op_attention(const ifd_attention_args* a, void* ws, int64_t ws_bytes, void* stream) {
  IFD_OP_REQUIRE(a != nullptr, "null arguments");
  const char* why = attention_check(*a);
  IFD_OP_REQUIRE(!why, why);
  if (!a->B || !a->Tq) return 0;
  if ((why = attention_tensor_check(*a, a->q, a->q_s)) || (why = attention_tensor_check(*a, a->out, a->out_s)) ||
      (a->Tk && ((why = attention_tensor_check(*a, a->k, a->k_s)) || (why = attention_tensor_check(*a, a->v, a->v_s)))))
    IFD_OP_REQUIRE(false, why);
  IFD_OP_REQUIRE(a->lse != nullptr, "a null lse");
  const int64_t need = ifd_op_attention_ws_bytes(a);
  IFD_OP_REQUIRE(ws_bytes >= need && (ws || !need) && !((uintptr_t)ws & 15), "workspace too small or not aligned to 16 bytes");
  const FwdPlan pl = fwd_plan(*a);
  IFD_OP_REQUIRE(pl.wgs < 0x7fffffff, "sizes beyond one launch");
  AttnK p = attention_kernel_args(*a);
  p.ws = (float*)ws;
  hipStream_t s = (hipStream_t)stream;
  return a->dtype == IFD_F32 ? run_fwd<float>(pl, p, s)
                             : a->dtype == IFD_BF16 ? run_fwd<__bf16>(pl, p, s) : run_fwd<_Float16>(pl, p, s);
}

}  // extern "C"
