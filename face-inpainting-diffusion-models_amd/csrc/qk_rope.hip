// Per-head RMS norm of queries and keys with the position rotation in the same pass, and its backward (include/ifd_ops.h).
//   n = x rstd w, rstd = (mean x^2 + eps)^-1/2; the first `rot` channels in pairs (a, b):
//   y_a = mscale (n_a cos t - n_b sin t), y_b = mscale (n_b cos t + n_a sin t), t = 2 pi pos turns[i]
//   backward: dn = the transposed rotation of dy, dw = sum dn x rstd, u = dn w, dx = rstd (u - x rstd mean(u x rstd))
// Bound by memory: every value is read once and written once. A head's D / 2 channel pairs are spread over a group of
// lanes, V pairs each, both members of a pair in one lane (two vector loads), so only the norm's sum crosses lanes. The
// angle depends on the token and the lane alone: it is computed once per token and reused for every head, and the lane groups
// that hold different heads of a token compute a share of its V angles each and exchange them (one each for eight groups and
// V = 8). It is an fp64 product whose whole and quarter turns are dropped before it is rounded to fp32 (2^-27 of a turn off
// at most); the product's own rounding passes that beyond positions of 2^27 (2^-15 of a turn at 2^40).
// fp32 throughout but for that: sums of D values, the hardware's reciprocal square root (1 ulp), sine and cosine. A workgroup's
// part of dw is an fp32 sum over its tokens and heads, the workgroups' parts are added in fp64: fp32 outputs of the backward
// are 1.1e-7 of their norm off (elementary fp32 operations with fp64 angles and sums: 6.6e-8).
#include <type_traits>
#include "lanes.h"
#include "ops.h"

namespace ifd {

struct QkK {  // strides in bytes
  const char *q, *k, *gq, *gk;  // inputs; gradients of the outputs
  char *oq, *ok;                // outputs (forward) or input gradients (backward)
  const float *wq, *wk;
  const int64_t* pos;
  const double* turns;
  float* part;
  int64_t qs[2], ks[2], gqs[2], gks[2], oqs[2], oks[2], ps[2];
  int qh, kh, gqh, gkh, oqh, okh;  // head strides (host check: a token's heads within 31 bits)
  int ntok, T, Hq, Hk, D, rot, norm, lg, hs, tpw, hsplit;
  float eps, mscale, rD;
};

// A lane's 2 V channels: m[0 .. V) from channel ia on, m[V .. 2V) from ib on. Pair j: interleaved (IL) m[2j], m[2j + 1]
// (ib = ia + V: one run of channels), else m[j], m[V + j].
template <typename T, int V, bool IL, bool BWD>
__global__ __launch_bounds__(256) void qk_rope_kernel(QkK p) {
  typedef T vec __attribute__((ext_vector_type(V)));
  constexpr int ES = sizeof(T);
  __shared__ float red[BWD ? 4 * 2 * 128 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int half = p.rot >> 1;
  const int sub = lane & (p.lg - 1), slot = lane / p.lg;
  const int u = sub * V;  // first channel pair of this lane
  const int tok_sub = slot / p.hs, head0 = slot - tok_sub * p.hs;
  const bool act = u < (p.D >> 1) && tok_sub < p.tpw;
  const bool rotated = act && u < half;
  const int ia = !act ? 0 : IL ? 2 * u : (u < half ? u : p.rot + (u - half));
  const int ib = !act ? 0 : IL ? ia + V : (u < half ? u + half : ia + ((p.D - p.rot) >> 1));
  constexpr int PA = IL ? 2 : 1, PB = IL ? 1 : V;  // member a of pair j is m[PA j], member b m[PA j + PB]
  float w[2][2 * V], dw[BWD ? 2 : 1][2 * V];      // weights and their gradients' sums: queries, keys
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const float* wp = x ? p.wk : p.wq;
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) w[x][j] = 1.f;
    if (wp) {  // (4-byte aligned: vector loads all the same)
      __builtin_memcpy(&w[x][0], wp + ia, 4 * V);
      __builtin_memcpy(&w[x][V], wp + ib, 4 * V);
    }
  }
#pragma unroll
  for (int x = 0; x < (BWD ? 2 : 1); ++x)
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) dw[x][j] = 0.f;

  // item: (group of tpw tokens, share of the heads)
  const int items = (p.ntok + p.tpw - 1) / p.tpw * p.hsplit;
  for (int it = blockIdx.x * 4 + wave; it < items; it += gridDim.x * 4) {
    const int tg = it / p.hsplit, hsh = it - tg * p.hsplit;
    const int tok = tg * p.tpw + tok_sub;
    const bool live = act && tok < p.ntok;
    const int b = live ? tok / p.T : 0, t = live ? tok - b * p.T : 0;
    float cs[V], sn[V];
    if (p.rot) {
      const double ps = (double)p.pos[b * p.ps[0] + t * p.ps[1]];
      const int first = tok_sub * p.hs * p.lg + sub;  // this lane's twin in the token's first group
      for (int j0 = 0; j0 < V; j0 += p.hs) {
        double f = rotated && j0 + head0 < V ? p.turns[u + j0 + head0] * ps : 0.0;
        // turns -> the nearest quarter and the rest, which alone is rounded to fp32 (at most 1/8 turn: 2^-27 off)
        f -= rint(f);
        const double quarter = rint(4.0 * f);
        const int k = (int)quarter;
        float s0, c0;
        sincospif(2.f * (float)fma(quarter, -0.25, f), &s0, &c0);
        float s = k & 1 ? c0 : s0, c = k & 1 ? s0 : c0;
        s *= k & 2 ? -p.mscale : p.mscale;
        c *= (k + 1) & 2 ? -p.mscale : p.mscale;
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j >= j0 && j < j0 + p.hs) {
            cs[j] = __shfl(c, first + (j - j0) * p.lg);
            sn[j] = __shfl(s, first + (j - j0) * p.lg);
          }
      }
    }
    auto heads = [&](auto isk_) {
      constexpr int isk = decltype(isk_)::value;
      const int H = isk ? p.Hk : p.Hq;
      const int64_t xs = isk ? p.kh : p.qh, gs = isk ? p.gkh : p.gqh, os = isk ? p.okh : p.oqh;
      const char* x0 = isk ? p.k + b * p.ks[0] + t * p.ks[1] : p.q + b * p.qs[0] + t * p.qs[1];
      const char* g0 = isk ? p.gk + b * p.gks[0] + t * p.gks[1] : p.gq + b * p.gqs[0] + t * p.gqs[1];
      char* o0 = isk ? p.ok + b * p.oks[0] + t * p.oks[1] : p.oq + b * p.oqs[0] + t * p.oqs[1];
      for (int h0 = hsh * p.hs; h0 < H; h0 += p.hs * p.hsplit) {
        const int hd = h0 + head0;
        const bool on = live && hd < H;
        vec va = {}, vb = {}, ga = {}, gb = {};  // lanes without a head add nothing to the sums
        if (on) {
          const char* x = x0 + hd * xs;
          va = *reinterpret_cast<const vec*>(x + ia * ES);
          vb = *reinterpret_cast<const vec*>(x + ib * ES);
          if (BWD) {
            const char* g = g0 + hd * gs;
            ga = *reinterpret_cast<const vec*>(g + ia * ES);
            gb = *reinterpret_cast<const vec*>(g + ib * ES);
          }
        }
        float m[2 * V], y[2 * V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          m[j] = (float)va[j];
          m[V + j] = (float)vb[j];
          y[j] = (float)ga[j];
          y[V + j] = (float)gb[j];
        }
        float rstd = 1.f;
        if (p.norm) {
          float ss = 0.f;
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) ss = fmaf(m[j], m[j], ss);
          ss = group_sum(ss, p.lg);
          rstd = __builtin_amdgcn_rsqf(fmaf(ss, p.rD, p.eps));  // 1 ulp
        }
        if (!BWD) {
          if (p.norm) {
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) m[j] *= rstd * w[isk][j];
          }
          if (rotated) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float na = m[PA * j], nb = m[PA * j + PB];
              m[PA * j] = na * cs[j] - nb * sn[j];
              m[PA * j + PB] = nb * cs[j] + na * sn[j];
            }
          }
        } else {
          if (rotated) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float na = y[PA * j], nb = y[PA * j + PB];
              y[PA * j] = na * cs[j] + nb * sn[j];
              y[PA * j + PB] = nb * cs[j] - na * sn[j];
            }
          }
          if (p.norm) {
            float dot = 0.f;
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) {
              m[j] *= rstd;
              dw[isk][j] = fmaf(y[j], m[j], dw[isk][j]);
              y[j] *= w[isk][j];
              dot = fmaf(y[j], m[j], dot);
            }
            dot = group_sum(dot, p.lg) * p.rD;
#pragma unroll
            for (int j = 0; j < 2 * V; ++j) y[j] = rstd * (y[j] - m[j] * dot);
          }
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) m[j] = y[j];
        }
        if (on) {
          vec oa, ob;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            oa[j] = (T)m[j];
            ob[j] = (T)m[V + j];
          }
          char* o = o0 + hd * os;
          *reinterpret_cast<vec*>(o + ia * ES) = oa;
          *reinterpret_cast<vec*>(o + ib * ES) = ob;
        }
      }
    };
    heads(std::integral_constant<int, 0>{});
    heads(std::integral_constant<int, 1>{});
  }
  if (BWD && p.norm) {
    // the workgroup's weight gradients: over the head slots of a wave, then over the waves
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) {
        float s = dw[BWD ? x : 0][j];
        for (int o = p.lg; o < 64; o <<= 1) s += __shfl_xor(s, o);
        if (slot == 0 && act) red[(wave * 2 + x) * 128 + (j < V ? ia + j : ib + j - V)] = s;
      }
    __syncthreads();
    const int x = threadIdx.x >> 7, ch = threadIdx.x & 127;
    if (ch < p.D) {
      float s = 0.f;
#pragma unroll
      for (int v = 0; v < 4; ++v) s += red[(v * 2 + x) * 128 + ch];
      p.part[((int64_t)blockIdx.x * 2 + x) * p.D + ch] = s;
    }
  }
}

// dw = the workgroups' sums in a fixed order, in fp64: a workgroup per (queries | keys, 8 channels), 128 walks each
__global__ __launch_bounds__(1024) void qk_dw_kernel(const float* __restrict__ part, int nwg, int D, float* dwq, float* dwk) {
  __shared__ double r[128][8];
  const int c = threadIdx.x & 7, g = threadIdx.x >> 3, ch = blockIdx.x * 8 + c, x = blockIdx.y;
  double s = 0.0;
  if (ch < D) {
#pragma unroll 8
    for (int i = g; i < nwg; i += 128) s += part[((int64_t)i * 2 + x) * D + ch];
  }
  r[g][c] = s;
  __syncthreads();
  for (int o = 64; o; o >>= 1) {
    if (g < o) r[g][c] += r[g + o][c];
    __syncthreads();
  }
  float* o = x ? dwk : dwq;
  if (g == 0 && ch < D && o) o[ch] = (float)r[0][c];
}

// ---------------------------------------------------------------------------------------------- host side
static const char* qk_check(const ifd_qk_args& a) {
  if (!dtype_ok(a.dtype)) return "dtype";
  if (a.B < 0 || a.T < 0 || a.Hq < 0 || a.Hk < 0 || a.D < 1) return "negative or zero sizes";
  if (a.D > 128 || a.D % 2) return "head width: at most 128 and even";
  if (a.rot < 0 || a.rot > a.D || a.rot % 2) return "rotated channels: even, at most the head width";
  if (!(a.eps >= 0.f) || !(a.eps < 3e38f)) return "eps must be finite and not negative";
  const int64_t lim = ((int64_t)1 << 31) / dtype_bytes(a.dtype) - 256;
  for (int64_t s : {a.q_s[2] * a.Hq, a.gq_s[2] * a.Hq, a.dq_s[2] * a.Hq, a.q_out_s[2] * a.Hq, a.k_s[2] * a.Hk,
                    a.gk_s[2] * a.Hk, a.dk_s[2] * a.Hk, a.k_out_s[2] * a.Hk})
    if (s > lim || s < -lim) return "a token's heads reach over more than 2 GiB";
  if ((int64_t)a.Hq + a.Hk > 1 << 20 || (int64_t)a.B * a.T * (a.Hq + a.Hk) >= (int64_t)1 << 31)
    return "sizes: 2^31 head rows and more";
  const int64_t es = dtype_bytes(a.dtype);
  for (const void* t : {a.q, a.k, a.gq, a.gk, (const void*)a.q_out, (const void*)a.k_out, (const void*)a.dq, (const void*)a.dk})
    if (!on(t, es)) return "a tensor's address off its elements";
  if (!on(a.wq, 4) || !on(a.wk, 4) || !on(a.dwq, 4) || !on(a.dwk, 4) || !on(a.pos, 8) || !on(a.turns, 8))
    return "weights, positions or frequencies: an address off its elements";
  return nullptr;
}

// Workgroups: enough to fill the chip, few enough that each walks over many tokens (4 x 4096 x 20 heads x 128 bf16, forward:
// 29.6 us with 1024, 5.7 TB/s; 30.2 with 2048, 36.5 with 512. Backward, where each leaves one partial row of weight
// gradients: 59.5 with 512; 67.3 with 1024, 82.9 with 256)
constexpr int QK_FWD_WGS = 1024, QK_WGS = 512;

static bool vec_ok(int V, int es, const ifd_qk_args& a, bool bwd) {
  if ((a.rot / 2) % V || ((a.D - a.rot) / 2) % V) return false;
  const int al = V * es;
  auto ok = [&](const void* p, const int64_t (&s)[3]) {
    return ((uintptr_t)p % al) == 0 && (s[0] * es) % al == 0 && (s[1] * es) % al == 0 && (s[2] * es) % al == 0;
  };
  if (a.Hq && (!ok(a.q, a.q_s) || (bwd ? !ok(a.gq, a.gq_s) || !ok(a.dq, a.dq_s) : !ok(a.q_out, a.q_out_s)))) return false;
  if (a.Hk && (!ok(a.k, a.k_s) || (bwd ? !ok(a.gk, a.gk_s) || !ok(a.dk, a.dk_s) : !ok(a.k_out, a.k_out_s)))) return false;
  return true;
}

template <typename T, int V, bool IL>
static int run_qk(QkK p, bool bwd, hipStream_t s) {
  const int nl = (p.D / 2 + V - 1) / V;
  p.lg = 1;
  while (p.lg < nl) p.lg <<= 1;
  const int slots = 64 / p.lg, H = std::max(p.Hq, p.Hk);
  p.hs = std::min(H, slots);
  p.tpw = slots / p.hs;
  // few tokens: a token's heads go to several waves
  const int64_t groups = cdiv(p.ntok, p.tpw);
  p.hsplit = groups >= 4096 ? 1 : (int)std::min<int64_t>(cdiv(H, p.hs), cdiv(4096, groups));
  const int64_t wgs = cdiv(groups * p.hsplit, 4);
  if (!bwd) {
    auto kern = qk_rope_kernel<T, V, IL, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)std::min<int64_t>(wgs, QK_FWD_WGS)), dim3(256), 0, s, p);
  } else {
    auto kern = qk_rope_kernel<T, V, IL, true>;
    hipLaunchKernelGGL(kern, dim3((unsigned)std::min<int64_t>(wgs, QK_WGS)), dim3(256), 0, s, p);
  }
  return (int)std::min<int64_t>(wgs, QK_WGS);
}
template <typename T, int V>
static int run_qk(const ifd_qk_args& a, QkK p, bool bwd, hipStream_t s) {
  return a.interleaved ? run_qk<T, V, true>(p, bwd, s) : run_qk<T, V, false>(p, bwd, s);
}

template <typename T>
static int run_qk_v(const ifd_qk_args& a, QkK p, bool bwd, hipStream_t s) {
  constexpr int es = sizeof(T);
  if (es == 2 && vec_ok(8, es, a, bwd)) return run_qk<T, es == 2 ? 8 : 4>(a, p, bwd, s);
  if (vec_ok(4, es, a, bwd)) return run_qk<T, 4>(a, p, bwd, s);
  return run_qk<T, 1>(a, p, bwd, s);
}

static int run_any(const ifd_qk_args& a, bool bwd, float* part, hipStream_t s) {
  const int64_t es = dtype_bytes(a.dtype);
  QkK p = {};
  p.q = (const char*)a.q; p.k = (const char*)a.k; p.gq = (const char*)a.gq; p.gk = (const char*)a.gk;
  p.oq = (char*)(bwd ? a.dq : a.q_out); p.ok = (char*)(bwd ? a.dk : a.k_out);
  p.wq = a.wq; p.wk = a.wk; p.pos = a.pos; p.turns = a.turns; p.part = part;
  p.qh = (int)(a.q_s[2] * es); p.kh = (int)(a.k_s[2] * es); p.gqh = (int)(a.gq_s[2] * es); p.gkh = (int)(a.gk_s[2] * es);
  p.oqh = (int)((bwd ? a.dq_s[2] : a.q_out_s[2]) * es); p.okh = (int)((bwd ? a.dk_s[2] : a.k_out_s[2]) * es);
  p.rD = 1.f / (float)a.D;
  for (int j = 0; j < 2; ++j) {
    p.qs[j] = a.q_s[j] * es; p.ks[j] = a.k_s[j] * es; p.gqs[j] = a.gq_s[j] * es; p.gks[j] = a.gk_s[j] * es;
    p.oqs[j] = (bwd ? a.dq_s[j] : a.q_out_s[j]) * es;
    p.oks[j] = (bwd ? a.dk_s[j] : a.k_out_s[j]) * es;
  }
  p.ps[0] = a.pos_s[0]; p.ps[1] = a.pos_s[1];
  p.ntok = a.B * a.T;
  p.T = a.T; p.Hq = a.Hq; p.Hk = a.Hk; p.D = a.D; p.rot = a.rot; 
  p.norm = a.norm != 0; p.eps = a.eps; p.mscale = a.mscale;
  if (a.dtype == IFD_F32) return run_qk_v<float>(a, p, bwd, s);
  if (a.dtype == IFD_BF16) return run_qk_v<__bf16>(a, p, bwd, s);
  return run_qk_v<_Float16>(a, p, bwd, s);
}

}  // namespace ifd

using namespace ifd;
extern "C" {

int ifd_op_qk_norm_rope(const ifd_qk_args* a, void* stream) {
  IFD_OP_REQUIRE(a != nullptr, "null arguments");
  const char* why = qk_check(*a);
  IFD_OP_REQUIRE(!why, why);
  if (!a->B || !a->T || !(a->Hq + a->Hk)) return 0;
  IFD_OP_REQUIRE((!a->Hq || (a->q && a->q_out)) && (!a->Hk || (a->k && a->k_out)), "a null tensor");
  IFD_OP_REQUIRE(!a->rot || (a->pos && a->turns), "a rotation without positions or frequencies");
  run_any(*a, false, nullptr, (hipStream_t)stream);
  return IFD_LAUNCH_STATUS();
}

int64_t ifd_op_qk_norm_rope_bwd_ws_bytes(const ifd_qk_args* a) {
  return a && !qk_check(*a) && a->norm ? (int64_t)QK_WGS * 2 * a->D * 4 : 0;
}

int ifd_op_qk_norm_rope_bwd(const ifd_qk_args* a, void* ws, int64_t ws_bytes, void* stream) {
  IFD_OP_REQUIRE(a != nullptr, "null arguments");
  const char* why = qk_check(*a);
  IFD_OP_REQUIRE(!why, why);
  const bool none = !a->B || !a->T || !(a->Hq + a->Hk);
  IFD_OP_REQUIRE(none || ((!a->Hq || (a->q && a->gq && a->dq)) && (!a->Hk || (a->k && a->gk && a->dk))), "a null tensor");
  IFD_OP_REQUIRE(none || !a->rot || (a->pos && a->turns), "a rotation without positions or frequencies");
  const int64_t need = ifd_op_qk_norm_rope_bwd_ws_bytes(a);
  IFD_OP_REQUIRE(ws_bytes >= need && (ws || !need), "workspace too small");
  IFD_OP_REQUIRE(on(ws, 4), "the workspace's address is off its elements");
  hipStream_t s = (hipStream_t)stream;
  int nwg = 0;
  if (!none) {
    nwg = run_any(*a, true, (float*)ws, s);
    if (int e = IFD_LAUNCH_STATUS()) return e;
  }
  if (a->norm && (a->dwq || a->dwk)) {
    hipLaunchKernelGGL(qk_dw_kernel, dim3((a->D + 7) / 8, 2), dim3(1024), 0, s, (const float*)ws, nwg, a->D, a->dwq, a->dwk);
    return IFD_LAUNCH_STATUS();
  }
  return 0;
}

}  // extern "C"
