// Per-head RMS norm of queries and keys with the position rotation in the same pass, and its backward (include/ifd_ops.h).
//   n = x rstd w, rstd = (mean x^2 + eps)^-1/2; the first `rot` channels in pairs (a, b):
//   y_a = mscale (n_a cos t - n_b sin t), y_b = mscale (n_b cos t + n_a sin t), t = 2 pi pos turns[i]
//   backward: dn = the transposed rotation of dy, dw = sum dn x rstd, u = dn w, dx = rstd (u - x rstd mean(u x rstd))
// Bound by memory: every value is read once and written once. A head's D / 2 channel pairs are spread over a group of
// lanes, V pairs each, both members of a pair in one lane (two vector loads), so only the norm's sum crosses lanes. The
// angle (fp64 product, whole turns dropped, fp32 sine and cosine: exact for any int64 position that fp64 holds) depends on
// the token and the lane alone: it is computed once per token and reused for every head.
#include "ops.h"

namespace ifd {

template <typename T, int V>
struct QkVec {
  typedef T vec __attribute__((ext_vector_type(V)));
  static __device__ __forceinline__ void load(const char* p, float (&o)[V]) {
    const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = (float)v[j];
  }
  static __device__ __forceinline__ void store(char* p, const float (&o)[V]) {
    vec v;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (T)o[j];
    *reinterpret_cast<vec*>(p) = v;
  }
};
template <typename T>
struct QkVec<T, 1> {
  static __device__ __forceinline__ void load(const char* p, float (&o)[1]) { o[0] = (float)*reinterpret_cast<const T*>(p); }
  static __device__ __forceinline__ void store(char* p, const float (&o)[1]) { *reinterpret_cast<T*>(p) = (T)o[0]; }
};

struct QkK {  // strides in bytes
  const char *q, *k, *gq, *gk;  // inputs; gradients of the outputs
  char *oq, *ok;                // outputs (forward) or input gradients (backward)
  const float *wq, *wk;
  const int64_t* pos;
  const double* turns;
  float* part;
  int64_t qs[3], ks[3], gqs[3], gks[3], oqs[3], oks[3], ps[2];
  int64_t ntok;
  int T, Hq, Hk, D, rot, interleaved, norm, lg, hs, tpw, hsplit;
  float eps, mscale;
};

template <typename T, int V, bool BWD>
__global__ __launch_bounds__(256) void qk_rope_kernel(QkK p) {
  typedef QkVec<T, V> X;
  constexpr int ES = sizeof(T);
  __shared__ float red[BWD ? 4 * 2 * 128 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int H = p.Hq + p.Hk, half = p.rot >> 1;
  const int sub = lane & (p.lg - 1), slot = lane / p.lg;
  const int u = sub * V;  // first channel pair of this lane
  const int tok_sub = slot / p.hs, head0 = slot - tok_sub * p.hs;
  const bool act = u < (p.D >> 1) && tok_sub < p.tpw;
  const bool rotated = u < half;
  // channels of the lane's pairs: ia + j, ib + j; interleaved: pairs (ia + 2j, ia + 2j + 1), read as ia.. and ib = ia + V..
  int ia, ib;
  if (!rotated) {
    ia = p.rot + (u - half);
    ib = ia + ((p.D - p.rot) >> 1);
  } else if (p.interleaved) {
    ia = 2 * u;
    ib = ia + V;
  } else {
    ia = u;
    ib = u + half;
  }
  const bool zip = rotated && p.interleaved;
  float wa[2][V], wb[2][V], da[2][V], db[2][V];  // weights and their gradients' sums: queries, keys
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const float* w = x ? p.wk : p.wq;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int ca = zip ? ia + 2 * j : ia + j, cb = zip ? ca + 1 : ib + j;
      wa[x][j] = act && w ? w[ca] : 1.f;
      wb[x][j] = act && w ? w[cb] : 1.f;
      da[x][j] = db[x][j] = 0.f;
    }
  }
  double tn[V];
#pragma unroll
  for (int j = 0; j < V; ++j) tn[j] = act && rotated ? p.turns[u + j] : 0.0;

  // item: (group of tpw tokens, share of the heads)
  const int64_t items = (p.ntok + p.tpw - 1) / p.tpw * p.hsplit;
  for (int64_t it = (int64_t)blockIdx.x * 4 + wave; it < items; it += (int64_t)gridDim.x * 4) {
    const int64_t tg = it / p.hsplit;
    const int hsh = (int)(it - tg * p.hsplit);
    const int64_t tok = tg * p.tpw + tok_sub;
    const bool live = act && tok < p.ntok;
    const int64_t b = live ? tok / p.T : 0, t = live ? tok - b * p.T : 0;
    float cs[V], sn[V];
    if (p.rot) {
      const double ps = (double)p.pos[b * p.ps[0] + t * p.ps[1]];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        double f = ps * tn[j];
        f -= rint(f);
        float s, c;
        sincospif(2.f * (float)f, &s, &c);
        cs[j] = c * p.mscale;
        sn[j] = s * p.mscale;
      }
    }
    for (int h0 = hsh * p.hs; h0 < H; h0 += p.hs * p.hsplit) {
      const int hd = h0 + head0;
      const bool on = live && hd < H && head0 < p.hs;
      const int isk = hd >= p.Hq, hh = isk ? hd - p.Hq : hd;
      float a[V] = {}, c[V] = {}, ga[V] = {}, gc[V] = {};
      if (on) {
        const char* x = isk ? p.k + b * p.ks[0] + t * p.ks[1] + hh * p.ks[2] : p.q + b * p.qs[0] + t * p.qs[1] + hh * p.qs[2];
        X::load(x + ia * ES, a);
        X::load(x + ib * ES, c);
        if (BWD) {
          const char* g =
              isk ? p.gk + b * p.gks[0] + t * p.gks[1] + hh * p.gks[2] : p.gq + b * p.gqs[0] + t * p.gqs[1] + hh * p.gqs[2];
          X::load(g + ia * ES, ga);
          X::load(g + ib * ES, gc);
        }
      }
      // interleaved: the two loads hold pairs (0 .. V/2 - 1) and (V/2 .. V - 1): separate the members
      auto unzip = [&](float (&x)[V], float (&y)[V]) {
        if (V == 1) return;  // ia, ib = the pair itself
        float m[2 * V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          m[j] = x[j];
          m[V + j] = y[j];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          x[j] = m[2 * j];
          y[j] = m[2 * j + 1];
        }
      };
      auto rezip = [&](float (&x)[V], float (&y)[V]) {
        if (V == 1) return;
        float m[2 * V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          m[2 * j] = x[j];
          m[2 * j + 1] = y[j];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          x[j] = m[j];
          y[j] = m[V + j];
        }
      };
      if (zip) {
        unzip(a, c);
        if (BWD) unzip(ga, gc);
      }
      float rstd = 1.f;
      if (p.norm) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) ss += a[j] * a[j] + c[j] * c[j];
        for (int o = p.lg >> 1; o; o >>= 1) ss += __shfl_xor(ss, o);
        rstd = 1.f / sqrtf(ss / (float)p.D + p.eps);
      }
      float ya[V], yc[V];
      if (!BWD) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float na = p.norm ? a[j] * rstd * (isk ? wa[1][j] : wa[0][j]) : a[j];
          const float nc = p.norm ? c[j] * rstd * (isk ? wb[1][j] : wb[0][j]) : c[j];
          ya[j] = rotated ? na * cs[j] - nc * sn[j] : na;
          yc[j] = rotated ? nc * cs[j] + na * sn[j] : nc;
        }
      } else {
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float na = rotated ? ga[j] * cs[j] + gc[j] * sn[j] : ga[j];
          const float nc = rotated ? gc[j] * cs[j] - ga[j] * sn[j] : gc[j];
          ya[j] = na;
          yc[j] = nc;
          if (p.norm) {
            a[j] *= rstd;
            c[j] *= rstd;
            // (inactive lanes hold zeros)
            if (isk) {
              da[1][j] += na * a[j];
              db[1][j] += nc * c[j];
            } else {
              da[0][j] += na * a[j];
              db[0][j] += nc * c[j];
            }
            ya[j] = na * (isk ? wa[1][j] : wa[0][j]);
            yc[j] = nc * (isk ? wb[1][j] : wb[0][j]);
            dot += ya[j] * a[j] + yc[j] * c[j];
          }
        }
        if (p.norm) {
          for (int o = p.lg >> 1; o; o >>= 1) dot += __shfl_xor(dot, o);
          dot /= (float)p.D;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            ya[j] = rstd * (ya[j] - a[j] * dot);
            yc[j] = rstd * (yc[j] - c[j] * dot);
          }
        }
      }
      if (zip) rezip(ya, yc);
      if (on) {
        char* o = isk ? p.ok + b * p.oks[0] + t * p.oks[1] + hh * p.oks[2]
                      : p.oq + b * p.oqs[0] + t * p.oqs[1] + hh * p.oqs[2];
        X::store(o + ia * ES, ya);
        X::store(o + ib * ES, yc);
      }
    }
  }
  if (BWD && p.norm) {
    // the workgroup's weight gradients: over the head slots of a wave, then over the waves
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float s = da[x][j], r = db[x][j];
        for (int o = p.lg; o < 64; o <<= 1) {
          s += __shfl_xor(s, o);
          r += __shfl_xor(r, o);
        }
        if (slot == 0 && u < (p.D >> 1)) {
          const int ca = zip ? ia + 2 * j : ia + j, cb = zip ? ca + 1 : ib + j;
          red[(wave * 2 + x) * 128 + ca] = s;
          red[(wave * 2 + x) * 128 + cb] = r;
        }
      }
    __syncthreads();
    const int x = threadIdx.x >> 7, ch = threadIdx.x & 127;
    if (ch < p.D) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) s += red[(w * 2 + x) * 128 + ch];
      p.part[((int64_t)blockIdx.x * 2 + x) * p.D + ch] = s;
    }
  }
}

// dw = the workgroups' sums in order, in fp64: one workgroup per (queries | keys, 32 channels), 8 partial walks each
__global__ __launch_bounds__(256) void qk_dw_kernel(const float* __restrict__ part, int nwg, int D, float* dwq, float* dwk) {
  __shared__ double r[8][32];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5, ch = blockIdx.x * 32 + c, x = blockIdx.y;
  double s = 0.0;
  if (ch < D)
    for (int i = g; i < nwg; i += 8) s += part[((int64_t)i * 2 + x) * D + ch];
  r[g][c] = s;
  __syncthreads();
  float* o = x ? dwk : dwq;
  if (g == 0 && ch < D && o) {
    for (int i = 1; i < 8; ++i) s += r[i][c];
    o[ch] = (float)s;
  }
}

// ---------------------------------------------------------------------------------------------- host side
static const char* qk_check(const ifd_qk_args& a) {
  if (!dtype_ok(a.dtype)) return "dtype";
  if (a.B < 0 || a.T < 0 || a.Hq < 0 || a.Hk < 0 || a.D < 1) return "negative or zero sizes";
  if (a.D > 128 || a.D % 2) return "head width: at most 128 and even";
  if (a.rot < 0 || a.rot > a.D || a.rot % 2) return "rotated channels: even, at most the head width";
  if (!(a.eps >= 0.f) || !(a.eps < 3e38f)) return "eps must be finite and not negative";
  if ((int64_t)a.Hq + a.Hk > 1 << 20 || (int64_t)a.B * a.T > (int64_t)1 << 40) return "sizes";
  return nullptr;
}

constexpr int QK_WGS = 1024;  // workgroups of the backward pass (each leaves one partial row of weight gradients)

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

template <typename T, int V>
static int run_qk(QkK p, bool bwd, int64_t ntok, hipStream_t s) {
  const int nl = (p.D / 2 + V - 1) / V;
  p.lg = 1;
  while (p.lg < nl) p.lg <<= 1;
  const int slots = 64 / p.lg, H = p.Hq + p.Hk;
  p.hs = std::min(H, slots);
  p.tpw = slots / p.hs;
  // few tokens: a token's heads go to several waves
  const int64_t groups = cdiv(ntok, p.tpw);
  p.hsplit = groups >= 4096 ? 1 : (int)std::min<int64_t>(cdiv(H, p.hs), cdiv(4096, groups));
  const int64_t wgs = cdiv(groups * p.hsplit, 4);
  if (!bwd) {
    auto kern = qk_rope_kernel<T, V, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)std::min<int64_t>(wgs, 1 << 20)), dim3(256), 0, s, p);
  } else {
    auto kern = qk_rope_kernel<T, V, true>;
    hipLaunchKernelGGL(kern, dim3((unsigned)std::min<int64_t>(wgs, QK_WGS)), dim3(256), 0, s, p);
  }
  return (int)std::min<int64_t>(wgs, QK_WGS);
}

template <typename T>
static int run_qk_v(const ifd_qk_args& a, QkK p, bool bwd, hipStream_t s) {
  constexpr int es = sizeof(T);
  const int64_t ntok = (int64_t)a.B * a.T;
  if (es == 2 && vec_ok(8, es, a, bwd)) return run_qk<T, es == 2 ? 8 : 4>(p, bwd, ntok, s);
  if (vec_ok(4, es, a, bwd)) return run_qk<T, 4>(p, bwd, ntok, s);
  return run_qk<T, 1>(p, bwd, ntok, s);
}

static int run_any(const ifd_qk_args& a, bool bwd, float* part, hipStream_t s) {
  const int64_t es = dtype_bytes(a.dtype);
  QkK p = {};
  p.q = (const char*)a.q; p.k = (const char*)a.k; p.gq = (const char*)a.gq; p.gk = (const char*)a.gk;
  p.oq = (char*)(bwd ? a.dq : a.q_out); p.ok = (char*)(bwd ? a.dk : a.k_out);
  p.wq = a.wq; p.wk = a.wk; p.pos = a.pos; p.turns = a.turns; p.part = part;
  for (int j = 0; j < 3; ++j) {
    p.qs[j] = a.q_s[j] * es; p.ks[j] = a.k_s[j] * es; p.gqs[j] = a.gq_s[j] * es; p.gks[j] = a.gk_s[j] * es;
    p.oqs[j] = (bwd ? a.dq_s[j] : a.q_out_s[j]) * es;
    p.oks[j] = (bwd ? a.dk_s[j] : a.k_out_s[j]) * es;
  }
  p.ps[0] = a.pos_s[0]; p.ps[1] = a.pos_s[1];
  p.ntok = (int64_t)a.B * a.T;
  p.T = a.T; p.Hq = a.Hq; p.Hk = a.Hk; p.D = a.D; p.rot = a.rot; p.interleaved = a.interleaved != 0;
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
  hipStream_t s = (hipStream_t)stream;
  int nwg = 0;
  if (!none) {
    nwg = run_any(*a, true, (float*)ws, s);
    if (int e = IFD_LAUNCH_STATUS()) return e;
  }
  if (a->norm && (a->dwq || a->dwk)) {
    hipLaunchKernelGGL(qk_dw_kernel, dim3((a->D + 31) / 32, 2), dim3(256), 0, s, (const float*)ws, nwg, a->D, a->dwq, a->dwk);
    return IFD_LAUNCH_STATUS();
  }
  return 0;
}

}  // extern "C"
