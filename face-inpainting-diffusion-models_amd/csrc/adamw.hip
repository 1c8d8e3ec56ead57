// AdamW over many tensors, states in 32 or in 8 bits, with the gradients' global norm (include/ifd_ops.h).
//   g' = c g; m = b1 m + (1 - b1) g'; v = b2 v + (1 - b2) g'^2;
//   p = p (1 - lr wd) - lr / (1 - b1^k) m / (sqrt(v) / sqrt(1 - b2^k) + eps)
// Bound by memory: 16 bytes a value with fp32 tensors and 8-bit states, 28 with 32-bit states, plus the norm's own pass
// over the gradients. The tensors' addresses travel in the kernel arguments (128 tensors a launch): no table to upload,
// nothing kept between steps. 93.6 M values, 8-bit states: step 289 us, 5.2 TB/s; norm 120. A wave owns blocks of 256
// values, four per lane; an 8-bit state's scale is its block's.
//
// 8-bit states. One byte is a small float, with one fp32 scale per block of 256 (largest magnitude / 1.875):
//   m: sign, 4 exponent bits, 3 fraction bits: 2^(e - 15) (1 + f / 8);  v: 5 exponent bits, 3 fraction bits: 2^(e - 31)
//   (1 + f / 8); byte 0 is 0. A relative step of 1/8 at every magnitude: v spans 2^31 below its block's largest value.
// The new byte is the value cut to 3 fraction bits after adding 16 random bits below them, so that it is right on average:
// with b2 = 0.999 v moves by less than half a step per update, and rounding to nearest would never let it fall. A v > 0
// never becomes 0 (the step would divide by eps). The random bits are a hash of the element's index and the step's key.
// Everything that decides a byte is computed in fp64 (full rate here), so it does not depend on how the compiler orders
// fp32 roundings; the step itself uses the moments before they are rounded, in fp32.
#include <cmath>
#include "lanes.h"
#include "ops.h"

namespace ifd {

constexpr int AW_T = 128;     // tensors of a launch (its tables fill the 4 KB of kernel arguments)
constexpr int64_t AW_MAX = (int64_t)1 << 31;  // values of a table entry: a longer tensor takes several
constexpr int AW_CHUNK = 16;  // blocks of a workgroup (93.6 M values, norm, step and values: 596 us; 604 with 8, 597 with 32)

struct AwTab {
  const void* p[AW_T];
  const void* g[AW_T];
  unsigned n[AW_T];
  int chunk0[AW_T];     // first workgroup of the tensor
  int block0[AW_T];     // first state block, relative to AwArgs::block0
  uint8_t types[AW_T];  // parameter's | gradient's << 4
  int count;
};
struct AwArgs {
  void *m, *v;
  float *ms, *vs;
  const double* clip;  // {norm, coefficient} or null
  int64_t block0;
  double b1, w1, b2, w2;
  float decay, step, eps, rbc2s;
  unsigned key;
};

// the tensor of workgroup `wg`: the last one whose first workgroup is not past it
__device__ __forceinline__ int aw_find(const AwTab& t, int wg) {
  const int lane = threadIdx.x & 63;
  int n = 0;
#pragma unroll
  for (int o = 0; o < AW_T; o += 64) n += __popcll(__ballot(o + lane < t.count && t.chunk0[min(o + lane, AW_T - 1)] <= wg));
  return __builtin_amdgcn_readfirstlane(n - 1);
}

// Values [i, i + 4) of a block, of which `left` lie inside the tensor (4: all). `block` is the same for the wave, and so is
// `whole`: a block inside the tensor whose address allows vector loads.
template <typename T>
struct AwMem {
  typedef T quad __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ f32x4 load(const void* block, int i, int left, bool whole) {
    const T* q = reinterpret_cast<const T*>(block) + i;
    if (whole) return __builtin_convertvector(*reinterpret_cast<const quad*>(q), f32x4);
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) r[j] = (float)q[j];
    return r;
  }
  static __device__ __forceinline__ void store(void* block, int i, int left, bool whole, f32x4 v) {
    T* q = reinterpret_cast<T*>(block) + i;
    const quad x = __builtin_convertvector(v, quad);
    if (whole) {
      *reinterpret_cast<quad*>(q) = x;
      return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) q[j] = x[j];
  }
};
__device__ __forceinline__ int aw_bytes(int dt) { return dt == IFD_F32 ? 4 : 2; }
__device__ __forceinline__ f32x4 aw_load(const void* base, int dt, int bi, int lane, int64_t n) {
  const char* b = reinterpret_cast<const char*>(base) + (int64_t)bi * (256 * aw_bytes(dt));
  const int64_t left = n - (int64_t)bi * 256;
  const bool whole = left >= 256 && !((uintptr_t)b & (4 * aw_bytes(dt) - 1));
  const int l4 = (int)(left < 256 ? left : 256) - 4 * lane;
  if (dt == IFD_F32) return AwMem<float>::load(b, 4 * lane, l4, whole);
  if (dt == IFD_BF16) return AwMem<__bf16>::load(b, 4 * lane, l4, whole);
  return AwMem<_Float16>::load(b, 4 * lane, l4, whole);
}
__device__ __forceinline__ void aw_store(void* base, int dt, int bi, int lane, int64_t n, f32x4 v) {
  char* b = reinterpret_cast<char*>(base) + (int64_t)bi * (256 * aw_bytes(dt));
  const int64_t left = n - (int64_t)bi * 256;
  const bool whole = left >= 256 && !((uintptr_t)b & (4 * aw_bytes(dt) - 1));
  const int l4 = (int)(left < 256 ? left : 256) - 4 * lane;
  if (dt == IFD_F32) return AwMem<float>::store(b, 4 * lane, l4, whole, v);
  if (dt == IFD_BF16) return AwMem<__bf16>::store(b, 4 * lane, l4, whole, v);
  return AwMem<_Float16>::store(b, 4 * lane, l4, whole, v);
}

// multiply / xor-shift mix (the multipliers: 2^32 times the fractions of the golden ratio, sqrt 2 and sqrt 3, odd)
__host__ __device__ __forceinline__ unsigned aw_mix(unsigned x) {
  x *= 0x9E3779B9u;
  x ^= x >> 15;
  x *= 0x6A09E667u;
  x ^= x >> 13;
  x *= 0xBB67AE85u;
  return x ^ (x >> 16);
}

// 1 / x to the last bit or so: the hardware's estimate and two Newton steps
__device__ __forceinline__ double recip(double x) {
  double r = __builtin_amdgcn_rcp(x);
  r = fma(r, fma(-x, r, 1.0), r);
  return fma(r, fma(-x, r, 1.0), r);
}
// NaN if one of the four is, else x
__device__ __forceinline__ float nan_or(float x, f32x4 v) {
  const float t = __builtin_elementwise_maximum(__builtin_elementwise_maximum(v[0], v[1]),
                                                __builtin_elementwise_maximum(v[2], v[3]));
  return t != t ? t : x;
}
__device__ __forceinline__ double hi_double(unsigned hi) { return __hiloint2double((int)hi, 0); }
__device__ __forceinline__ double m_value(unsigned c) {  // without the scale
  const unsigned k = c & 127u;
  return hi_double(k ? (0x3F000000u + (k << 17)) | ((c & 128u) << 24) : 0u);
}
__device__ __forceinline__ double v_value(unsigned c) { return hi_double(c ? 0x3E000000u + (c << 17) : 0u); }

// The byte of y = |x| / scale: the random bits lie in the double's high word, so the low word never decides. What lies under
// the smallest value (1.125 2^-bias) is that value; for m, at random, that or 0.
__device__ __forceinline__ unsigned m_code(double x, double inv, unsigned r16) {
  const double y = fabs(x) * inv;
  const unsigned hi = (unsigned)__double2hiint(y), tiny = 0x3F020000u;
  unsigned k = min(((max(hi, tiny) + (r16 << 1)) >> 17) - ((1023u - 15u) << 3), 127u);
  if (__any(hi < tiny)) {  // (rare: no lane pays for it otherwise)
    const double t = 0x1.2p-15;
    if (y * 65536.0 + t * (double)r16 < t * 65536.0) k = 0;
  }
  return k ? k | (((unsigned)__double2hiint(x) >> 24) & 128u) : 0u;
}
__device__ __forceinline__ unsigned v_code(double x, double inv, unsigned r16) {
  const double y = x * inv;
  const unsigned hi = (unsigned)__double2hiint(y), tiny = 0x3E020000u;
  const unsigned k = min(((max(hi, tiny) + (r16 << 1)) >> 17) - ((1023u - 31u) << 3), 255u);
  return y > 0.0 ? k : 0u;
}

template <int BITS>
__global__ __launch_bounds__(256) void adamw_multi_kernel(const AwTab t, const AwArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ti = aw_find(t, blockIdx.x);
  const int64_t n = t.n[ti];
  const int pt = t.types[ti] & 15, gt = t.types[ti] >> 4;
  void* pp = const_cast<void*>(t.p[ti]);
  const void* gp = t.g[ti];
  double coef = 1.0;
  if (a.clip) {
    const double norm = a.clip[0];
    if (!(norm < __builtin_huge_val())) return;  // a NaN or infinite gradient: no step
    coef = a.clip[1];
  }
  const double w1 = a.w1 * coef, w2 = a.w2 * (coef * coef);
  const int nblk = (int)((n + 255) >> 8);
  const int b0 = (blockIdx.x - t.chunk0[ti]) * AW_CHUNK;
  for (int bi = b0 + wave; bi < min(nblk, b0 + AW_CHUNK); bi += 4) {
    const int left = (int)min(n - (int64_t)bi * 256, (int64_t)256) - 4 * lane;  // this lane's values inside the tensor
    const int64_t blk = a.block0 + t.block0[ti] + bi, e = blk * 256;
    const f32x4 p0 = aw_load(pp, pt, bi, lane, n), g0 = aw_load(gp, gt, bi, lane, n);
    f32x4 mf, vf;
    if (BITS == 8) {
      unsigned* mc = reinterpret_cast<unsigned*>(reinterpret_cast<unsigned char*>(a.m) + e);
      unsigned* vc = reinterpret_cast<unsigned*>(reinterpret_cast<unsigned char*>(a.v) + e);
      const unsigned cm = mc[lane], cv = vc[lane];
      const double sm = a.b1 * (double)a.ms[blk], sv = a.b2 * (double)a.vs[blk];
      double m[4], v[4];
      double xm = 0.0, xv = 0.0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double g = g0[j];
        m[j] = fma(m_value((cm >> (8 * j)) & 255u), sm, w1 * g);
        v[j] = fma(v_value((cv >> (8 * j)) & 255u), sv, w2 * (g * g));
        mf[j] = (float)m[j];
        vf[j] = (float)v[j];
        xm = fmax(xm, fabs(m[j]));
        xv = fmax(xv, v[j]);
      }
      // the scale rounds max |x| / 1.875 to fp32: rounding keeps order, so the largest rounded value of the lanes is it.
      // fmax drops a NaN: it is found in the fp32 moments, where a maximum that keeps it is one instruction.
      const float am = wave_max_nonneg(nan_or((float)(xm * (1.0 / 1.875)), mf));
      const float av = wave_max_nonneg(nan_or((float)(xv * (1.0 / 1.875)), vf));
      const double im = am > 0.f ? recip(am) : 0.0, iv = av > 0.f ? recip(av) : 0.0;
      unsigned nm = 0, nv = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const unsigned r = aw_mix((unsigned)e + 4u * lane + j + a.key);
        nm |= m_code(m[j], im, r & 0xFFFFu) << (8 * j);
        nv |= v_code(v[j], iv, r >> 16) << (8 * j);
      }
      if (left < 4) {  // what lies behind the tensor's end stays 0
        const unsigned in = left > 0 ? (1u << (8 * left)) - 1 : 0u;
        nm &= in;
        nv &= in;
      }
      mc[lane] = nm;
      vc[lane] = nv;
      if (lane == 0) {
        a.ms[blk] = am;
        a.vs[blk] = av;
      }
    } else {
      f32x4* mm = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(a.m) + e);
      f32x4* vv = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(a.v) + e);
      const float w1f = (float)a.w1, b2 = (float)a.b2, w2f = (float)a.w2, c = (float)coef;
      mf = mm[lane];
      vf = vv[lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float g = g0[j] * c;
        mf[j] = mf[j] + (g - mf[j]) * w1f;
        vf[j] = vf[j] * b2 + w2f * g * g;
      }
      mm[lane] = mf;
      vv[lane] = vf;
    }
    f32x4 q;
#pragma unroll
    for (int j = 0; j < 4; ++j)  // hardware square root and reciprocal: 1 ulp each, of the step
      q[j] = p0[j] * a.decay -
             a.step * (mf[j] * __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_sqrtf(vf[j]), a.rbc2s, a.eps)));
    aw_store(pp, pt, bi, lane, n, q);
  }
}

// sums of squares in fp64, one per workgroup
__global__ __launch_bounds__(256) void grad_sq_kernel(const AwTab t, double* __restrict__ part) {
  __shared__ double r[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ti = aw_find(t, blockIdx.x);
  const int64_t n = t.n[ti];
  const int nblk = (int)((n + 255) >> 8);
  const int b0 = (blockIdx.x - t.chunk0[ti]) * AW_CHUNK;
  const void* gp = t.g[ti];
  const int gt = t.types[ti] >> 4, b1 = min(nblk, b0 + AW_CHUNK);
  double s = 0.0;
  for (int bi = b0 + wave; bi < b1; bi += 16) {
    f32x4 g[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      g[u] = bi + 4 * u < b1 ? aw_load(gp, gt, bi + 4 * u, lane, n) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) s += (double)g[u][j] * (double)g[u][j];
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  if (lane == 0) r[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (r[0] + r[1]) + (r[2] + r[3]);
}
__global__ __launch_bounds__(1024) void grad_norm_kernel(const double* __restrict__ part, int64_t n, double max_norm,
                                                         double* __restrict__ out) {
  __shared__ double r[1024];
  double s = 0.0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += part[i];
  r[threadIdx.x] = s;
  __syncthreads();
  for (int k = 512; k; k >>= 1) {
    if ((int)threadIdx.x < k) r[threadIdx.x] += r[threadIdx.x + k];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const double norm = sqrt(r[0]), c = max_norm / (norm + 1e-6);
    out[0] = norm;
    out[1] = c < 1.0 ? c : 1.0;
  }
}

// the values that 8-bit states stand for
__global__ __launch_bounds__(256) void state_values_kernel(const unsigned* __restrict__ m, const float* __restrict__ ms,
                                                           const unsigned* __restrict__ v, const float* __restrict__ vs,
                                                           int64_t nquad, f32x4* __restrict__ mo, f32x4* __restrict__ vo) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nquad; i += (int64_t)gridDim.x * 256) {
    const unsigned cm = m[i], cv = v[i];
    const double sm = ms[i >> 6], sv = vs[i >> 6];
    f32x4 a, b;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = (float)(m_value((cm >> (8 * j)) & 255u) * sm);
      b[j] = (float)(v_value((cv >> (8 * j)) & 255u) * sv);
    }
    mo[i] = a;
    vo[i] = b;
  }
}

// ---------------------------------------------------------------------------------------------- host side
// Calls fn(table, workgroups, first workgroup over all launches) for every AW_T tensors that have a gradient and values.
template <typename F>
static int for_tables(int nt, const void* const* p, const void* const* g, const int64_t* n, const uint8_t* pt,
                      const uint8_t* gt, F fn) {
  AwTab t;
  t.count = 0;
  int64_t blocks = 0, chunks = 0, before = 0;
  auto flush = [&]() {
    const int e = t.count ? fn(t, (unsigned)chunks, before) : 0;
    before += chunks;
    chunks = 0;
    t.count = 0;
    return e;
  };
  for (int i = 0; i < nt; ++i) {
    for (int64_t at = 0; at < n[i]; at += AW_MAX) {
      const int64_t k = std::min(n[i] - at, AW_MAX), nb = cdiv(k, 256);
      if (g[i]) {
        t.p[t.count] = p ? (const char*)p[i] + at * dtype_bytes(pt[i]) : nullptr;
        t.g[t.count] = (const char*)g[i] + at * dtype_bytes(gt[i]);
        t.n[t.count] = (unsigned)k;
        t.types[t.count] = (uint8_t)((pt ? pt[i] : 0) | gt[i] << 4);
        t.chunk0[t.count] = (int)chunks;
        t.block0[t.count] = (int)blocks;
        chunks += cdiv(nb, AW_CHUNK);
        if (++t.count == AW_T)
          if (int e = flush()) return e;
      }
      blocks += nb;
    }
  }
  return flush();
}

static const char* tensors_check(int nt, const void* const* g, const int64_t* n, const uint8_t* gt) {
  if (nt < 0 || (nt && (!g || !n || !gt))) return "tensor list";
  int64_t blocks = 0;
  for (int i = 0; i < nt; ++i) {
    if (n[i] < 0 || n[i] >= (int64_t)1 << 38) return "tensor size";
    if (g[i] && gt[i] > IFD_F16) return "gradient type";
    if ((uintptr_t)g[i] % (gt[i] == IFD_F32 ? 4 : 2)) return "a gradient's address is not a multiple of its element";
    blocks += cdiv(n[i], 256);
  }
  if (blocks >= 0x7fffffff) return "more than 2^31 blocks of 256 values";
  return nullptr;
}

}  // namespace ifd

using namespace ifd;
extern "C" {

int64_t ifd_op_grad_norm_ws_bytes(int nt, const int64_t* n) {
  int64_t c = 0;
  for (int i = 0; i < nt && n; ++i) c += n[i] > 0 ? cdiv(cdiv(n[i], 256), AW_CHUNK) : 0;
  return 8 * c;
}

int ifd_op_grad_norm(int nt, const void* const* g, const int64_t* n, const uint8_t* gtype, double max_norm,
                     double* norm_coef, void* ws, int64_t ws_bytes, void* stream) {
  const char* why = tensors_check(nt, g, n, gtype);
  IFD_OP_REQUIRE(!why, why);
  IFD_OP_REQUIRE(norm_coef != nullptr, "null norm_coef");
  IFD_OP_REQUIRE(max_norm >= 0.0, "max_norm must not be negative");
  const int64_t need = ifd_op_grad_norm_ws_bytes(nt, n);
  IFD_OP_REQUIRE(ws_bytes >= need && (ws || !need), "workspace too small");
  IFD_OP_REQUIRE(on(ws, 8) && on(norm_coef, 8), "norm_coef or the workspace: an address off its elements");
  hipStream_t s = (hipStream_t)stream;
  double* part = (double*)ws;
  int64_t total = 0;
  const int rc = for_tables(nt, nullptr, g, n, nullptr, gtype, [&](const AwTab& t, unsigned wgs, int64_t before) {
    hipLaunchKernelGGL(grad_sq_kernel, dim3(wgs), dim3(256), 0, s, t, part + before);
    total = before + wgs;
    return launch_status("ifd_op_grad_norm");
  });
  if (rc) return rc;
  hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(1024), 0, s, part, total, max_norm, norm_coef);
  return IFD_LAUNCH_STATUS();
}

int ifd_op_adamw(const ifd_adamw_args* a, void* stream) {
  IFD_OP_REQUIRE(a != nullptr, "null arguments");
  const char* why = tensors_check(a->nt, a->g, a->n, a->gtype);
  IFD_OP_REQUIRE(!why, why);
  IFD_OP_REQUIRE(a->bits == 8 || a->bits == 32, "states have 8 or 32 bits");
  IFD_OP_REQUIRE(a->step >= 1, "step counts from 1");
  IFD_OP_REQUIRE(a->b1 >= 0.0 && a->b1 < 1.0 && a->b2 >= 0.0 && a->b2 < 1.0 && a->eps > 0.0, "b1, b2 or eps");
  IFD_OP_REQUIRE(a->block0 >= 0, "block0");
  if (!a->nt) return 0;
  IFD_OP_REQUIRE(a->p && a->ptype && a->m && a->v && (a->bits == 32 || (a->m_scale && a->v_scale)), "a null tensor");
  IFD_OP_REQUIRE(!((uintptr_t)a->m & 15) && !((uintptr_t)a->v & 15), "states must be aligned to 16 bytes");
  IFD_OP_REQUIRE(on(a->m_scale, 4) && on(a->v_scale, 4) && on(a->norm_coef, 8), "scales or norm_coef: an address off its elements");
  for (int i = 0; i < a->nt; ++i) {
    IFD_OP_REQUIRE(a->ptype[i] <= IFD_F16, "parameter type");
    IFD_OP_REQUIRE(a->p[i] || !a->g[i] || !a->n[i], "a gradient without its parameter");
    IFD_OP_REQUIRE((uintptr_t)a->p[i] % (a->ptype[i] == IFD_F32 ? 4 : 2) == 0,
                   "a parameter's address is not a multiple of its element");
  }
  AwArgs k = {};
  k.m = a->m; k.v = a->v; k.ms = a->m_scale; k.vs = a->v_scale; k.clip = a->norm_coef; k.block0 = a->block0;
  k.b1 = a->b1; k.w1 = 1.0 - a->b1; k.b2 = a->b2; k.w2 = 1.0 - a->b2;
  k.decay = (float)(1.0 - a->lr * a->wd);
  k.step = (float)(a->lr / (1.0 - std::pow(a->b1, a->step)));
  k.eps = (float)a->eps;
  k.rbc2s = (float)(1.0 / std::sqrt(1.0 - std::pow(a->b2, a->step)));
  k.key = aw_mix(aw_mix(a->seed) + (unsigned)a->step);
  hipStream_t s = (hipStream_t)stream;
  return for_tables(a->nt, a->p, a->g, a->n, a->ptype, a->gtype, [&](const AwTab& t, unsigned wgs, int64_t) {
    if (a->bits == 8)
      hipLaunchKernelGGL(adamw_multi_kernel<8>, dim3(wgs), dim3(256), 0, s, t, k);
    else
      hipLaunchKernelGGL(adamw_multi_kernel<32>, dim3(wgs), dim3(256), 0, s, t, k);
    return launch_status("ifd_op_adamw");
  });
}

int ifd_op_state_values(const void* m, const float* m_scale, const void* v, const float* v_scale, int64_t nblocks,
                        float* m_out, float* v_out, void* stream) {
  IFD_OP_REQUIRE(nblocks >= 0 && nblocks < 0x7fffffff, "nblocks");
  if (!nblocks) return 0;
  IFD_OP_REQUIRE(m && v && m_scale && v_scale && m_out && v_out, "a null tensor");
  IFD_OP_REQUIRE(!(((uintptr_t)m | (uintptr_t)v) & 3) && !(((uintptr_t)m_out | (uintptr_t)v_out) & 15),
                 "states must be aligned to 4 bytes, outputs to 16");
  IFD_OP_REQUIRE(on(m_scale, 4) && on(v_scale, 4), "a scale's address is off its elements");
  hipLaunchKernelGGL(state_values_kernel, dim3((unsigned)std::min<int64_t>(cdiv(nblocks, 4), 16384)), dim3(256), 0,
                     (hipStream_t)stream, (const unsigned*)m, m_scale, (const unsigned*)v, v_scale, nblocks * 64,
                     (f32x4*)m_out, (f32x4*)v_out);
  return IFD_LAUNCH_STATUS();
}

}  // extern "C"
