// Device pieces of the attention kernels (attn_fwd.hip, attn_bwd.hip): MFMA fragments, LDS tiles, masks.
//
// All matrix products are 32x32 MFMA tiles with fp32 accumulators. Lane l = (l32, h): l32 = l & 31, h = l >> 5.
//   operands   a lane holds 16 bytes of one row (A: row l32; B: column l32): CE consecutive channels of chunk
//              2 ks + h of k-step ks (16-bit types: one 32x32x16 MFMA per k-step; fp32: four 32x32x2).
//   results    register i of a lane is row 8 (i / 4) + 4 h + i % 4, column l32.
// A product's result feeds the next product as its B operand without moving between lanes: contraction slot (h, j) of
// step t is taken to be the row that register it already is (16-bit: rows 16 t + 8 (j / 4) + 4 h + j % 4; fp32:
// 8 t + 4 h + j), and the A operand is read from LDS in that row order, transposed (16-bit: ds_read_b64_tr_b16, which
// hands each lane four rows of one column; fp32: four ds_read_b32).
//
// LDS tiles are row-major [rows][DP], filled by LDS-DMA (no registers between), 16-byte chunk c of row r at position
// c ^ swz(r). LDS serves 256 bytes a cycle: 16 rows of one chunk (row reads), four chunks of four consecutive rows
// (transposed reads) and, in fp32, eight chunks of two rows four apart must cover the 64 banks once. Measured: 4.0 cycles
// a row read and 2.3 a transposed read of a wave, twice that where two rows meet in a bank. The 128-byte rows (16-bit,
// DP = 64) take an order that repeats every 8 rows although its row reads meet in pairs (8 cycles): the transposed reads
// then differ by constants alone, which saves the registers that decide how many waves fit (forward, 4096 tokens x 32
// heads, causal: 95 us against 102 with the order that never meets).
#pragma once
#include "ops.h"

namespace ifd {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 hf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 hf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 hf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_c;

template <typename T>
struct AttnT;
template <>
struct AttnT<__bf16> {
  typedef bf16x8 frag;
  typedef bf16x4 quad;
  typedef bf16x2 pair;
  static constexpr int PS = 2;  // contraction steps per 32 rows
  static constexpr int MS = 1;  // MFMAs per operand pair; products of several accumulators take turns (a dependent MFMA waits)
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, int, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct AttnT<_Float16> {
  typedef hf16x8 frag;
  typedef hf16x4 quad;
  typedef hf16x2 pair;
  static constexpr int PS = 2, MS = 1;
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, int, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct AttnT<float> {
  typedef f32x4 frag;
  typedef f32x4 quad;
  typedef f32x2 pair;
  static constexpr int PS = 4, MS = 4;
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, int j, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  }
};

// Bytes of a head's row in LDS: the head width that the products cover (dp: 64, 96 or 128), rounded to a power of two
constexpr int attn_row_bytes(int dp, int es) { return (dp == 96 ? 128 : dp) * es; }

template <typename T, int DP>
struct AttnTile {
  typedef AttnT<T> A;
  typedef typename A::frag frag;
  static constexpr int ES = sizeof(T), CE = 16 / ES, ROWB = attn_row_bytes(DP, ES), NCH = ROWB / 16;
  static constexpr int KS = DP / CE / 2, DT = DP / 32, PS = A::PS;

  static __device__ __forceinline__ int swz(int r) {
    if (ES == 4) return ((r & 7) << 1) | ((r >> 3) & 1);
    return NCH == 8 ? ((r & 3) << 1) | ((r >> 2) & 1) : ((r & 3) << 2) | ((r >> 2) & 3);
  }

  // rows [r0, r0 + 32) as A operands of k-step ks (row l32, chunk 2 ks + h)
  static __device__ __forceinline__ frag row(const lds_c* tile, int r0, int ks, int l32, int h) {
    return *(const __attribute__((address_space(3))) frag*)(tile + r0 * ROWB + l32 * ROWB +
                                                            (((2 * ks) ^ (h ^ swz(l32))) << 4));
  }
  // rows [r0, r0 + 32) transposed as the A operand of contraction step t: column 32 dt + l32
  static __device__ __forceinline__ frag col(const lds_c* tile, int r0, int t, int dt, int lane) {
    const int h = lane >> 5, l32 = lane & 31;
    if constexpr (ES == 2) {
      const int i = lane & 15;
      const int c = dt * 4 + (((lane >> 4) & 1) << 1) + ((i & 3) >> 1);
      s16x8 f;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = 16 * t + 8 * u + 4 * h + (i >> 2);
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(tile + r0 * ROWB + r * ROWB + ((c ^ swz(r)) << 4) +
                                                       ((i & 1) << 3)));
#pragma unroll
        for (int j = 0; j < 4; ++j) f[4 * u + j] = x[j];
      }
      return __builtin_bit_cast(frag, f);
    } else {
      frag f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 8 * t + 4 * h + j;
        f[j] = *(const __attribute__((address_space(3))) float*)(tile + r0 * ROWB + r * ROWB +
                                                                 (((dt * 8 + (l32 >> 2)) ^ swz(r)) << 4) +
                                                                 ((l32 & 3) << 2));
      }
      return f;
    }
  }
  // a result tile's registers of contraction step t as an operand. In the 16-bit types P and dS are rounded to T here, to
  // nearest, once: the matrix units take no wider operand at their rate (fp32 products run at an eighth of it). The results'
  // error grows from 1.7e-3 of their norm, their own rounding, to 2.3e-3 (bf16; fp16 2.1e-4 to 3.0e-4). fp16 holds dS down to
  // 2^-24: gradients much smaller than 1 need a loss scale, as any fp16 gradient does.
  static __device__ __forceinline__ frag pack(const f32x16& s, int t) {
    frag f;
    if constexpr (ES == 2) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const f32x2 v = {s[8 * t + j], s[8 * t + j + 1]};
        const typename A::pair p = __builtin_convertvector(v, typename A::pair);
        f[j] = p[0];
        f[j + 1] = p[1];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = s[4 * t + j];
    }
    return f;
  }
  // 16 bytes of a row in global memory as an operand: zeros past D or for an absent row
  static __device__ __forceinline__ frag gload(const char* rowp, bool ok, int ks, int h, int D) {
    const int c = 2 * ks + h;
    u32x4 z = {0, 0, 0, 0};
    if (ok && c * CE < D) z = *reinterpret_cast<const u32x4*>(rowp + c * 16);
    return __builtin_bit_cast(frag, z);
  }
};

// LDS-DMA of 16 bytes per lane, from `off` bytes past base to dst + 16 lane. (The host pass of a template that calls the
// builtin in its body drops the kernel's stub without a message: it stays inside these two functions.)
__device__ __forceinline__ void dma_quad(const char* base, int off, lds_c* dst) {
  const __amdgpu_buffer_rsrc_t rs =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), (short)0, 0x7ffffff0, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16, off, 0, 0, 0);
}
// LDS-DMA of one 4-byte word per lane, from `off` bytes past base to dst + 4 lane
__device__ __forceinline__ void dma_word(const float* base, int off, lds_c* dst) {
  const __amdgpu_buffer_rsrc_t rs =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), (short)0, 0x7ffffff0, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 4, off, 0, 0, 0);
}

// LDS-DMA of ROWS rows of a [token][D] matrix into a tile by NW waves (wave w of them). Rows past `nrows` repeat the
// last one and chunks past D repeat chunk 0: what they hold is real data of the same matrix, and the products either
// multiply it by zeros or drop its result.
template <typename T, int DP, int ROWS, int NW>
struct AttnStage {
  typedef AttnTile<T, DP> TL;
  static constexpr int RPI = 1024 / TL::ROWB;            // rows per DMA instruction (64 lanes x 16 bytes)
  static constexpr int NI = ROWS / RPI / NW;             // instructions per wave
  static_assert(ROWS % (RPI * NW) == 0, "tile rows divide over the waves");
  static constexpr int ROWS_STEP = RPI * NW, NCB = ROWS_STEP >= 16 ? 1 : 16 / ROWS_STEP;  // swz repeats every 16 rows
  int row, cb[NCB];  // of instruction 0; of instruction i: row + i ROWS_STEP, cb[i % NCB]

  __device__ __forceinline__ void init(int w, int lane, int D) {
    row = w * RPI + lane / TL::NCH;
#pragma unroll
    for (int i = 0; i < NCB; ++i) {
      const int c = (lane % TL::NCH) ^ TL::swz(row + i * ROWS_STEP);
      cb[i] = c * TL::CE < D ? c * 16 : 0;
    }
  }
  // base: the tile's first row; stride in bytes (host check: 128 rows stay within 31 bits)
  __device__ __forceinline__ void load(const char* base, int stride, int nrows, lds_c* tile, int w) const {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = min(row + i * ROWS_STEP, nrows - 1);
      dma_quad(base, r * stride + cb[i % NCB], tile + (w + NW * i) * 1024);
    }
  }
};

__device__ __forceinline__ void lds_zero(lds_c* q) { *(__attribute__((address_space(3))) u32x4*)q = u32x4{0, 0, 0, 0}; }
__device__ __forceinline__ f32x4 lds_quad(const lds_c* q) { return *(const __attribute__((address_space(3))) f32x4*)q; }

__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// max / sum with the other half of a wave (lane ^ 32)
__device__ __forceinline__ float xhalf(float v) { return __shfl_xor(v, 32); }

struct AttnK {  // kernel arguments: strides in bytes
  const char *q, *k, *v, *dout;
  char *out, *dq, *dk, *dv;
  float* lse;
  const int *kv_len, *q_start;
  int64_t qb, qh, kb, kh, vb, vh, ob, oh, gb, gh, dqb, dqh, dkb, dkh, dvb, dvh;
  int qt, kt, vt, ot, gt, dqt, dkt, dvt;  // token strides
  int B, Tq, Tk, Hq, Hk, D, G, causal, nblk, nsplit, nsplit_q;
  float c, scale;  // c = scale log2(e)
  float *ws, *ws_kv, *ws_q;  // backward: lse2 and delta, the key pass' shares, the row pass' shares
};

__device__ __forceinline__ int seq_len(const AttnK& p, int b) {
  if (!p.kv_len) return p.Tk;
  const int n = p.kv_len[b];
  return n < 0 ? 0 : (n > p.Tk ? p.Tk : n);
}
// keys that row i of sequence b sees: [0, limit); what the last of some rows sees bounds what is loaded for them
__device__ __forceinline__ int row_limit(const AttnK& p, int qs, int len, int i) {
  if (!p.causal) return len;
  const int64_t n = (int64_t)qs + i + 1;  // q_start is any int32
  return n < 0 ? 0 : (n > len ? len : (int)n);
}
__device__ __forceinline__ int q_first(const AttnK& p, int b) { return p.q_start ? p.q_start[b] : p.Tk - p.Tq; }

// Workgroups are dealt to the eight XCDs in turn: give each XCD a contiguous range, so that blocks that read the same
// keys share an L2.
__device__ __forceinline__ int xcd_order(int bid, int n) {
  const int full = n & ~7;
  return bid < full ? (bid & 7) * (full >> 3) + (bid >> 3) : bid;
}

// attn_fwd.hip: what is wrong with a tensor's pointer or strides (nullptr: nothing), and the kernels' form of the arguments
const char* attention_tensor_check(const ifd_attention_args& a, const void* p, const int64_t (&s)[3]);
AttnK attention_kernel_args(const ifd_attention_args& a);

}  // namespace ifd
