// Device pieces shared by the kernels on the tile-major 4-bit operands (sqmp_pack_fq7 with
// J = 2): the few-row products (sqmp_gemv.hip) and the expert products (sqmp_experts.hip).
//
// Operand geometry.  A weight block is 32 rows; per 64-position stage lane (r16 = lane & 15,
// q = lane >> 4) holds 16 bytes: dwords [j][s] of row 16 j + r16, each the 8 codes of positions
// 8 c .. 8 c + 7 with c = 4 (q & 1) + 2 s + (q >> 1).  As the A operand of a 16 x 16 x 32 MFMA
// (j selects the 16 rows, s the 32-position half of the stage) they meet the 8 activations of
// the same positions in the B operand, whose lane r16 is a token: C register r of lane (r16, q)
// is y[token r16][row 16 j + 4 q + r].
#pragma once
#include "sqmp_mfma.h"

namespace sqmp {
namespace w4 {

// Buffer loads from a wave-uniform base: the lane's offset stays in one register, the stage's is a
// scalar (64-bit addresses would cost two registers and two additions per load)
__device__ inline __amdgpu_buffer_rsrc_t rsrc_of(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, -1, 0x00020000);
}
__device__ inline u32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)voff, (int)soff, 0));
}
__device__ inline uint64_t load8(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_bit_cast(uint64_t, __builtin_amdgcn_raw_buffer_load_b64(r, (int)voff, (int)soff, 0));
}
__device__ inline uint32_t load2(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  return (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, (int)voff, (int)soff, 0);
}
__device__ inline uint32_t load4(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)voff, (int)soff, 0);
}

// activations of the gated experts' epilogue (fp32 in, fp32 out)
enum Act { ACT_NONE = 0, ACT_SILU = 1, ACT_GELU = 2 };

template <int ACT>
__device__ inline float act_fn(float g) {
  if constexpr (ACT == ACT_SILU) return g / (1.f + expf(-g));
  if constexpr (ACT == ACT_GELU) return 0.5f * g * (1.f + erff(g * 0.70710678118654752f));
  return g;
}

// 8 values of D in registers: 16 bytes, or 32 for fp32
template <class DT> struct Frag {
  u32x4 v[1];
};
template <> struct Frag<F32> {
  u32x4 v[2];
};

template <class DT>
__device__ inline Frag<DT> load_frag(const typename DT::T* p) {
  Frag<DT> f;
  constexpr int n = sizeof(f.v) / 16;
#pragma unroll
  for (int i = 0; i < n; ++i) f.v[i] = ((const u32x4*)p)[i];
  return f;
}

template <class DT>
__device__ inline void mfma(f32x4& acc, const Frag<DT>& a, const Frag<DT>& b) {
  constexpr int n = sizeof(a.v) / 16;
#pragma unroll
  for (int i = 0; i < n; ++i) Mfma<DT>::run(acc, a.v[i], b.v[i]);
}

// 4 bytes 0 .. 15 -> floats: as e4m3 such a byte is n 2^-9 (0 .. 7 the subnormals, 8 .. 15 the first
// binade, one step of 2^-9), so one conversion with a scale of 2^9 makes two of them.  (The 2^9 in the
// weight's scale instead overflows from 2^119 on)
__device__ inline void nibbles_to_f32(uint32_t b, float (&n)[4]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(b, 512.0f, false);
  const f2 hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(b, 512.0f, true);
  n[0] = lo[0], n[1] = lo[1], n[2] = hi[0], n[3] = hi[1];
}

// one dword of codes and its scale -> 8 values D(code * s).  (bf16 by Dec::run: by scaled conversions
// the few-row kernel runs 10.1 us instead of 8.8 at 8 x 11008 x 4096; the tiles use them, DecHalf)
template <class DT>
__device__ inline Frag<DT> decode(uint32_t w, typename DT::T s, const DecK& k) {
  Frag<DT> f;
  const uint16_t b = __builtin_bit_cast(uint16_t, s);
  f.v[0] = Dec<DT>::run(w, Dec<DT>::prep((uint32_t)b), k);
  return f;
}
// (n - 8) s = fma(n, s, -8 s): 8 s is exact, so fp32 rounds once, and bf16 s (8 + 4 significant bits)
// not before the cast (scales below 2^125: 8 s is finite)
template <>
__device__ inline Frag<F32> decode<F32>(uint32_t w, float s, const DecK&) {
  const float m8 = -8.f * s;
  float b[4], c[4];  // nibbles 0, 2, 4, 6 and 1, 3, 5, 7
  nibbles_to_f32(w & 0x0F0F0F0Fu, b);
  nibbles_to_f32((w >> 4) & 0x0F0F0F0Fu, c);
  // element 2 i is nibble i, element 2 i + 1 nibble 4 + i
  const float o[8] = {b[0], b[2], c[0], c[2], b[1], b[3], c[1], c[3]};
  Frag<F32> f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f.v[e >> 2][e & 3] = __float_as_uint(__builtin_fmaf(o[e], s, m8));
  return f;
}
// Half of decode: the values at dwords h and h + 2 of the fragment (elements 2h, 2h + 1, 2h + 4,
// 2h + 5), for kernels that spread the decoding between their MFMAs; prep: the prepared scale
template <class DT> struct DecHalf;
template <> struct DecHalf<F16> {
  __device__ static inline void run(u32x4& f, uint32_t w, uint32_t prep, const DecK& k, int h) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 s2 = __builtin_bit_cast(h2, prep);
    const _Float16 off = h ? (_Float16)72.0f : (_Float16)1032.0f;
    const uint32_t m = h ? k.m1 : k.m0, c = h ? k.c1 : k.c0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      h2 v = __builtin_bit_cast(h2, and_or(i ? w >> 8 : w, m, c));
      v = (v - h2{off, off}) * s2;
      f[h + 2 * i] = __builtin_bit_cast(uint32_t, v);
    }
  }
};
template <> struct DecHalf<BF16> {
  __device__ static inline void run(u32x4& f, uint32_t w, uint32_t prep, const DecK&, int h) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    const float s = __uint_as_float(prep), m8 = -8.f * s;
    float n[4];
    nibbles_to_f32((h ? w >> 4 : w) & 0x0F0F0F0Fu, n);
    const f2 lo = {__builtin_fmaf(n[0], s, m8), __builtin_fmaf(n[2], s, m8)};
    const f2 hi = {__builtin_fmaf(n[1], s, m8), __builtin_fmaf(n[3], s, m8)};
    f[h] = __builtin_bit_cast(uint32_t, __builtin_convertvector(lo, bf2));
    f[h + 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, bf2));
  }
};

}  // namespace w4
}  // namespace sqmp
