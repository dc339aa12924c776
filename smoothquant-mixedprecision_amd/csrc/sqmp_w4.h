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

// one dword of codes and its scale -> 8 values D(code * s)
template <class DT>
__device__ inline Frag<DT> decode(uint32_t w, typename DT::T s, const DecK& k) {
  Frag<DT> f;
  const uint16_t b = __builtin_bit_cast(uint16_t, s);
  f.v[0] = Dec<DT>::run(w, Dec<DT>::prep((uint32_t)b), k);
  return f;
}
// fp32: (n - 8) s = fma(n, s, -8 s): 8 s is exact, so the one rounding is that of code * s
template <>
__device__ inline Frag<F32> decode<F32>(uint32_t w, float s, const DecK&) {
  const float m8 = -8.f * s;
  const uint32_t b = w & 0x0F0F0F0Fu, c = (w >> 4) & 0x0F0F0F0Fu;
  float o[8];
  o[0] = (float)(b & 0xFFu), o[2] = (float)(c & 0xFFu);
  o[4] = (float)((b >> 8) & 0xFFu), o[6] = (float)((c >> 8) & 0xFFu);
  o[1] = (float)((b >> 16) & 0xFFu), o[3] = (float)((c >> 16) & 0xFFu);
  o[5] = (float)(b >> 24), o[7] = (float)(c >> 24);
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
    const float s = __uint_as_float(prep), m8 = -8.0f * s;
    uint32_t b = (h ? w >> 4 : w) & 0x0F0F0F0Fu;
    asm volatile("" : "+v"(b));  // (keeps the byte form: v_cvt_f32_ubyte0..3)
    const f2 lo = {__builtin_fmaf((float)(b & 0xFFu), s, m8), __builtin_fmaf((float)((b >> 16) & 0xFFu), s, m8)};
    const f2 hi = {__builtin_fmaf((float)((b >> 8) & 0xFFu), s, m8), __builtin_fmaf((float)(b >> 24), s, m8)};
    f[h] = __builtin_bit_cast(uint32_t, __builtin_convertvector(lo, bf2));
    f[h + 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, bf2));
  }
};

}  // namespace w4
}  // namespace sqmp
