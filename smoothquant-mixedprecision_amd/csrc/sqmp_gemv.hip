// Few-row products with 4-bit weights: y[m][n] = D( sum_p x[m][p] W[n][p] + bias[n] ),
// 1 <= m <= 64 rows (the decoding form of fake_quant.py:306's F.linear), and the same per expert
// of a mixture (ragged rows).  W = D(code * scale) at the Kp coded positions, then the S_pad
// exact salient columns.
//
// What bounds it: the weight bytes (N Kp / 2 codes + scales), read once; for single weights of a few
// MB the latency of one trip to HBM.  So a wave streams whole 1-KiB stages of the tile-major codes
// straight into registers, decodes them there and feeds the MFMA with the tokens in the B slot: the
// matrix work of 16 tokens is that of one.  A workgroup owns one block of 32 weight rows (or, where
// blocks are few, its halves go to two workgroups on one XCD, which share the lines) and its NW
// waves take the K stages round robin (consecutive stages are consecutive memory), U stages of loads
// in flight each; the NW partial sums meet in LDS and are added in a fixed order, so results do not
// depend on timing.  x comes as 16-byte fragments from L2, or, where its rows are unaligned or the
// weight has an order of its own, gathered into LDS while the first codes are on their way.
// Measured (kernel alone): 1 x 4096 x 4096 fp16 4.5 us (8.7 MB: 1.9 TB/s, 1.7 us at the rate of a
// large copy; latency), 8 x 11008 x 4096 bf16 9.3 us (2.6 TB/s; decoding, and 344 blocks on 256
// CUs), 1 x 32000 x 4096 15.1 us (4.5 TB/s), 64 x 4096 x 11008 15.9 us (1.6 TB/s; two groups of tokens
// decode everything twice), 8 tokens to 2 of 8 experts, 22016 x 4096: 67.8 us (335 MB: 4.9 TB/s).
#include "sqmp_w4_launch.h"

namespace sqmp {
namespace w4 {

// GB: 1 = groups of whole 64-position stages, 2 = groups of 32, 0 = any multiple of 8
// MT: 16-row token tiles per pass; J: 16-row halves of the block per workgroup (1: two workgroups,
// neighbours on one XCD, share the block's lines); NW waves; U stages in flight; STAGE: the rows of
// x gathered into LDS first; NX > 0 (16-bit types): a stage's rows come as 8 NX whole 128-byte
// lines and are turned into fragments in a wave's own corner of LDS (fragments straight from L2
// touch every line four times); ACT / EXP: the expert forms
template <class DT, int GB, int MT, int J, int NW, int U, bool STAGE, int NX, bool EXP, int ACT>
__global__ __launch_bounds__(NW * 64) void gemv_kernel(const GemvArgs a) {
  typedef typename DT::T T;
  constexpr int SZ = sizeof(T);
  constexpr int RS = 16 * J + 4;  // floats per token row of a partial (+ 4: spreads the LDS banks)
  static_assert(ACT == ACT_NONE || J == 2, "gate and up rows meet in one workgroup");
  __shared__ __attribute__((aligned(16))) float red[NW * MT * 16 * RS];
  static_assert(NX == 0 || (MT == (NX + 1) / 2 && SZ == 2 && !STAGE), "whole lines: 16-bit rows");
  constexpr int PASS = NX == 1 ? 8 : 16 * MT;  // tokens per pass over the weights
  constexpr int XP = 144;         // bytes of a row of the corner (128 + 16: spreads the banks)
  constexpr int CORNER = 8 * NX * XP, NC = NX <= 2 ? 2 : 1;  // two corners a wave where they are small
  __shared__ __attribute__((aligned(16))) unsigned char turn[NX > 0 ? NW * NC * CORNER : 16];
  extern __shared__ __attribute__((aligned(16))) unsigned char xs[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int r16 = lane & 15, q = lane >> 4;
  int nb = blockIdx.x, half = 0;
  if constexpr (J == 1) {
    nb = ((int)blockIdx.x >> 4) * 8 + (blockIdx.x & 7), half = (blockIdx.x >> 3) & 1;
    if (nb * 32 + half * 16 >= a.N) return;
  }
  const int nblk = (a.N + 255) / 256 * 8;  // 32-row blocks of one weight's operands
  const int nkp = a.Kp / 64, nkm = a.nk, nks = a.S_pad / 64;
  // one weight: every pass of tokens has workgroups of its own (blockIdx.y)
  int lo = (int)blockIdx.y * PASS, hi = min(a.M, lo + PASS);
  long wb = nb;
  if constexpr (EXP) {
    lo = a.offsets[blockIdx.y];
    hi = a.offsets[blockIdx.y + 1];
    wb += (long)blockIdx.y * nblk;
  }
  const __amdgpu_buffer_rsrc_t rW = rsrc_of(a.codes + wb * nkp * 256);
  const __amdgpu_buffer_rsrc_t rS = rsrc_of((const T*)a.scale + wb * a.ngw * 32);
  const T* sal = (const T*)a.sal + wb * nks * 2048 + lane * 32 + half * 16;
  const uint32_t vw = (uint32_t)lane * 16 + half * 8, vs = (uint32_t)(r16 * 2 + half) * SZ;
  const DecK dk = make_deck();
  const int c0 = 4 * (q & 1) + (q >> 1);  // chunk of s = 0; s = 1: + 2

  struct Codes {
    uint32_t w[2 * J];               // [j][s]
    T s[GB == 0 ? 2 * J : J];        // scales of the row halves (GB 0: for either s)
  };
  auto scale_at = [&](uint32_t voff, uint32_t soff, T* d) {
    if constexpr (SZ == 2 && J == 2) {
      const uint32_t v = load4(rS, voff, soff);
      d[0] = __builtin_bit_cast(T, (uint16_t)v), d[1] = __builtin_bit_cast(T, (uint16_t)(v >> 16));
    } else if constexpr (SZ == 2) {
      d[0] = __builtin_bit_cast(T, (uint16_t)load2(rS, voff, soff));
    } else if constexpr (J == 2) {
      const uint64_t v = load8(rS, voff, soff);
      d[0] = __uint_as_float((uint32_t)v), d[1] = __uint_as_float((uint32_t)(v >> 32));
    } else {
      d[0] = __uint_as_float(load4(rS, voff, soff));
    }
  };
  auto load_w = [&](int kt, Codes& c) {
    if constexpr (J == 2) {
      const u32x4 v = load16(rW, vw, (uint32_t)kt * 1024);
#pragma unroll
      for (int i = 0; i < 4; ++i) c.w[i] = v[i];
    } else {
      const uint64_t v = load8(rW, vw, (uint32_t)kt * 1024);
      c.w[0] = (uint32_t)v, c.w[1] = (uint32_t)(v >> 32);
    }
    if constexpr (GB == 0) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int g = min((kt * 64 + 8 * (c0 + 2 * s)) / a.Gw, a.ngw - 1);
        scale_at(vs + (uint32_t)g * 32 * SZ, 0, c.s + J * s);
      }
    } else if constexpr (GB == 1) {
      scale_at(vs, (uint32_t)group_of(kt, a) * 32 * SZ, c.s);
    } else {
      scale_at(vs + (uint32_t)min(2 * kt + (q & 1), a.ngw - 1) * 32 * SZ, 0, c.s);
    }
  };

  for (int m0 = lo; m0 < hi; m0 += PASS) {
    // this lane's tokens (rows past the end repeat the last one; their columns of C are dropped)
    const T* xp[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = min(m0 + 16 * i + r16, hi - 1);
      long xr = m;
      if constexpr (EXP) {
        if (a.rows) xr = a.rows[m] / a.top_k;
      }
      xp[i] = STAGE ? (const T*)xs + (long)(m - lo) * ((a.Kp + a.S_pad) + 16 / SZ) + 8 * c0
                    : (const T*)a.x + xr * a.ldx + 8 * c0;
    }
    f32x4 acc[MT][J];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Stage {
      Codes c;
      Frag<DT> x[MT][2];
      u32x4 line[NX > 0 ? NX : 1];
    };
    // this lane's pieces of the lines: row 8 i + lane / 8 (loads of rows past the end left out by
    // predicates cost more than they save: 4.8 us instead of 4.4 at 1 x 4096 x 4096)
    const T* lp[NX > 0 ? NX : 1];
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      const int m = min(m0 + 8 * i + (lane >> 3), hi - 1);
      long xr = m;
      if constexpr (EXP) {
        if (a.rows) xr = a.rows[m] / a.top_k;
      }
      lp[i] = (const T*)a.x + xr * a.ldx + 8 * (lane & 7);
    }
    auto load_x = [&](int kt, Stage& st) {
      if constexpr (NX > 0) {
#pragma unroll
        for (int i = 0; i < NX; ++i) st.line[i] = *(const u32x4*)(lp[i] + (long)kt * 64);
      } else {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int s = 0; s < 2; ++s) st.x[i][s] = load_frag<DT>(xp[i] + (long)kt * 64 + 16 * s);
      }
    };
    auto compute = [&](Stage& st, int u) {
      if constexpr (NX > 0) {
        // (the LDS operations of one wave run in order: the reads see the writes, and the next
        // writes to this half come after these reads)
        unsigned char* t = turn + (wave * NC + (u % NC)) * CORNER;
#pragma unroll
        for (int i = 0; i < NX; ++i)
          *(u32x4*)(t + (8 * i + (lane >> 3)) * XP + (lane & 7) * 16) = st.line[i];
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int r = NX == 1 ? r16 & 7 : 16 * i + r16;
#pragma unroll
          for (int s = 0; s < 2; ++s)
            st.x[i][s] = load_frag<DT>((const T*)(t + r * XP + (c0 + 2 * s) * 16));
        }
        asm volatile("" ::: "memory");
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const Frag<DT> w = decode<DT>(st.c.w[2 * j + s], st.c.s[GB == 0 ? J * s + j : j], dk);
#pragma unroll
          for (int i = 0; i < MT; ++i) mfma<DT>(acc[i][j], w, st.x[i][s]);
        }
    };
    int kt = wave;
    Stage st[U];
    if constexpr (STAGE) {
      // the first codes are on their way while the rows are gathered
#pragma unroll
      for (int u = 0; u < U; ++u) load_w(min(kt + u * NW, nkm - 1), st[u].c);
      const int L = a.Kp + a.S_pad, LP = L + 16 / SZ, M = hi - lo;
      const T* x = (const T*)a.x;
      for (int p = threadIdx.x; p < L; p += NW * 64) {
        int k = -1;
        if (p < a.Kp) k = a.amap[p];
        else if (p - a.Kp < a.S) k = a.salient[p - a.Kp];
        T v[16];
#pragma unroll
        for (int m = 0; m < 16; ++m)
          if (m < M) v[m] = k >= 0 ? x[(long)(lo + m) * a.ldx + k] : (T)0.f;
#pragma unroll
        for (int m = 0; m < 16; ++m)
          if (m < M) ((T*)xs)[(long)m * LP + p] = v[m];
      }
      __syncthreads();
    }
    bool first = STAGE;
    for (; kt + (U - 1) * NW < nkm; kt += U * NW) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!first) load_w(kt + u * NW, st[u].c);
        load_x(kt + u * NW, st[u]);
      }
      first = false;
#pragma unroll
      for (int u = 0; u < U; ++u) compute(st[u], u);
    }
    for (; kt < nkm; kt += NW) {
      load_w(kt, st[0].c);
      load_x(kt, st[0]);
      compute(st[0], 0);
    }
    // the exact salient columns: operand fragments as they are
    for (int kd = wave; kd < nks; kd += NW) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        Frag<DT> x[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) x[i] = load_frag<DT>(xp[i] + (long)(nkp + kd) * 64 + 16 * s);
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const Frag<DT> w = load_frag<DT>(sal + (long)kd * 2048 + j * 16 + s * 8);
#pragma unroll
          for (int i = 0; i < MT; ++i) mfma<DT>(acc[i][j], w, x[i]);
        }
      }
    }
    // partial sums to LDS: red[wave][token][row of the block]
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j)
        *(f32x4*)(red + ((wave * MT + i) * 16 + r16) * RS + 16 * j + 4 * q) = acc[i][j];
    __syncthreads();
    const int nm = min(PASS, hi - m0);
    constexpr int NO = ACT == ACT_NONE ? 16 * J : 16;  // outputs per token of this workgroup
    for (int t = threadIdx.x; t < nm * NO; t += NW * 64) {
      const int m = t / NO, r = t % NO;
      const int n = (ACT == ACT_NONE ? nb * 32 + half * 16 : nb * 16) + r;
      float v = 0.f, u = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        v += red[(w * MT * 16 + m) * RS + r];
        if constexpr (ACT != ACT_NONE) u += red[(w * MT * 16 + m) * RS + r + 16];
      }
      if (n >= a.n_out) continue;
      if constexpr (ACT != ACT_NONE) v = act_fn<ACT>(v) * u;
      if (a.bias) v += DT::to_f(((const T*)a.bias)[n]);
      ((T*)a.y)[(long)(m0 + m) * a.n_out + n] = DT::from_f(v);
    }
    __syncthreads();  // the next pass writes red again
  }
}

// LDS a call may use for gathered rows (with the partial sums, up to 36 KiB at 16 waves and 32 rows,
// below 64 KiB)
constexpr long STAGE_BYTES = 27 * 1024;
static long stage_bytes(int dtype, int M, int Kp, int S_pad) {
  return (long)(M < 16 ? M : 16) * ((Kp + S_pad) * (dtype == SQMP_F32 ? 4L : 2L) + 16);
}

template <class DT, int GB, bool EXP, int ACT>
static int launch(const GemvArgs& a, int E, int max_rows, hipStream_t s) {
  const int nb = cdiv(a.N, 32);
  const size_t xb = a.amap ? (size_t)stage_bytes(DT::id, a.M, a.Kp, a.S_pad) : 0;
  const int groups = a.M <= 16 ? 1 : cdiv(a.M, 16);  // of 16 tokens (one weight)
#define SQMP_GV(MT, J, NW, U, ST, NX)                                                                  \
  gemv_kernel<DT, GB, MT, J, NW, U, ST, NX, EXP, ACT>                                                  \
      <<<dim3((J) == 1 ? cdiv(nb, 8) * 16 : nb, EXP ? E : groups), dim3((NW) * 64), xb, s>>>(a)
  // Waves per workgroup, and whether a block's halves go to two workgroups, by how many blocks
  // there are for the 256 CUs.  8 waves / 16 waves / 8 waves and halves / 16 and halves, one row, one
  // card: 32 blocks of K 4096 4.9 / 4.7 / 4.1 / 4.1 us, 128 of K 4096 5.2 / 4.9 / 4.4 / 4.4, of K 11008
  // 10.1 / 9.4 / 7.9 / 8.4, 256 of K 2048 (fp32) 8.5 / 8.1 / 8.6 / 10.1, 344 of K 4096 8.1 / 9.2 / 8.8
  // / 10.6, 1000 of K 4096 19.7 / 21.6 / 20.8 / 28.8
  constexpr int N1 = DT::id == SQMP_F32 ? 0 : 1, N2 = DT::id == SQMP_F32 ? 0 : 2;
  if constexpr (EXP) {
    // 8 / 4 waves by the blocks of all experts, 2 rows each: K 4096 (fp16) 256 blocks 6.7 / 7.7 us, 512 10.3 /
    // 10.5, 1024 18.8 / 17.0, 1536 26.3 / 24.0, 2048 34.0 / 31.1, 5504 81 / 77; K 2048 (bf16) 1024 13.5 / 11.7,
    // 2048 23.5 / 20.1, 5632 58 / 50
    if (max_rows <= 16) {
      if ((long)nb * E >= 1024) {
        if (max_rows <= 8) SQMP_GV(1, 2, 4, 4, false, N1); else SQMP_GV(1, 2, 4, 4, false, N2);
      } else {
        if (max_rows <= 8) SQMP_GV(1, 2, 8, 4, false, N1); else SQMP_GV(1, 2, 8, 4, false, N2);
      }
    } else {
      SQMP_GV(2, 2, 8, 2, false, (DT::id == SQMP_F32 ? 0 : 4));
    }
  } else {
#define SQMP_GVX(J, NW)                                                                            \
  if (a.amap) SQMP_GV(1, J, NW, 4, true, 0);                                                       \
  else if (a.M <= 8) SQMP_GV(1, J, NW, 4, false, N1);                                              \
  else SQMP_GV(1, J, NW, 4, false, N2)
    if constexpr (DT::id != SQMP_F32) {
      // 17 .. 64 rows where groups of 16 are more than the CUs: groups of 32, a decoded fragment feeds
      // two MFMAs (16 / 32 a group, fp16: 64 rows x 4096 x 4096 9.8 / 7.7 us, x 11008 x 4096 25.9 / 17.0; 32
      // x 32000 x 4096 39.6 / 26.3; but 32 x 4096 x 4096 5.8 / 7.4, 64 x 1024 x 4096 5.4 / 7.1)
      if (a.M > 16 && !a.amap && nb * groups > 256) {
        const int groups = cdiv(a.M, 32);
        SQMP_GV(2, 2, 8, 2, false, 4);
        SQMP_LAUNCH_CHECK();
        return SQMP_OK;
      }
    }
    const int blocks = nb * groups;
    if (blocks <= 192) { SQMP_GVX(1, 8); }
    else if (blocks <= 320) { SQMP_GVX(2, 16); }
    else { SQMP_GVX(2, 8); }
#undef SQMP_GVX
  }
#undef SQMP_GV
  SQMP_LAUNCH_CHECK();
  return SQMP_OK;
}

template <class DT, bool EXP, int ACT>
static int by_group(const GemvArgs& a, int E, int max_rows, hipStream_t s) {
  if (a.Gw % 64 == 0) return launch<DT, 1, EXP, ACT>(a, E, max_rows, s);
  if (a.Gw == 32) return launch<DT, 2, EXP, ACT>(a, E, max_rows, s);
  if (a.Gw % 8 == 0) return launch<DT, 0, EXP, ACT>(a, E, max_rows, s);
  return SQMP_EUNSUPPORTED;
}

// Whether a single weight goes to the expert tiles: more than 32 rows of a wide one (64 rows, few-row
// kernel / tiles: N 11008 17.0 / 24.6 us, 32000 43.9 / 38.5; 32 rows of 32000 26.3 / 34.6)
static bool gemv_takes_tiles(int dtype, int M, int N) {
  return dtype != SQMP_F32 && M > 32 && cdiv(N, 32) > 700;
}

static int check_operand(const void* x, long ldx, int cols, int dtype, int N, int Kp, int S_pad,
                         int Gw, int ngw, bool gathered = false) {
  if (N <= 0 || Kp <= 0 || Kp % 128 || S_pad < 0 || S_pad % 64 || Gw <= 0 || ngw <= 0)
    return SQMP_EINVAL;
  if (dtype != SQMP_F32 && dtype != SQMP_F16 && dtype != SQMP_BF16) return SQMP_EUNSUPPORTED;
  if (gathered) return ldx > 0 && cols == Kp ? SQMP_OK : SQMP_EINVAL;
  if (cols != Kp && (cols <= 0 || cols > Kp || cols % 64 || S_pad > 0)) return SQMP_EINVAL;
  const long per16 = dtype == SQMP_F32 ? 4 : 8;  // whole 16-byte loads of x
  if (ldx < (long)cols + S_pad || ldx % per16 || (size_t)x % 16) return SQMP_EINVAL;
  return SQMP_OK;
}

}  // namespace w4

// (0 where the few-row kernel runs, which splits K inside a workgroup)
extern "C" size_t sqmp_gemv_workspace_bytes(int dtype, int M, int N, int Kp) {
  if (N <= 0 || Kp <= 0 || !w4::gemv_takes_tiles(dtype, M, N)) return 0;
  return w4::expert_tiles_workspace(1, M, N, Kp);
}

extern "C" size_t sqmp_expert_workspace_bytes(int dtype, int E, int slots, int N, int Kp) {
  if (E <= 0 || slots < 12L * E || N <= 0 || Kp <= 0 || dtype == SQMP_F32) return 0;
  return w4::expert_tiles_workspace(E, slots, N, Kp);
}

// whether sqmp_gemv_w4 gathers these rows itself (amap)
extern "C" int sqmp_gemv_gathers(int dtype, int M, int Kp, int S_pad) {
  return M <= (dtype == SQMP_F32 ? SQMP_GEMV_MAX_ROWS : 16) &&
         w4::stage_bytes(dtype, M, Kp, S_pad) <= w4::STAGE_BYTES;
}

extern "C" int sqmp_gemv_w4(const void* x, long ldx, int cols, const int32_t* amap,
                            const int32_t* salient, int S, const void* codes_t, const void* scale_t,
                            const void* sal_t, const void* bias, void* y, int dtype, int M, int N,
                            int Kp, int S_pad, int Gw, int ngw, void* workspace, size_t ws_bytes,
                            void* stream) {
  SQMP_DEVICE_GUARD(stream);
  if (!x || !codes_t || !scale_t || !y || (S_pad > 0 && !sal_t)) return SQMP_EINVAL;
  if (M < 0 || M > SQMP_GEMV_MAX_ROWS) return SQMP_EINVAL;
  if (S < 0 || S > S_pad || (S > 0 && amap && !salient)) return SQMP_EINVAL;
  const int st = w4::check_operand(x, ldx, cols, dtype, N, Kp, S_pad, Gw, ngw, amap != nullptr);
  if (st != SQMP_OK) return st;
  if (amap && !sqmp_gemv_gathers(dtype, M, Kp, S_pad)) return SQMP_EUNSUPPORTED;
  if (M == 0) return SQMP_OK;
  w4::GemvArgs a{};
  a.x = x, a.ldx = ldx, a.codes = (const uint32_t*)codes_t, a.scale = scale_t, a.sal = sal_t;
  a.bias = bias, a.y = y, a.M = M, a.N = N, a.n_out = N;
  a.amap = amap, a.salient = salient, a.S = S;
  a.Kp = Kp, a.S_pad = S_pad, a.Gw = Gw, a.ngw = ngw, a.nk = cols / 64;
  w4::set_groups(a);
  hipStream_t s = (hipStream_t)stream;
  if (w4::gemv_takes_tiles(dtype, M, N) && w4::expert_tiles_ok(a, dtype, 1, M))
    return w4::launch_expert_tiles(a, dtype, 1, M, w4::ACT_NONE,
                                   workspace && ws_bytes >= w4::expert_tiles_workspace(1, M, N, Kp)
                                       ? (float*)workspace : nullptr, s);
  if (dtype == SQMP_F32) return w4::by_group<F32, false, w4::ACT_NONE>(a, 1, M, s);
  if (dtype == SQMP_F16) return w4::by_group<F16, false, w4::ACT_NONE>(a, 1, M, s);
  return w4::by_group<BF16, false, w4::ACT_NONE>(a, 1, M, s);
}

extern "C" int sqmp_expert_linear_w4(const void* x, long ldx, int cols, const int32_t* rows, int top_k,
                                     const int32_t* offsets, int E, const void* codes_t,
                                     const void* scale_t, const void* sal_t, void* y, int dtype,
                                     int slots, int x_rows, int N, int n_out, int Kp, int S_pad, int Gw,
                                     int ngw, int act, void* workspace, size_t ws_bytes,
                                     void* stream) {
  SQMP_DEVICE_GUARD(stream);
  if (!x || !offsets || !codes_t || !scale_t || !y || (S_pad > 0 && !sal_t)) return SQMP_EINVAL;
  if (slots < 0 || x_rows < 0 || E <= 0 || E > 65535 || top_k <= 0) return SQMP_EINVAL;
  if (act < w4::ACT_NONE || act > w4::ACT_GELU) return SQMP_EINVAL;
  // gated: blocks of 16 gate and 16 up rows, n_out of the outputs kept
  if (act != w4::ACT_NONE ? (N % 32 || n_out <= N / 2 - 16 || n_out > N / 2) : n_out != N)
    return SQMP_EINVAL;
  const int st = w4::check_operand(x, ldx, cols, dtype, N, Kp, S_pad, Gw, ngw);
  if (st != SQMP_OK) return st;
  if (slots == 0) return SQMP_OK;
  w4::GemvArgs a{};
  a.x = x, a.ldx = ldx, a.codes = (const uint32_t*)codes_t, a.scale = scale_t, a.sal = sal_t;
  a.y = y, a.N = N, a.n_out = n_out, a.Kp = Kp, a.S_pad = S_pad, a.Gw = Gw, a.ngw = ngw, a.nk = cols / 64;
  a.rows = rows, a.offsets = offsets, a.top_k = top_k;
  w4::set_groups(a);
  hipStream_t s = (hipStream_t)stream;
  // tiles from 12 rows per expert on (few-row kernel / tiles, 8 experts, 4096 -> 2 x 11008 gated: 8 rows
  // each 111 / 133 us, 16: 124 / 115, 24: 184 / 150; 64 of 2048 -> 2 x 1408: 6 rows 48 / 63, 12: 73 / 60);
  // SQMP_EXPERT_ROWS = 0 / a tile height overrides (A/B)
  const char* k = knob("SQMP_EXPERT_ROWS");
  if (w4::expert_tiles_ok(a, dtype, E, x_rows) && (k ? atoi(k) > 0 : slots >= 12L * E))
    return w4::launch_expert_tiles(a, dtype, E, slots, act,
                                   workspace && ws_bytes >= w4::expert_tiles_workspace(E, slots, N, Kp)
                                       ? (float*)workspace : nullptr, s);
  // the most rows an expert can have where a token picks it once (any count is right: more take
  // more passes), or twice the mean where that is less
  const int most = rows ? x_rows : cdiv(slots, top_k), twice = cdiv(slots, E) * 2;
  const int est = most <= 8 || most < twice ? most : twice;
#define SQMP_EX(DTT)                                                                  \
  switch (act) {                                                                      \
    case w4::ACT_SILU: return w4::by_group<DTT, true, w4::ACT_SILU>(a, E, est, s);    \
    case w4::ACT_GELU: return w4::by_group<DTT, true, w4::ACT_GELU>(a, E, est, s);    \
    default: return w4::by_group<DTT, true, w4::ACT_NONE>(a, E, est, s);              \
  }
  if (dtype == SQMP_F32) SQMP_EX(F32)
  if (dtype == SQMP_F16) SQMP_EX(F16)
  SQMP_EX(BF16)
#undef SQMP_EX
}

}  // namespace sqmp
