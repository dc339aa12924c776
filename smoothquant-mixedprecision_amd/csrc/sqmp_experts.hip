// Products grouped by expert for many rows: z[slot] = D( W_e x[row(slot)] ) over the ragged
// segments offsets[e] .. offsets[e + 1], W_e = D(code * scale) (+ exact salient columns), or
// D( act(gate) * up ) for weights whose rows are 16 gate and 16 up rows in turn.
//
// What bounds it: the MFMA (2 slots N K flops) from some 100 rows per expert on, the decoding of the
// codes (13 VALU per 8 in fp16, 20 in bf16) and their bytes below.  A workgroup of 8 waves computes
// up to 128 or 256 slots of one expert by 256 weight rows:
//   * each wave owns 32 weight rows; their codes and scales go straight from the tile-major
//     operands to registers, stages ahead, and are decoded there between the MFMAs -- a decoded
//     fragment feeds all the tile's tokens, and no weight passes through LDS;
//   * the activation rows go to an LDS ring by LDS-DMA, gathered by the slot -> row list as they
//     are loaded, so the tokens are never copied into expert order;
//   * the last tile of an expert runs 64 rows (of 256: 64, 128 or 192), so a ragged segment wastes
//     less than 64 rows of MFMA;
//   * gate and up rows of one output are the two accumulators of one lane: the activation and the
//     product happen in registers, half the output bytes, no second launch;
//   * the tiles of the last, partial round of workgroups are split along K (join_kernel).
// The grid holds every tile that any split of `slots` over the experts can need; the tiles that
// exist are found from the offsets on the GPU (no host synchronisation), the rest return.
// Measured: 16384 x 4096 x 4096 as one expert 423 us (1300 TFLOP/s, 256-row tiles; a library product of
// 8192^3 reaches 1200 on that card), 2 of 8 experts x 2048 tokens, 4096 -> 2 x 11008 gated 710 us
// (1040 TFLOP/s; 616 us at the library's rate), 11008 -> 4096 357 + 20 us of join (980; 295 us); 509
// tokens x 6 of 64, 2048 -> 1408 gated bf16 97 + 13 us (40 us of bytes at the rate of a large copy):
// there the vector pipe decodes for 41 % and the MFMA runs for 27 % of the time.
#include "sqmp_w4_launch.h"

namespace sqmp {
namespace w4 {

typedef int rsrc_t __attribute__((ext_vector_type(4)));

__device__ inline rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  const uint64_t a = (uint64_t)(size_t)base;
  rsrc_t r;
  r[0] = (int)__builtin_amdgcn_readfirstlane((uint32_t)a);
  r[1] = (int)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xFFFFu);
  r[2] = (int)__builtin_amdgcn_readfirstlane(bytes);
  r[3] = 0x00020000;
  return r;
}

// LDS-DMA of 16 B per lane to the wave-uniform LDS base + 16 * lane (no register output: nothing
// of it is in flight that the compiler could reuse).  From asm, because the compiler would wait
// for every LDS-DMA before the next LDS read; s_nop 0: the wait state after the M0 write.
__device__ inline void dma16(const rsrc_t& r, uint32_t voff, uint32_t soff, unsigned char* lds) {
  const uint32_t m0v = __builtin_amdgcn_readfirstlane(
      (uint32_t)(size_t)(__attribute__((address_space(3))) unsigned char*)lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(m0v),
               "v"(voff), "s"(r), "s"(soff)
               : "memory", "m0");
}
template <int N>
__device__ inline void vmwait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ inline void barrier() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");  // no LDS read moves above the barrier
  __builtin_amdgcn_sched_barrier(0);
}
__device__ inline int brev3(int c) { return ((c & 1) << 2) | (c & 2) | ((c >> 2) & 1); }

constexpr int TILE_N = 256;      // weight rows per tile

// A kernel of tiles of up to 16 IMAX slots: a ring of RB bytes of activations in LDS, OCC waves per
// SIMD (two workgroups per CU at 4); SPLIT: waves 0-3 issue all LDS-DMA and waves 4-7 run at a
// higher wave priority
template <int IMAX_, int RB_, int OCC_, bool SPLIT_>
struct Shape {
  static constexpr int IMAX = IMAX_, RB = RB_, OCC = OCC_, ROWS = 16 * IMAX_;
  static constexpr bool SPLIT = SPLIT_;
  static constexpr int CAP = OCC_ == 4 ? 512 : 256;  // workgroups the 256 CUs hold at once
  // of a tile of 16 I slots: ring stages, and stages of codes in registers ahead -- deeper for
  // few rows, whose stages are shorter than a load
  static constexpr int ring(int I) { return RB_ / (I * 2048) < 8 ? RB_ / (I * 2048) : 8; }
  static constexpr int ahead(int I) { return I == 4 ? 4 : 2; }
};
using Large = Shape<16, 131072, 1, true>;
using Medium = Shape<8, 65536, 4, false>;

// What a workgroup computes: expert e, slots [m0, m1), weight tile tn, part `part` of `parts` of the
// K stages (`split`: its place among the split tiles)
struct Tile {
  int e, m0, m1, tn, part, parts, split;
};

// The tiles of all experts are numbered by expert, groups of up to 4 row tiles, weight tile, row
// tile (the row tiles of a group read the same weights).  Whole rounds of `cap` workgroups (those
// the GPU holds at once) take a tile each, in contiguous runs per XCD; the tiles of the last,
// partial round are split along K into as many parts as fit the round, at most smax, whose fp32
// sums meet in the workspace (join_kernel).  join: workgroup bid is the bid-th split tile, whole.
// dense_rows: the segment of a single weight, without offsets.  false: nothing to do
template <int TILE_ROWS>
__device__ inline bool find_tile(const int32_t* offsets, int dense_rows, int E, int tiles_n, int cap,
                                 int smax, int bid, bool join, Tile& t) {
  const int lane = threadIdx.x & 63;
  const int per = (E + 63) >> 6;  // experts per lane (E <= 256: at most 4)
  const int e0 = lane * per;
  int off[5], cnt = 0;
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    const int x = min(e0 + min(i, per), E);
    off[i] = offsets ? offsets[x] : x > 0 ? dense_rows : 0;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < per) cnt += (off[i + 1] - off[i] + TILE_ROWS - 1) / TILE_ROWS;
  int incl = cnt;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(incl, d, 64);
    if (lane >= d) incl += v;
  }
  const int nwg = __builtin_amdgcn_readfirstlane(__shfl(incl, 63, 64)) * tiles_n;
  const int whole = smax > 1 ? nwg / cap * cap : nwg, left = nwg - whole;
  const int parts = left > 0 ? max(1, min(smax, cap / left)) : 1;
  int wg;
  t.part = 0, t.parts = 1, t.split = 0;
  if (join) {
    if (bid >= left || parts == 1) return false;
    wg = whole + bid;
    t.parts = parts, t.split = bid;
  } else if (bid < whole) {
    const int xcd = bid & 7, q = whole >> 3, r = whole & 7;
    wg = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (bid >> 3);
  } else {
    const int b = bid - whole;
    if (b >= left * parts) return false;
    t.split = b / parts, t.part = b - t.split * parts, t.parts = parts;
    wg = whole + t.split;
  }
  // the lane, then the expert within it, whose tiles hold wg
  const uint64_t mask = __ballot(incl * tiles_n > wg);
  const int src = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)mask) - 1);
  int rem = wg - __shfl(incl - cnt, src, 64) * tiles_n;
  int found = 0, lo = 0, hi = 0, done = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int a = __shfl(off[i], src, 64), b = __shfl(off[i + 1], src, 64);
    const int n = i < per ? (b - a + TILE_ROWS - 1) / TILE_ROWS * tiles_n : 0;
    if (!done && rem < n) found = src * per + i, lo = a, hi = b, done = 1;
    if (!done) rem -= n;
  }
  const int tiles_m = (hi - lo + TILE_ROWS - 1) / TILE_ROWS;
  const int gid = rem / (4 * tiles_n), first = gid * 4, gsz = min(tiles_m - first, 4);
  const int in_g = rem - gid * 4 * tiles_n;
  t.e = __builtin_amdgcn_readfirstlane(found);
  t.m0 = __builtin_amdgcn_readfirstlane(lo + (first + in_g % gsz) * TILE_ROWS);
  t.m1 = __builtin_amdgcn_readfirstlane(min(hi, lo + (first + in_g % gsz + 1) * TILE_ROWS));
  t.tn = __builtin_amdgcn_readfirstlane(in_g / gsz);
  t.part = __builtin_amdgcn_readfirstlane(t.part), t.parts = __builtin_amdgcn_readfirstlane(t.parts);
  t.split = __builtin_amdgcn_readfirstlane(t.split);
  return true;
}

// One tile (or one K part of it) of 16 I slots (I / 4 LDS-DMA pieces per wave and stage)
template <class DT, int GB, bool GATED, class SH, int I>
__device__ inline void run_tile(const GemvArgs& a, int act, const Tile& t, unsigned char* lds,
                                float* part_sums) {
  typedef typename DT::T T;
  constexpr int J = 2, NA = I / 4, PF = I == 16 || (I == 8 && SH::OCC == 4) ? 2 : 3;
  constexpr int SLOT = I * 16 * 128, RING = SH::ring(I), DW = SH::ahead(I);
  constexpr int NO = SH::SPLIT ? 2 : 1;  // waves whose pieces a loading wave issues
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int r16 = lane & 15, q = lane >> 4;
  const int e = t.e, m0 = t.m0, nm = t.m1 - t.m0, tn = t.tn;
  const int nks_all = a.S_pad / 64, nkm_all = a.nk;
  // this part's stages: codes [k0, nkm), then (last part) the salient ones up to nkt
  const int k0 = (int)((long)nkm_all * t.part / t.parts) & ~3;
  const bool last = t.part + 1 == t.parts;
  const int nkm = last ? nkm_all : (int)((long)nkm_all * (t.part + 1) / t.parts) & ~3;
  const int nks = last ? nks_all : 0, nkt = nkm + nks;

  // activation rows: piece i of a wave = rows 64 i + 8 wave + (lane >> 3); the lane brings the
  // chunk that belongs at physical place lane & 7 of its row (chunk c at brev3(c) ^ (row / 2))
  const T* xb = (const T*)a.x;
  if (!a.rows) xb += (long)m0 * a.ldx;
  const rsrc_t rA = make_rsrc(xb, 0xFFFFFFFFu);
  uint32_t a_off[NO][NA];
#pragma unroll
  for (int o = 0; o < NO; ++o)
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int row = 64 * i + 8 * ((wave + 4 * o) & 7) + (lane >> 3);
      const int rr = min(row, nm - 1);  // (rows past the segment repeat its last one)
      const long xr = a.rows ? a.rows[m0 + rr] / a.top_k : rr;
      a_off[o][i] = (uint32_t)(xr * a.ldx * (long)sizeof(T)) +
                    (uint32_t)(brev3((lane & 7) ^ ((row >> 1) & 7)) << 4);
    }
  const bool loads = !SH::SPLIT || wave < 4;
  auto issue_a = [&](int kt) {
    if (!loads) return;
    unsigned char* slot = lds + (kt % RING) * SLOT + wave * 1024;
#pragma unroll
    for (int o = 0; o < NO; ++o)
#pragma unroll
      for (int i = 0; i < NA; ++i)
        dma16(rA, a_off[o][i], (uint32_t)kt * 128, slot + o * 4096 + i * 8192);
  };
  // One barrier per BPS stages (short stages: two).  Before it this wave's part of those stages has
  // to be in LDS -- at most the LDS-DMA of the stages behind them (the youngest operations; codes
  // loads among them only make it wait for more) is in flight; after it everyone's part is, and
  // nobody reads the BPS stages before any more, whose ring places the next loads take.
  constexpr int BPS = I == 4 && SH::OCC == 4 ? 2 : 1, FLY = RING - 2 * BPS;
  auto enter = [&](int kt) {
    if (BPS == 2 && ((kt - k0) & 1)) return;
    if (loads) {
      if (nkt - BPS - kt >= FLY) vmwait<FLY * NO * NA>(); else vmwait<0>();
    }
    barrier();
#pragma unroll
    for (int b = 0; b < BPS; ++b)
      if (kt + RING - BPS + b < nkt) issue_a(kt + RING - BPS + b);
  };

  // weights
  const long wb = (long)e * ((a.N + 255) / 256 * 8) + tn * 8 + wave;
  const __amdgpu_buffer_rsrc_t rW = rsrc_of(a.codes + wb * (a.Kp / 64) * 256);
  const __amdgpu_buffer_rsrc_t rS = rsrc_of((const T*)a.scale + wb * a.ngw * 32);
  struct Codes {
    u32x4 w;
    uint32_t s;
  };
  auto load_w = [&](int kt, Codes& c) {
    c.w = load16(rW, (uint32_t)lane * 16, (uint32_t)kt * 1024);
    if constexpr (GB == 1) c.s = load4(rS, (uint32_t)r16 * 4, (uint32_t)group_of(kt, a) * 64);
    else c.s = load4(rS, (uint32_t)min(2 * kt + (q & 1), a.ngw - 1) * 64 + (uint32_t)r16 * 4, 0);
  };

  f32x4 acc[I][J];
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const DecK dk = make_deck();
  uint32_t a_lo[2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
    a_lo[s] = (uint32_t)(r16 * 128 + ((brev3(4 * (q & 1) + 2 * s + (q >> 1)) ^ ((r16 >> 1) & 7)) << 4));
  auto lda = [&](const unsigned char* slot, int t) {
    return *(const u32x4*)(slot + (t % I) * 2048 + a_lo[t / I]);
  };
  // 2 I blocks (sub-step t / I, token tile t % I) with the fragments read PF blocks ahead
  auto blocks = [&](const unsigned char* slot, auto bf, auto hook) {
    u32x4 f[PF + 1];
#pragma unroll
    for (int t = 0; t < PF; ++t) f[t] = lda(slot, t);
#pragma unroll
    for (int t = 0; t < 2 * I; ++t) {
      if (t + PF < 2 * I) f[(t + PF) % (PF + 1)] = lda(slot, t + PF);
#pragma unroll
      for (int j = 0; j < J; ++j) Mfma<DT>::run(acc[t % I][j], bf(t / I, j), f[t % (PF + 1)]);
      hook(t);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // Codes are decoded between the MFMAs: sub-step 1 of this stage in its first blocks, sub-step 0 of
  // the next one in the blocks that no longer use it, so vector and matrix pipes work side by side
  // and a stage starts with its MFMAs.  (The compiler waits for codes by counting its own loads only,
  // which makes it wait for LDS-DMA issued in between as well: codes are loaded far ahead.)
  Codes cs[DW];
#pragma unroll
  for (int p = 0; p < (RING - BPS > DW ? RING - BPS : DW); ++p) {
    if (p < RING - BPS && k0 + p < nkt) issue_a(k0 + p);
    if (p < DW) load_w(min(k0 + p, nkm - 1), cs[p]);
  }
  u32x4 bf[2][J];
  auto dec = [&](const Codes& c, int s, int n) {  // half n & 1 of fragment [s][n / 2]
    const int j = n >> 1;
    DecHalf<DT>::run(bf[s][j], c.w[2 * j + s], Dec<DT>::prep(j ? c.s >> 16 : c.s & 0xFFFFu), dk, n & 1);
  };
#pragma unroll
  for (int n = 0; n < 2 * J; ++n) dec(cs[0], 0, n);
  auto step = [&](int kt, Codes& c, const Codes& next) {
    enter(kt);
    blocks(lds + (kt % RING) * SLOT, [&](int s, int j) -> const u32x4& { return bf[s][j]; },
           [&](int t) {
             if (t < 2 * J) dec(c, 1, t);
             if (t == 2 * J) load_w(min(kt + DW, nkm - 1), c);
             if (t >= I && t < I + 2 * J) dec(next, 0, t - I);
           });
  };
  if (SH::SPLIT && wave >= 4) __builtin_amdgcn_s_setprio(1);
  for (int kt = k0; kt < nkm; kt += DW)
#pragma unroll
    for (int u = 0; u < DW; ++u)
      if (kt + u < nkm) step(kt + u, cs[u], cs[(u + 1) % DW]);
  // the exact salient columns: fragments as they are
  for (int kd = 0; kd < nks; ++kd) {
    const int kt = nkm + kd;
    const T* sal = (const T*)a.sal + (wb * nks_all + kd) * 2048 + lane * 32;
    u32x4 d[2][J];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int j = 0; j < J; ++j) d[s][j] = *(const u32x4*)(sal + j * 16 + s * 8);
    enter(kt);
    blocks(lds + (kt % RING) * SLOT, [&](int s, int j) -> const u32x4& { return d[s][j]; },
           [](int) {});
  }
  if (SH::SPLIT && wave >= 4) __builtin_amdgcn_s_setprio(0);

  const int tid = threadIdx.x, er = r16, eq = q;
  if (t.parts > 1) {  // fp32 sums in fragment order (16 bytes a lane, whole lines)
    f32x4* ps = (f32x4*)part_sums + (long)(t.split * t.parts + t.part) * (SH::IMAX * J * 512) + tid;
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j) ps[(i * J + j) * 512] = acc[i][j];
    return;
  }
  // epilogue: the tile in LDS (16-B chunk c of row m at c ^ (m & 15)), then whole rows out
  constexpr int TNO = GATED ? TILE_N / 2 : TILE_N;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  barrier();
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int m = 16 * i + er;
#pragma unroll
    for (int j = 0; j < (GATED ? 1 : J); ++j) {
      const int nl = GATED ? 16 * wave + 4 * eq : 32 * wave + 16 * j + 4 * eq;
      T v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float f = acc[i][j][r];
        if constexpr (!GATED)
          if (a.bias && tn * TILE_N + nl + r < a.N) f += DT::to_f(((const T*)a.bias)[tn * TILE_N + nl + r]);
        if constexpr (GATED)
          f = (act == ACT_SILU ? act_fn<ACT_SILU>(f) : act_fn<ACT_GELU>(f)) * acc[i][1][r];
        v[r] = DT::from_f(f);
      }
      *(uint64_t*)(lds + m * (TNO * 2) + (((nl >> 3) ^ (m & 15)) << 4) + (nl & 4) * 2) = *(const uint64_t*)v;
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  barrier();
  constexpr int CPR = TNO / 8;
  const int n0 = tn * TNO;
  T* y = (T*)a.y + (long)m0 * a.n_out + n0;
  const bool vec = a.n_out % 8 == 0 && (size_t)a.y % 16 == 0;
  for (int k = tid; k < nm * CPR; k += 512) {
    const int m = k / CPR, c = k % CPR;
    const u32x4 val = *(const u32x4*)(lds + m * (TNO * 2) + ((c ^ (m & 15)) << 4));
    const int n = n0 + 8 * c;
    if (vec) {
      if (n < a.n_out) *(u32x4*)(y + (long)m * a.n_out + 8 * c) = val;
    } else {
      const T* v = (const T*)&val;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < a.n_out) y[(long)m * a.n_out + 8 * c + i] = v[i];
    }
  }
}

template <class DT, int GB, bool GATED, class SH>
__global__ __launch_bounds__(512, SH::OCC) void expert_tiles_kernel(const GemvArgs a, int E,
                                                                    int tiles_n, int act, int smax,
                                                                    float* part_sums) {
  constexpr int RB = SH::RB;
  constexpr int EPI = SH::ROWS * (GATED ? TILE_N / 2 : TILE_N) * 2;
  __shared__ __attribute__((aligned(16))) unsigned char lds[RB > EPI ? RB : EPI];
  Tile t;
  if (!find_tile<SH::ROWS>(a.offsets, a.M, E, tiles_n, SH::CAP, smax, blockIdx.x, false, t)) return;
  const int nm = t.m1 - t.m0;
  if constexpr (SH::IMAX >= 16) {
    if (nm > 192) return run_tile<DT, GB, GATED, SH, 16>(a, act, t, lds, part_sums);
    if (nm > 128) return run_tile<DT, GB, GATED, SH, 12>(a, act, t, lds, part_sums);
  }
  if constexpr (SH::IMAX >= 8) {
    if (nm > 64) return run_tile<DT, GB, GATED, SH, 8>(a, act, t, lds, part_sums);
  }
  run_tile<DT, GB, GATED, SH, 4>(a, act, t, lds, part_sums);
}

// The split tiles: their parts' sums added in the order of K, activation, one rounding.  blockIdx.y:
// a 16-row slice of the tile and two of its waves' columns (small blocks: few tiles have to keep
// every CU reading)
template <class DT, bool GATED, class SH>
__global__ __launch_bounds__(128) void join_kernel(const GemvArgs a, int E, int tiles_n, int act,
                                                   int smax, const float* part_sums) {
  typedef typename DT::T T;
  Tile t;
  if (!find_tile<SH::ROWS>(a.offsets, a.M, E, tiles_n, SH::CAP, smax, blockIdx.x, true, t)) return;
  const int i = blockIdx.y >> 2, lane = threadIdx.x & 63;
  const int wave = (blockIdx.y & 3) * 2 + (threadIdx.x >> 6);
  const int m = 16 * i + (lane & 15), q = lane >> 4;
  if (16 * i >= t.m1 - t.m0) return;
  const f32x4* ps = (const f32x4*)part_sums + (long)t.split * t.parts * (SH::IMAX * 1024) + i * 1024 + 64 * wave + lane;
  f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll 4
  for (int p = 0; p < t.parts; ++p) {
    s[0] += ps[(long)p * (SH::IMAX * 1024)];
    s[1] += ps[(long)p * (SH::IMAX * 1024) + 512];
  }
  if (m >= t.m1 - t.m0) return;
  T* y = (T*)a.y + (long)(t.m0 + m) * a.n_out;
#pragma unroll
  for (int j = 0; j < (GATED ? 1 : 2); ++j) {
    const int n0 = GATED ? t.tn * 128 + 16 * wave + 4 * q : t.tn * 256 + 32 * wave + 16 * j + 4 * q;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float f = s[j][r];
      if constexpr (GATED) f = (act == ACT_SILU ? act_fn<ACT_SILU>(f) : act_fn<ACT_GELU>(f)) * s[1][r];
      const int n = n0 + r;
      if (n < a.n_out) y[n] = DT::from_f(a.bias ? f + DT::to_f(((const T*)a.bias)[n]) : f);
    }
  }
}

// The tile height, by the mean rows of an expert.  128 / 256 rows, us, 2 of 8 experts, ragged: 4096 ->
// 2 x 11008 gated, fp16, 128 rows each 275 / 367, 512: 694 / 725, 1024: 1293 / 1293, 2048: 2513 / 2490, 4096:
// 5019 / 5081; bf16 512: 726 / 732, 1024: 1326 / 1283, 2048: 2576 / 2479, 4096: 5177 / 5043.  The way down has
// fewer tiles and depends on how full their last round is: 11008 -> 4096 fp16 1024: 638 / 660, 2048: 1289 /
// 1407, 4096: 2453 / 2715; bf16 1536: 964 / 937, 2048: 1301 / 1396, 4096: 2552 / 2695; 4096 -> 4096 fp16 2048:
// 470 / 449 and 472 / 502 on two cards.  SQMP_EXPERT_ROWS overrides (A/B)
static int tile_rows(int E, int slots) {
  const char* k = knob("SQMP_EXPERT_ROWS");
  const int r = k && atoi(k) > 0 ? atoi(k) : slots / E < 2048 ? 128 : 256;
  return r <= 128 ? 128 : 256;
}

// The parts a tile of the last round may be split into: at least 8 stages each, and only where
// the last round is a good part of the whole (fewer than 4 full rounds at the least)
static int max_parts(int E, int slots, int N, int Kp) {
  const int rows = tile_rows(E, slots), cap = rows == 256 ? Large::CAP : Medium::CAP;
  if ((long)cdiv(slots, rows) * cdiv(N, TILE_N) >= 4L * cap) return 1;
  const int p = Kp / 64 / 8;
  return p < 2 ? 1 : p > 16 ? 16 : p;
}

size_t expert_tiles_workspace(int E, int slots, int N, int Kp) {
  if (slots <= 0 || max_parts(E, slots, N, Kp) == 1) return 0;
  const int rows = tile_rows(E, slots), cap = rows == 256 ? Large::CAP : Medium::CAP;
  // the parts of one round: no more than cap, and no more than every tile in max_parts
  const long tiles = ((long)slots / rows + (slots < E ? slots : E)) * cdiv(N, TILE_N);
  const long most = tiles * max_parts(E, slots, N, Kp);
  return (size_t)(most < cap ? most : cap) * rows * TILE_N * sizeof(float);
}

template <class DT, int GB, bool GATED, class SH>
static int launch_tiles(const GemvArgs& a, int E, int slots, int act, float* ws, hipStream_t s) {
  const int tiles_n = cdiv(a.N, TILE_N);
  const int smax = ws ? max_parts(E, slots, a.N, a.Kp) : 1;
  const long tiles = ((long)slots / SH::ROWS + (slots < E ? slots : E)) * tiles_n;
  const long extra = smax > 1 ? (tiles * smax < SH::CAP ? tiles * smax : SH::CAP) : 0;
  const long grid = tiles + extra;
  if (grid > 0x7FFFFFFFL) return SQMP_EUNSUPPORTED;
  expert_tiles_kernel<DT, GB, GATED, SH><<<dim3((unsigned)grid), dim3(512), 0, s>>>(a, E, tiles_n, act, smax, ws);
  SQMP_LAUNCH_CHECK();
  if (smax > 1) {
    const long nj = tiles < SH::CAP / 2 ? tiles : SH::CAP / 2;  // two parts or more: at most cap / 2
    join_kernel<DT, GATED, SH><<<dim3((unsigned)nj, SH::IMAX * 4), dim3(128), 0, s>>>(a, E, tiles_n, act, smax, ws);
    SQMP_LAUNCH_CHECK();
  }
  return SQMP_OK;
}

template <class DT, int GB, bool GATED>
static int by_shape(const GemvArgs& a, int E, int slots, int act, float* ws, hipStream_t s) {
  if (tile_rows(E, slots) == 128) return launch_tiles<DT, GB, GATED, Medium>(a, E, slots, act, ws, s);
  return launch_tiles<DT, GB, GATED, Large>(a, E, slots, act, ws, s);
}

template <class DT>
static int by_group_act(const GemvArgs& a, int E, int slots, int act, float* ws, hipStream_t s) {
  if (a.Gw == 32)
    return act != ACT_NONE ? by_shape<DT, 2, true>(a, E, slots, act, ws, s) : by_shape<DT, 2, false>(a, E, slots, act, ws, s);
  return act != ACT_NONE ? by_shape<DT, 1, true>(a, E, slots, act, ws, s) : by_shape<DT, 1, false>(a, E, slots, act, ws, s);
}

bool expert_tiles_ok(const GemvArgs& a, int dtype, int E, long x_rows) {
  // fp16 / bf16, groups of 32 or of whole stages, a 32-bit offset to every activation
  return (dtype == SQMP_F16 || dtype == SQMP_BF16) && (a.Gw % 64 == 0 || a.Gw == 32) && E <= 256 &&
         (a.rows ? x_rows : 256) * a.ldx * 2 < 0xFFFF0000L;
}

int launch_expert_tiles(const GemvArgs& a, int dtype, int E, int slots, int act, float* ws,
                        hipStream_t s) {
  return dtype == SQMP_F16 ? by_group_act<F16>(a, E, slots, act, ws, s) : by_group_act<BF16>(a, E, slots, act, ws, s);
}

}  // namespace w4
}  // namespace sqmp
