// Arguments and launchers shared by the few-row kernel (sqmp_gemv.hip) and the expert tiles
// (sqmp_experts.hip).
#pragma once
#include "sqmp_w4.h"

namespace sqmp {
namespace w4 {

struct GemvArgs {
  const void* x;          // D rows of Kp + S_pad positions, row stride ldx elements
  long ldx;
  const uint32_t* codes;  // tile-major operands of one weight, or of E of them
  const void* scale;
  const void* sal;
  const void* bias;       // D [N] or NULL
  void* y;                // D [M][N_out]
  int M, N;               // rows (dense form); weight rows (gated: gate and up rows together)
  int Kp, S_pad, Gw, ngw;
  int nk;                  // stages of codes that x holds: Kp / 64, or fewer (the rest is padding)
  // x in an order of its own (STAGE): operand position p is column amap[p] (< 0: zero), position
  // Kp + j the column salient[j], j < S
  const int32_t *amap, *salient;
  int S;
  // expert form
  const int32_t* rows;     // slot -> flat (token * top_k + j), or NULL: x row = slot
  const int32_t* offsets;  // [E + 1]
  int top_k;
  uint32_t gmul;           // stage -> group (set_groups)
  int n_out;               // columns of y (gated: N / 2 rounded; else N)
};

// The group of stage kt is kt / d, d = Gw / 64 stages per group, without a division: kt m / 2^31
// with m = ceil(2^31 / d) exceeds kt / d by kt (m d - 2^31) / (d 2^31) < 1 / d while kt d < 2^31
// (d and kt are below 2^15 for rows of up to 2 million positions)
inline void set_groups(GemvArgs& a) {
  const uint32_t d = a.Gw >= 64 ? (uint32_t)a.Gw / 64 : 1;
  a.gmul = (uint32_t)(((1ull << 31) + d - 1) / d);
}
__device__ inline int group_of(int kt, const GemvArgs& a) {
  return min((int)__umulhi((uint32_t)kt * 2u, a.gmul), a.ngw - 1);
}

// The tile kernels (many rows per weight): whether they take the call (x_rows: rows of x); the
// bytes of the workspace in which the K parts of split tiles meet (0: none); the launch (ws NULL: no
// tile is split).  a.offsets NULL: one weight, slots = a.M rows.
bool expert_tiles_ok(const GemvArgs& a, int dtype, int E, long x_rows);
size_t expert_tiles_workspace(int E, int slots, int N, int Kp);
int launch_expert_tiles(const GemvArgs& a, int dtype, int E, int slots, int act, float* ws,
                        hipStream_t s);

}  // namespace w4
}  // namespace sqmp
