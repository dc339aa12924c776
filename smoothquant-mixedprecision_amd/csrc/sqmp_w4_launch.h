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
  // expert form
  const int32_t* rows;     // slot -> flat (token * top_k + j), or NULL: x row = slot
  const int32_t* offsets;  // [E + 1]
  int top_k;
  int n_out;               // columns of y (gated: N / 2 rounded; else N)
};

// The tile kernels (many rows per weight): whether they take the call (x_rows: rows of x); the
// bytes of the workspace in which the K parts of split tiles meet (0: none); the launch (ws NULL: no
// tile is split).  a.offsets NULL: one weight, slots = a.M rows.
bool expert_tiles_ok(const GemvArgs& a, int dtype, int E, long x_rows);
size_t expert_tiles_workspace(int E, int slots, int N, int Kp);
int launch_expert_tiles(const GemvArgs& a, int dtype, int E, int slots, int act, float* ws,
                        hipStream_t s);

}  // namespace w4
}  // namespace sqmp
