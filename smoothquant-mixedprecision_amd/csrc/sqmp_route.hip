// Routing of tokens to experts, and the way back.
//
//   sqmp_route        per token the k largest logits (ties: the lowest index; NaN counts as the
//                     largest, -inf is never chosen), their softmax weights, and the plan below
//   sqmp_plan_routes  the plan alone, for ids chosen elsewhere: the chosen (token, expert) pairs
//                     f = token * k + j in stable order by expert --
//                       offsets[e] = pairs of experts below e, rows[slot] = f, slots[f] = slot
//                     (-1 in ids, slots and the rows behind the last pair: nothing chosen)
//   sqmp_combine      y[t] = D( sum_j w[t][j] z[slots[t][j]] ), fp32 sums in the order of j
//   sqmp_pack_rows    the activation operand of packed weights (columns gathered by a map)
//
// The order is a counting sort: a block of 256 tokens counts its pairs per expert, an exclusive
// scan over the blocks places them, and inside a block the pairs are ranked 64 at a time by
// ballots.  No atomics: slots depend on the ids alone.
#include "sqmp_common.h"

namespace sqmp {
namespace route {

constexpr int TB = 256;          // tokens (and threads) per block
constexpr int E_MAX = 256, K_MAX = 16;
constexpr int NWAVE = TB / 64;

// descending order of floats as unsigned order: NaN highest, -0 equal to +0
__device__ inline uint32_t order_key(float v) {
  if (v != v) return 0xFFFFFFFFu;
  uint32_t u = __float_as_uint(v);
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
constexpr uint32_t KEY_NEG_INF = 0x007FFFFFu;  // order_key(-inf)

__device__ inline float key_value(uint32_t k) {
  if (k == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// lanes of the wave whose expert equals this lane's (nbits bits of e are compared)
__device__ inline uint64_t same_expert(int e, int nbits) {
  uint64_t m = ~0ull;
  for (int b = 0; b < nbits; ++b) {
    const uint64_t bal = __ballot((e >> b) & 1);
    m &= ((e >> b) & 1) ? bal : ~bal;
  }
  return m;
}

// Ranks of a block's pairs.  cnt[chunk][e]: pairs of expert e in 64-pair chunk `chunk`.
__device__ inline void count_chunks(const int32_t* ids, long f0, long f1, int E, int nbits,
                                    uint16_t* cnt) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int chunks = (int)((f1 - f0 + 63) / 64);
  for (int i = threadIdx.x; i < chunks * E; i += TB) cnt[i] = 0;
  __syncthreads();
  for (int c = wave; c < chunks; c += NWAVE) {
    const long f = f0 + c * 64 + lane;
    int e = f < f1 ? ids[f] : -1;
    if (e < 0 || e >= E) e = E;  // nothing chosen
    const uint64_t m = same_expert(e, nbits);
    if (e < E && (m & ((1ull << lane) - 1)) == 0) cnt[c * E + e] = (uint16_t)__popcll(m);
  }
  __syncthreads();
}

// hist[blk][e] of one block's ids
__device__ inline void block_hist(const uint16_t* cnt, int chunks, int E, int32_t* hist) {
  for (int e = threadIdx.x; e < E; e += TB) {
    int s = 0;
    for (int c = 0; c < chunks; ++c) s += cnt[c * E + e];
    hist[e] = s;
  }
}

// start[e] = first slot of this block's pairs of expert e; writes the pairs' slots
__device__ inline void scatter(const int32_t* ids, long f0, long f1, int E, int nbits,
                               const uint16_t* cnt, int32_t* at /* LDS [E], consumed */,
                               uint16_t* base /* LDS [chunks][E] */, int32_t* rows,
                               int32_t* slots, int total) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int chunks = (int)((f1 - f0 + 63) / 64);
  for (int e = threadIdx.x; e < E; e += TB) {
    int s = 0;
    for (int c = 0; c < chunks; ++c) {
      base[c * E + e] = (uint16_t)s;
      s += cnt[c * E + e];
    }
  }
  __syncthreads();
  for (int c = wave; c < chunks; c += NWAVE) {
    const long f = f0 + c * 64 + lane;
    int e = f < f1 ? ids[f] : -1;
    if (e < 0 || e >= E) e = E;
    const uint64_t m = same_expert(e, nbits);
    if (f < f1) {
      int slot = -1;
      if (e < E) {
        slot = at[e] + base[c * E + e] + (int)__popcll(m & ((1ull << lane) - 1));
        rows[slot] = (int32_t)f;
      }
      slots[f] = slot;
      if (f >= total) rows[f] = -1;  // behind the last pair
    }
  }
}

// at[e] (LDS) = exclusive prefix of tot[e] (+ base[e]); returns the total.  E <= 256 = TB
__device__ inline int scan_experts(const int32_t* tot, const int32_t* base, int E, int32_t* at,
                                   int32_t* tmp, int32_t* offsets) {
  const int e = threadIdx.x;
  int v = e < E ? tot[e] : 0;
  tmp[e] = v;
  __syncthreads();
  for (int d = 1; d < TB; d <<= 1) {
    const int add = e >= d ? tmp[e - d] : 0;
    __syncthreads();
    tmp[e] += add;
    __syncthreads();
  }
  const int total = tmp[TB - 1];
  if (e < E) {
    at[e] = tmp[e] - v + (base ? base[e] : 0);
    if (offsets) offsets[e] = tmp[e] - v;
  }
  if (offsets && e == 0) offsets[E] = total;
  __syncthreads();
  return total;
}

// The k largest of a token's E logits, one thread per token; rows staged in LDS (coalesced).
template <class DT, int KT>
__device__ inline void top_k_rows(const typename DT::T* logits, long ldl, int t0, int nt, int E,
                                  int k, int normalize, float* tile, float* weights,
                                  int32_t* ids) {
  const int pitch = E | 1;  // odd: a thread per row is conflict free
  constexpr int ROWS = 64;  // tokens staged at once
  for (int r0 = 0; r0 < nt; r0 += ROWS) {
    const int nr = min(ROWS, nt - r0);
    __syncthreads();
    for (int i = threadIdx.x; i < nr * E; i += TB) {
      const int r = i / E, e = i - r * E;
      tile[r * pitch + e] = DT::to_f(logits[(t0 + r0 + r) * ldl + e]);
    }
    __syncthreads();
    if ((int)threadIdx.x < nr) {
      const float* row = tile + threadIdx.x * pitch;
      uint32_t key[KT];
      int idx[KT];
#pragma unroll
      for (int j = 0; j < KT; ++j) key[j] = KEY_NEG_INF, idx[j] = -1;
      for (int e = 0; e < E; ++e) {
        const uint32_t ke = order_key(row[e]);
        if (ke > key[KT - 1]) {  // strictly: equal logits keep the lower index
          uint32_t ck = ke;
          int ci = e;
          bool up = false;  // inserted: the rest moves down one place, equal logits included
#pragma unroll
          for (int j = 0; j < KT; ++j) {
            up = up || ck > key[j];
            const uint32_t ok = key[j];
            const int oi = idx[j];
            key[j] = up ? ck : ok, idx[j] = up ? ci : oi;
            ck = up ? ok : ck, ci = up ? oi : ci;
          }
        }
      }
      const float top = key_value(key[0]);
      float ex[KT], den = 0.f;
#pragma unroll
      for (int j = 0; j < KT; ++j) {
        ex[j] = idx[j] >= 0 && j < k ? expf(key_value(key[j]) - top) : 0.f;
        den += ex[j];
      }
      if (!normalize && idx[0] >= 0) {
        den = 0.f;
        for (int e = 0; e < E; ++e) den += expf(row[e] - top);
      }
      const long f = (long)(t0 + r0 + threadIdx.x) * k;
#pragma unroll
      for (int j = 0; j < KT; ++j)
        if (j < k) {
          weights[f + j] = idx[j] >= 0 ? ex[j] / den : 0.f;
          ids[f + j] = idx[j];
        }
    }
  }
  __syncthreads();
}

struct Args {
  const void* logits;  // NULL: ids are given
  long ldl;
  int T, E, k, normalize;
  float* weights;
  int32_t* ids;
  int32_t *offsets, *rows, *slots;
  int32_t* hist;       // [blocks][E]
};

__host__ __device__ inline int bits_of(int E) {  // values 0 .. E
  int b = 0;
  while ((1 << b) <= E) ++b;
  return b;
}

constexpr int TILE_F = 64 * (E_MAX | 1);           // floats of the logits tile
constexpr int MAX_CHUNKS = TB * K_MAX / 64;        // 64
// LDS: the tile, then (reused) two [chunks][E] tables of 16 bits
constexpr int LDS_WORDS = TILE_F > MAX_CHUNKS * E_MAX ? TILE_F : MAX_CHUNKS * E_MAX;

// one block of tokens: choose (or read) the ids and count them; ONE: the only block finishes
template <class DT, int KT, bool ONE>
__global__ __launch_bounds__(TB) void route_kernel(const Args a) {
  __shared__ float lds[LDS_WORDS];
  __shared__ int32_t at[E_MAX], tmp[TB], tot[E_MAX];
  const int t0 = blockIdx.x * TB, nt = min(TB, a.T - t0);
  if (a.logits)
    top_k_rows<DT, KT>((const typename DT::T*)a.logits, a.ldl, t0, nt, a.E, a.k, a.normalize, lds,
                       a.weights, a.ids);
  __threadfence_block();
  __syncthreads();
  const long f0 = (long)t0 * a.k, f1 = f0 + (long)nt * a.k;
  const int nbits = bits_of(a.E);
  uint16_t* cnt = (uint16_t*)lds;
  const int chunks = (int)((f1 - f0 + 63) / 64);
  count_chunks(a.ids, f0, f1, a.E, nbits, cnt);
  if constexpr (!ONE) {
    block_hist(cnt, chunks, a.E, a.hist + (long)blockIdx.x * a.E);
  } else {
    block_hist(cnt, chunks, a.E, tot);
    __syncthreads();
    const int total = scan_experts(tot, nullptr, a.E, at, tmp, a.offsets);
    scatter(a.ids, f0, f1, a.E, nbits, cnt, at, cnt + MAX_CHUNKS * E_MAX, a.rows, a.slots, total);
  }
}

// hist[blk][e] -> exclusive scan over the blocks, hist[blocks][e] = the expert's total
__global__ __launch_bounds__(TB) void scan_kernel(int32_t* hist, int blocks, int E) {
  __shared__ int32_t part[TB];
  const int e = blockIdx.x;
  const int per = (blocks + TB - 1) / TB;
  const int b0 = min((int)threadIdx.x * per, blocks), b1 = min(b0 + per, blocks);
  int s = 0;
  for (int b = b0; b < b1; ++b) s += hist[(long)b * E + e];
  part[threadIdx.x] = s;
  __syncthreads();
  for (int d = 1; d < TB; d <<= 1) {
    const int add = (int)threadIdx.x >= d ? part[threadIdx.x - d] : 0;
    __syncthreads();
    part[threadIdx.x] += add;
    __syncthreads();
  }
  int run = part[threadIdx.x] - s;
  for (int b = b0; b < b1; ++b) {
    const int v = hist[(long)b * E + e];
    hist[(long)b * E + e] = run;
    run += v;
  }
  if (threadIdx.x == TB - 1) hist[(long)blocks * E + e] = part[TB - 1];
}

__global__ __launch_bounds__(TB) void scatter_kernel(const Args a, int blocks) {
  __shared__ float lds[LDS_WORDS];
  __shared__ int32_t at[E_MAX], tmp[TB];
  const int t0 = blockIdx.x * TB, nt = min(TB, a.T - t0);
  const long f0 = (long)t0 * a.k, f1 = f0 + (long)nt * a.k;
  const int nbits = bits_of(a.E);
  uint16_t* cnt = (uint16_t*)lds;
  const int total = scan_experts(a.hist + (long)blocks * a.E, a.hist + (long)blockIdx.x * a.E, a.E,
                                 at, tmp, blockIdx.x == 0 ? a.offsets : nullptr);
  count_chunks(a.ids, f0, f1, a.E, nbits, cnt);
  scatter(a.ids, f0, f1, a.E, nbits, cnt, at, cnt + MAX_CHUNKS * E_MAX, a.rows, a.slots, total);
}

template <class DT, int KT>
static int launch(const Args& a, hipStream_t s) {
  const int blocks = cdiv(a.T, TB);
  if (blocks == 1) {
    route_kernel<DT, KT, true><<<dim3(1), dim3(TB), 0, s>>>(a);
    SQMP_LAUNCH_CHECK();
    return SQMP_OK;
  }
  route_kernel<DT, KT, false><<<dim3(blocks), dim3(TB), 0, s>>>(a);
  SQMP_LAUNCH_CHECK();
  scan_kernel<<<dim3(a.E), dim3(TB), 0, s>>>(a.hist, blocks, a.E);
  SQMP_LAUNCH_CHECK();
  scatter_kernel<<<dim3(blocks), dim3(TB), 0, s>>>(a, blocks);
  SQMP_LAUNCH_CHECK();
  return SQMP_OK;
}

template <class DT>
static int by_k(const Args& a, hipStream_t s) {
  if (a.k <= 2) return launch<DT, 2>(a, s);
  if (a.k <= 4) return launch<DT, 4>(a, s);
  if (a.k <= 8) return launch<DT, 8>(a, s);
  return launch<DT, 16>(a, s);
}

// ---------------------------------------------------------------- combine
template <class DT, int V>
__global__ __launch_bounds__(256) void combine_kernel(const typename DT::T* __restrict__ z,
                                                      const int32_t* __restrict__ slots,
                                                      const float* __restrict__ w,
                                                      typename DT::T* __restrict__ y, long T,
                                                      int k, int H) {
  typedef typename DT::T T_;
  const int per = (H + V - 1) / V;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= T * per) return;
  const long t = i / per;
  const int h = (int)(i - t * per) * V;
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.f;
  for (int j = 0; j < k; ++j) {
    const int s = slots[t * k + j];
    if (s < 0) continue;  // nothing chosen
    const float wj = w[t * k + j];
    struct __attribute__((aligned(sizeof(T_) * V))) Vec { T_ e[V]; };
    const Vec zv = *(const Vec*)(z + (long)s * H + h);
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = __builtin_fmaf(wj, DT::to_f(zv.e[v]), acc[v]);
  }
  struct __attribute__((aligned(sizeof(T_) * V))) Out { T_ e[V]; } o;
#pragma unroll
  for (int v = 0; v < V; ++v) o.e[v] = DT::from_f(acc[v]);
  *(Out*)(y + t * H + h) = o;
}

template <class DT>
static int launch_combine(const void* z, const int32_t* slots, const float* w, void* y, int T,
                          int k, int H, hipStream_t s) {
  typedef typename DT::T T_;
  constexpr int V = 16 / sizeof(T_);
  const bool vec = H % V == 0 && (size_t)z % 16 == 0 && (size_t)y % 16 == 0;
  const long n = (long)T * (vec ? H / V : H);
  const long blocks = (n + 255) / 256;
  if (blocks > 0x7FFFFFFFL) return SQMP_EUNSUPPORTED;
  if (vec)
    combine_kernel<DT, V><<<dim3((unsigned)blocks), dim3(256), 0, s>>>((const T_*)z, slots, w, (T_*)y, T, k, H);
  else
    combine_kernel<DT, 1><<<dim3((unsigned)blocks), dim3(256), 0, s>>>((const T_*)z, slots, w, (T_*)y, T, k, H);
  SQMP_LAUNCH_CHECK();
  return SQMP_OK;
}

// ---------------------------------------------------------------- pack rows
// out[i][p] = x[row(i)][amap[p]] (0 where amap[p] < 0), then the salient columns.  With offsets:
// output row i is slot i, row(i) = rows[i] / top_k (or i), and amap is the map of i's expert.
template <class T>
__global__ __launch_bounds__(256) void pack_rows_kernel(
    const T* __restrict__ x, long ldx, long R, const int32_t* __restrict__ amap, int Kp,
    const int32_t* __restrict__ salient, int S, int S_pad, const int32_t* __restrict__ rows,
    int top_k, const int32_t* __restrict__ offsets, int E, long map_stride, T* __restrict__ out) {
  const long i = blockIdx.x;
  long xr = i;
  if (offsets) {
    if (i >= offsets[E]) return;
    if (rows) xr = rows[i] / top_k;
    if (map_stride) {
      int lo = 0, hi = E - 1;  // the last expert with offsets[e] <= i
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (offsets[mid] <= i) lo = mid; else hi = mid - 1;
      }
      amap += (long)lo * map_stride;
    }
  }
  const int L = Kp + S_pad;
  for (int p = threadIdx.x; p < L; p += 256) {
    int k = -1;
    if (p < Kp) k = amap[p];
    else if (p - Kp < S) k = salient[p - Kp];
    out[i * L + p] = k >= 0 ? x[xr * ldx + k] : (T)0;
  }
}

}  // namespace route

extern "C" size_t sqmp_route_workspace_bytes(int T, int E) {
  if (T <= route::TB || E <= 0) return 0;  // one block: no workspace
  return ((size_t)cdiv(T, route::TB) + 1) * (size_t)E * sizeof(int32_t);
}

static int route_check(int T, int E, int k, const void* offsets, const void* rows,
                       const void* slots, const void* ids, const void* ws, size_t ws_bytes) {
  if (T < 0 || E <= 0 || k <= 0) return SQMP_EINVAL;
  if (E > route::E_MAX || k > route::K_MAX || (long)T * k > 0x7FFFFFFFL - 4096) return SQMP_EUNSUPPORTED;
  if (!offsets || (T > 0 && (!rows || !slots || !ids))) return SQMP_EINVAL;
  const size_t need = sqmp_route_workspace_bytes(T, E);
  if (need > 0 && (!ws || ws_bytes < need)) return SQMP_EWORKSPACE;
  return SQMP_OK;
}

__global__ void zero_offsets_kernel(int32_t* offsets, int n) {
  for (int i = threadIdx.x; i < n; i += 256) offsets[i] = 0;
}

extern "C" int sqmp_route(const void* logits, long ldl, int dtype, int T, int E, int top_k,
                          int normalize, float* weights, int32_t* ids, int32_t* offsets,
                          int32_t* rows, int32_t* slots, void* workspace, size_t ws_bytes,
                          void* stream) {
  SQMP_DEVICE_GUARD(stream);
  const int st = route_check(T, E, top_k, offsets, rows, slots, ids, workspace, ws_bytes);
  if (st != SQMP_OK) return st;
  if (top_k > E || ldl < E || (T > 0 && (!logits || !weights))) return SQMP_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  if (T == 0) {
    zero_offsets_kernel<<<dim3(1), dim3(256), 0, s>>>(offsets, E + 1);
    SQMP_LAUNCH_CHECK();
    return SQMP_OK;
  }
  const route::Args a{logits, ldl, T, E, top_k, normalize, weights, ids, offsets, rows, slots,
                      (int32_t*)workspace};
  switch (dtype) {
    case SQMP_F32: return route::by_k<F32>(a, s);
    case SQMP_F16: return route::by_k<F16>(a, s);
    case SQMP_BF16: return route::by_k<BF16>(a, s);
    default: return SQMP_EUNSUPPORTED;
  }
}

extern "C" int sqmp_plan_routes(const int32_t* ids, int T, int E, int top_k, int32_t* offsets,
                                int32_t* rows, int32_t* slots, void* workspace, size_t ws_bytes,
                                void* stream) {
  SQMP_DEVICE_GUARD(stream);
  const int st = route_check(T, E, top_k, offsets, rows, slots, ids, workspace, ws_bytes);
  if (st != SQMP_OK) return st;
  hipStream_t s = (hipStream_t)stream;
  if (T == 0) {
    zero_offsets_kernel<<<dim3(1), dim3(256), 0, s>>>(offsets, E + 1);
    SQMP_LAUNCH_CHECK();
    return SQMP_OK;
  }
  const route::Args a{nullptr, 0, T, E, top_k, 0, nullptr, const_cast<int32_t*>(ids), offsets,
                      rows, slots, (int32_t*)workspace};
  return route::launch<F32, 2>(a, s);
}

extern "C" int sqmp_combine(const void* z, int dtype, int T, int top_k, int H,
                            const int32_t* slots, const float* weights, void* y, void* stream) {
  SQMP_DEVICE_GUARD(stream);
  if (T < 0 || top_k <= 0 || H <= 0) return SQMP_EINVAL;
  if (T == 0) return SQMP_OK;
  if (!z || !slots || !weights || !y) return SQMP_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case SQMP_F32: return route::launch_combine<F32>(z, slots, weights, y, T, top_k, H, s);
    case SQMP_F16: return route::launch_combine<F16>(z, slots, weights, y, T, top_k, H, s);
    case SQMP_BF16: return route::launch_combine<BF16>(z, slots, weights, y, T, top_k, H, s);
    default: return SQMP_EUNSUPPORTED;
  }
}

extern "C" int sqmp_pack_rows(const void* x, long ldx, int dtype, int R, const int32_t* amap,
                              int Kp, const int32_t* salient, int S, int S_pad,
                              const int32_t* rows, int top_k, const int32_t* offsets, int E,
                              long map_stride, void* out, void* stream) {
  SQMP_DEVICE_GUARD(stream);
  if (R < 0 || Kp <= 0 || S < 0 || S_pad < S || ldx <= 0) return SQMP_EINVAL;
  if (R == 0) return SQMP_OK;
  if (!x || !amap || !out || (S > 0 && !salient)) return SQMP_EINVAL;
  if ((rows || map_stride) && !offsets) return SQMP_EINVAL;
  if (offsets && (E <= 0 || top_k <= 0)) return SQMP_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == SQMP_F32)
    route::pack_rows_kernel<uint32_t><<<dim3(R), dim3(256), 0, s>>>(
        (const uint32_t*)x, ldx, R, amap, Kp, salient, S, S_pad, rows, top_k, offsets, E, map_stride, (uint32_t*)out);
  else if (dtype == SQMP_F16 || dtype == SQMP_BF16)
    route::pack_rows_kernel<uint16_t><<<dim3(R), dim3(256), 0, s>>>(
        (const uint16_t*)x, ldx, R, amap, Kp, salient, S, S_pad, rows, top_k, offsets, E, map_stride, (uint16_t*)out);
  else
    return SQMP_EUNSUPPORTED;
  SQMP_LAUNCH_CHECK();
  return SQMP_OK;
}

}  // namespace sqmp
