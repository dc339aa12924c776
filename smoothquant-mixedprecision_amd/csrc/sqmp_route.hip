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
// What bounds it: launches and latency for a decoding batch (one launch up to 256 tokens), the
// logits' bytes for prompts.  A token's logits are spread over 4 lanes, read once in 16-byte
// pieces where they are aligned; each lane keeps its k largest in registers as keys that hold
// the value's order and the index (so every compare-exchange is a max and a min, and ties go to
// the lower index), and two merges over the lanes leave the k largest of all.  The order of the
// pairs is a counting sort: a block of 256 tokens ranks its pairs 64 at a time by ballots, an
// exclusive scan over the blocks places them: slots depend on the ids alone.
#include "sqmp_common.h"

namespace sqmp {
namespace route {

constexpr int TB = 256;          // tokens per block
constexpr int NT = 1024;         // threads per block: 4 lanes per token
constexpr int NWAVE = NT / 64;
constexpr int E_MAX = 256, K_MAX = 16;
constexpr int MAX_CHUNKS = TB * K_MAX / 64;       // 64-pair chunks of a block
constexpr int PER_WAVE = MAX_CHUNKS / NWAVE;      // of a wave
constexpr int PITCH = MAX_CHUNKS + 4;             // of an expert's chunk counts (8-byte rows)

// Keys whose unsigned order is the order of (value, lower index first): NaN highest, -0 as +0.
// 16-bit types: value and index in 32 bits; fp32: in 64.  (index 0xFFFF / ~0: none)
template <class DT> struct Key;
template <> struct Key<F32> {
  typedef uint64_t K;
  static constexpr K NEG_INF = (K)0x007FFFFFu << 32;  // of -inf, below every index
  __device__ static inline K make(float v, int e) {
    uint32_t u = __float_as_uint(v);
    if (v != v) u = 0x7FFFFFFFu;
    if (u == 0x80000000u) u = 0u;
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((K)u << 32) | (uint32_t)~e;
  }
  __device__ static inline int index(K k) { return (int)~(uint32_t)k; }
  __device__ static inline bool chosen(K k) { return (k >> 32) > 0x007FFFFFu; }
  __device__ static inline float value(K k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
  }
  __device__ static inline K shfl(K k, int x) {
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)k, x, 64);
    const uint32_t hi = (uint32_t)__shfl_xor((int)(uint32_t)(k >> 32), x, 64);
    return ((K)hi << 32) | lo;
  }
};
template <class DT, uint32_t INF> struct Key16 {
  typedef uint32_t K;
  typedef typename DT::T T;
  static constexpr K NEG_INF = (K)(0x7FFFu - INF) << 16;  // ~(0x8000 | INF)
  __device__ static inline K make(T v, int e) {
    uint32_t u = (uint32_t)__builtin_bit_cast(uint16_t, v);
    if ((u & 0x7FFFu) > INF) u = 0x7FFFu;
    if (u == 0x8000u) u = 0u;
    u = (u & 0x8000u) ? (~u & 0xFFFFu) : (u | 0x8000u);
    return (u << 16) | (uint32_t)(0xFFFF - e);
  }
  __device__ static inline int index(K k) { return 0xFFFF - (int)(k & 0xFFFFu); }
  __device__ static inline bool chosen(K k) { return (k >> 16) > (NEG_INF >> 16); }
  __device__ static inline float value(K k) {
    const uint32_t u = k >> 16;
    const uint16_t b = (uint16_t)((u & 0x8000u) ? (u & 0x7FFFu) : ~u);
    return DT::to_f(__builtin_bit_cast(T, b));
  }
  __device__ static inline K shfl(K k, int x) { return (K)__shfl_xor((int)k, x, 64); }
};
template <> struct Key<F16> : Key16<F16, 0x7C00u> {};
template <> struct Key<BF16> : Key16<BF16, 0x7F80u> {};

// list (descending) <- the KT largest of list and c
template <class K, int KT>
__device__ inline void insert(K (&list)[KT], K c) {
#pragma unroll
  for (int j = 0; j < KT; ++j) {
    const K a = list[j];
    list[j] = c > a ? c : a;
    c = c > a ? a : c;
  }
}

// list <- the KT largest of the lanes lane and lane ^ x: the larger of a[j] and b[KT - 1 - j] are
// those, in bitonic order; sorted by log2(KT) rounds of exchanges
template <class DT, int KT>
__device__ inline void merge(typename Key<DT>::K (&list)[KT], int x) {
  typedef typename Key<DT>::K K;
  K o[KT];
#pragma unroll
  for (int j = 0; j < KT; ++j) o[j] = Key<DT>::shfl(list[j], x);
#pragma unroll
  for (int j = 0; j < KT; ++j) list[j] = list[j] > o[KT - 1 - j] ? list[j] : o[KT - 1 - j];
#pragma unroll
  for (int d = KT / 2; d >= 1; d >>= 1)
#pragma unroll
    for (int j = 0; j < KT; ++j)
      if ((j & d) == 0) {
        const K a = list[j], b = list[j + d];
        list[j] = a > b ? a : b;
        list[j + d] = a > b ? b : a;
      }
}

struct Args {
  const void* logits;  // NULL: ids are given
  long ldl;
  int T, E, k, normalize;
  float* weights;
  int32_t* ids;
  int32_t *offsets, *rows, *slots;
  int32_t* hist;       // [blocks][E], then [E] totals
  int blocks;
};

// lane c of a token's four visits its share of the logits: f(value, index)
template <class DT, class F>
__device__ inline void each_logit(const typename DT::T* row, int E, int c, bool vec, F f) {
  typedef typename DT::T T;
  constexpr int V = 16 / sizeof(T);
  if (vec) {  // whole 16-byte pieces, piece p to lane p % 4
    for (int p = c; p * V < E; p += 4) {
      struct __attribute__((aligned(16))) P { T v[V]; };
      const P x = *(const P*)(row + p * V);
#pragma unroll
      for (int i = 0; i < V; ++i) f(x.v[i], p * V + i);
    }
  } else {
    for (int e = c; e < E; e += 4) f(row[e], e);
  }
}

// ids (and weights) of the block's tokens; lid: the ids again, in LDS
template <class DT, int KT>
__device__ inline void choose(const Args& a, int t0, int nt, uint16_t* lid) {
  typedef typename DT::T T;
  typedef Key<DT> KY;
  typedef typename KY::K K;
  const int tok = threadIdx.x >> 2, c = threadIdx.x & 3;
  const int t = t0 + min(tok, nt - 1);  // (idle lanes repeat the last token)
  const T* row = (const T*)a.logits + t * a.ldl;
  constexpr int V = 16 / sizeof(T);
  const bool vec = a.E % V == 0 && a.ldl % V == 0 && (size_t)a.logits % 16 == 0;
  K list[KT];
#pragma unroll
  for (int j = 0; j < KT; ++j) list[j] = 0;
  each_logit<DT>(row, a.E, c, vec, [&](T v, int e) { insert<K, KT>(list, KY::make(v, e)); });
  merge<DT, KT>(list, 1);
  merge<DT, KT>(list, 2);
  // lane c finishes the choices j = c, c + 4, ...
  constexpr int PER = (KT + 3) / 4;
  const float top = KY::value(list[0]);
  K own[PER];
  float ex[PER], den = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    own[i] = list[4 * i];
#pragma unroll
    for (int x = 1; x < 4; ++x)
      if (4 * i + x < KT && c == x) own[i] = list[4 * i + x];
    const bool sel = 4 * i + c < a.k && 4 * i + c < KT && KY::chosen(own[i]);
    ex[i] = sel ? expf(KY::value(own[i]) - top) : 0.f;
    den += ex[i];
  }
  if (!a.normalize) {
    // (exp2 of a rounded product: the difference d, log2 e and the product are off by half a step each at
    // most, a term exp(d) so by 1.5 |d| steps of itself and the sum by 1.5 times the weighted mean of
    // |d|, which is 3.3 at most for 256 logits (255 of them 4.3 below the first): 5 steps, 6e-7)
    den = 0.f;
    each_logit<DT>(row, a.E, c, vec, [&](T v, int) {
      den += __builtin_amdgcn_exp2f((DT::to_f(v) - top) * 1.44269504f);
    });
  }
  den += __shfl_xor(den, 1, 64);
  den += __shfl_xor(den, 2, 64);
  if (tok < nt) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = 4 * i + c;
      if (j < a.k) {
        const bool sel = KY::chosen(own[i]);
        const int id = sel ? KY::index(own[i]) : -1;
        const long f = (long)t * a.k + j;
        a.weights[f] = sel ? ex[i] / den : 0.f;
        a.ids[f] = id;
        lid[tok * a.k + j] = (uint16_t)(sel ? id : a.E);
      }
    }
  }
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

// exclusive prefix over the E experts of v (thread e); *total: their sum.  tmp: LDS [E_MAX]
__device__ inline int scan_experts(int v, int32_t* tmp, int* total) {
  const int e = threadIdx.x;
  if (e < E_MAX) tmp[e] = v;
  __syncthreads();
  for (int d = 1; d < E_MAX; d <<= 1) {
    const int add = e >= d && e < E_MAX ? tmp[e - d] : 0;
    __syncthreads();
    if (e < E_MAX) tmp[e] += add;
    __syncthreads();
  }
  *total = tmp[E_MAX - 1];
  return e < E_MAX ? tmp[e] - v : 0;
}

// one block of tokens: its ids, and the rank of each of its pairs among the block's pairs of the
// same expert.  ONE (the only block): the slots themselves; else the ranks, left in slots
template <class DT, int KT, bool ONE>
__global__ __launch_bounds__(NT) void route_kernel(const Args a) {
  __shared__ __attribute__((aligned(8))) uint16_t cnt[PITCH * E_MAX];  // [expert][chunk]
  __shared__ uint16_t lid[TB * K_MAX];
  __shared__ int32_t tmp[E_MAX], start[E_MAX];
  const int t0 = blockIdx.x * TB, nt = min(TB, a.T - t0);
  const int np = nt * a.k, chunks = (np + 63) / 64;
  const long f0 = (long)t0 * a.k;
  if (a.logits) {
    choose<DT, KT>(a, t0, nt, lid);
  } else {
    for (int i = threadIdx.x; i < np; i += NT) {
      const int e = a.ids[f0 + i];
      lid[i] = (uint16_t)(e < 0 || e >= a.E ? a.E : e);
    }
  }
  const int quads = (chunks + 3) / 4;
  for (int i = threadIdx.x; i < quads * a.E; i += NT)
    *(uint64_t*)(cnt + (i / quads) * PITCH + (i % quads) * 4) = 0;
  __syncthreads();
  // pairs of each expert in every chunk, and a pair's rank inside its chunk
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int nbits = 32 - __clz(a.E);  // values 0 .. E
  int my_e[PER_WAVE], my_r[PER_WAVE];
#pragma unroll
  for (int i = 0; i < PER_WAVE; ++i) {
    const int c = wave + i * NWAVE, f = c * 64 + lane;
    my_e[i] = a.E, my_r[i] = 0;
    if (c < chunks) {
      my_e[i] = f < np ? lid[f] : a.E;
      const uint64_t m = same_expert(my_e[i], nbits);
      my_r[i] = (int)__popcll(m & ((1ull << lane) - 1));
      if (my_e[i] < a.E && my_r[i] == 0) cnt[my_e[i] * PITCH + c] = (uint16_t)__popcll(m);
    }
  }
  __syncthreads();
  // cnt -> pairs of the expert in earlier chunks, four chunks at a time; the block's count
  int s = 0;
  if ((int)threadIdx.x < a.E) {
    uint64_t* row = (uint64_t*)(cnt + threadIdx.x * PITCH);
    for (int c = 0; c < quads; ++c) {
      const uint64_t v = row[c];
      uint64_t o = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o |= (uint64_t)(uint16_t)s << (16 * i);
        s += (int)((v >> (16 * i)) & 0xFFFFu);
      }
      row[c] = o;
    }
  }
  int total = 0;
  if constexpr (ONE) {
    const int at = scan_experts(s, tmp, &total);
    if ((int)threadIdx.x < a.E) start[threadIdx.x] = at, a.offsets[threadIdx.x] = at;
    if (threadIdx.x == 0) a.offsets[a.E] = total;
  } else {
    if ((int)threadIdx.x < a.E) a.hist[(long)blockIdx.x * a.E + threadIdx.x] = s;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER_WAVE; ++i) {
    const int c = wave + i * NWAVE, f = c * 64 + lane, e = my_e[i];
    if (c < chunks && f < np) {
      int slot = e < a.E ? cnt[e * PITCH + c] + my_r[i] : -1;
      if constexpr (ONE) {
        if (e < a.E) {
          slot += start[e];
          a.rows[slot] = f;
        }
        if (f >= total) a.rows[f] = -1;  // behind the last pair
      }
      a.slots[f0 + f] = slot;
    }
  }
}

// hist[blk][e] -> exclusive scan over the blocks, the expert's total behind
__global__ __launch_bounds__(256) void scan_kernel(int32_t* hist, int blocks, int E) {
  __shared__ int32_t part[256];
  const int e = blockIdx.x, tid = threadIdx.x;
  int32_t* h = hist + e;
  int run = 0;
  for (int b0 = 0; b0 < blocks; b0 += 256) {
    const int v = b0 + tid < blocks ? h[(long)(b0 + tid) * E] : 0;
    part[tid] = v;
    __syncthreads();
    for (int d = 1; d < 256; d <<= 1) {
      const int add = tid >= d ? part[tid - d] : 0;
      __syncthreads();
      part[tid] += add;
      __syncthreads();
    }
    if (b0 + tid < blocks) h[(long)(b0 + tid) * E] = run + part[tid] - v;
    run += part[255];
    __syncthreads();
  }
  if (tid == 0) hist[(long)E * blocks + e] = run;
}

// ranks in slots -> slots, and rows.  SCANNED: hist holds the scan of scan_kernel; else (few
// blocks) every block adds up the counts of the blocks before it by itself
constexpr int SELF_SCAN_BLOCKS = 512;
template <bool SCANNED>
__global__ __launch_bounds__(NT) void place_kernel(const Args a) {
  __shared__ int32_t tmp[E_MAX], start[E_MAX], count[E_MAX];
  const int e = threadIdx.x;
  if constexpr (!SCANNED) {
    // thread (group c, expert ex): every groups-th block, 8 loads in flight; summed in LDS
    const int groups = NT / a.E, ex = e % a.E, c = e / a.E;
    if (e < a.E) count[e] = start[e] = 0;
    __syncthreads();
    int before = 0, all = 0;
    if (c < groups) {
      for (int b0 = c; b0 < a.blocks; b0 += 8 * groups) {
        int v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int b = b0 + i * groups;
          v[i] = b < a.blocks ? a.hist[(long)b * a.E + ex] : 0;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          all += v[i];
          before += b0 + i * groups < (int)blockIdx.x ? v[i] : 0;
        }
      }
      atomicAdd(&count[ex], all);   // (LDS; whole numbers: the order does not matter)
      atomicAdd(&start[ex], before);
    }
    __syncthreads();
  } else if (e < a.E) {
    count[e] = a.hist[(long)a.E * a.blocks + e];
    start[e] = a.hist[(long)blockIdx.x * a.E + e];
  }
  int total = 0;
  const int at = scan_experts(e < a.E ? count[e] : 0, tmp, &total);
  if (e < a.E) {
    start[e] += at;
    if (blockIdx.x == 0) a.offsets[e] = at;
  }
  if (blockIdx.x == 0 && e == 0) a.offsets[a.E] = total;
  __syncthreads();
  const int t0 = blockIdx.x * TB, np = min(TB, a.T - t0) * a.k;
  const long f0 = (long)t0 * a.k;
  for (int i = threadIdx.x; i < np; i += NT) {
    const long f = f0 + i;
    const int r = a.slots[f];
    if (r >= 0) {
      const int slot = start[a.ids[f]] + r;
      a.slots[f] = slot;
      a.rows[slot] = (int32_t)f;
    }
    if (f >= total) a.rows[f] = -1;  // behind the last pair
  }
}

template <class DT, int KT>
static int launch(const Args& a, hipStream_t s) {
  if (a.blocks == 1) {
    route_kernel<DT, KT, true><<<dim3(1), dim3(NT), 0, s>>>(a);
    SQMP_LAUNCH_CHECK();
    return SQMP_OK;
  }
  route_kernel<DT, KT, false><<<dim3(a.blocks), dim3(NT), 0, s>>>(a);
  SQMP_LAUNCH_CHECK();
  if (a.blocks <= SELF_SCAN_BLOCKS) {
    place_kernel<false><<<dim3(a.blocks), dim3(NT), 0, s>>>(a);
    SQMP_LAUNCH_CHECK();
    return SQMP_OK;
  }
  scan_kernel<<<dim3(a.E), dim3(256), 0, s>>>(a.hist, a.blocks, a.E);
  SQMP_LAUNCH_CHECK();
  place_kernel<true><<<dim3(a.blocks), dim3(NT), 0, s>>>(a);
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
// A thread holds 16 bytes of one token's output and adds its k rows in the order of j.  What bounds
// it: bytes, each read and written once; 16384 x 6 x 2048 bf16 97 us (4.86 TB/s).
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
                      (int32_t*)workspace, cdiv(T, route::TB)};
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
                      rows, slots, (int32_t*)workspace, cdiv(T, route::TB)};
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
