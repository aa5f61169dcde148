// Routing of tokens to experts and the weighted sum back: the plan of a
// mixture-of-experts layer whose products run in grouped.cu (int8 weights)
// and matvec.cu (4-bit weights).
//
//   route    logits [T, E] -> the k best experts of every token and their
//            weights, and the (token, slot) pairs sorted by expert;
//   combine  out[t] = sum_j weight[t, j] * y[pos[t, j]] (+ residual[t]).
#include <atomic>
#include <cmath>

#include "../../include/qlinear_b200.h"
#include "common.cuh"
#include "internal.h"

namespace qlin {
namespace {

constexpr int ROUTE_THREADS = 512;
constexpr int ROUTE_WARPS = ROUTE_THREADS / 32;
constexpr int ROUTE_BLOCKS = 148;      // at most, one a SM: the second kernel's blocks read all blocks' counts
constexpr int SORT_BATCH = 8;          // tokens whose choices a warp holds at a time
constexpr float NEG_INF = -INFINITY;

struct RouteParams {
  const void* logits;
  int64_t ld;
  int64_t T;
  int E, Ep, k;       // Ep: E rounded up to 4, the stride of a block's counts
  int sigmoid, renorm;
  int64_t tokens;     // of a block, a multiple of ROUTE_WARPS
  int blocks;
  int32_t* ids;       // [T, k]
  float* weights;     // [T, k]
  int32_t* offsets;   // [E + 1]
  int32_t* rows;      // [T * k]
  int32_t* pos;       // [T, k]
  int32_t* counts;    // [blocks, Ep] rows of each expert in each block
};

// A logit and its expert as one unsigned number: larger for larger logits (-0
// as +0, NaN as -inf), for equal ones larger for lower experts; 0 is below all.
// 16-bit logits leave room for the expert in 32 bits.
template <int DT> struct RouteKey {
  using T = uint64_t;
  static __device__ __forceinline__ T make(float v, int e) {
    const uint32_t b = __float_as_uint(v != v ? NEG_INF : v + 0.0f);
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xFFFFu - (uint32_t)e);
  }
  static __device__ __forceinline__ float value(T k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
  }
  static __device__ __forceinline__ int expert(T k) { return (int)(0xFFFFu - ((uint32_t)k & 0xFFFFu)); }
};
template <int DT> struct RouteKey16 {
  using T = uint32_t;
  static __device__ __forceinline__ T make(float v, int e) {
    const auto h = Elem<DT>::from_f(v != v ? NEG_INF : v + 0.0f);  // exact: v has this type
    const uint32_t b = *reinterpret_cast<const uint16_t*>(&h);
    return (b & 0x8000u ? ~b & 0xFFFFu : b | 0x8000u) << 16 | (0xFFFFu - (uint32_t)e);
  }
  static __device__ __forceinline__ float value(T k) {
    const uint32_t u = k >> 16;
    const uint16_t b = (uint16_t)(u & 0x8000u ? u & 0x7FFFu : ~u);
    return Elem<DT>::to_f(*reinterpret_cast<const typename Elem<DT>::T*>(&b));
  }
  static __device__ __forceinline__ int expert(T k) { return (int)(0xFFFFu - (k & 0xFFFFu)); }
};
template <> struct RouteKey<DT_BF16> : RouteKey16<DT_BF16> {};
template <> struct RouteKey<DT_F16> : RouteKey16<DT_F16> {};

// log(1 / (1 + exp(-v))) without overflow on either side
__device__ __forceinline__ float log_sigmoid(float v) { return fminf(v, 0.0f) - log1pf(expf(-fabsf(v))); }

// The choices of SORT_BATCH tokens, slot j in lane j; -1 behind the last.
__device__ __forceinline__ void load_choices(const RouteParams& p, int64_t t0, int64_t t1, int lane,
                                             int (&id)[SORT_BATCH]) {
#pragma unroll
  for (int u = 0; u < SORT_BATCH; ++u) id[u] = lane < p.k && t0 + u < t1 ? p.ids[(t0 + u) * p.k + lane] : -1;
}

// Rows of each expert among one warp's tokens, to cnt [E] (zeros on entry).
__device__ __forceinline__ void count_choices(const RouteParams& p, int64_t t0, int64_t t1, int lane, int32_t* cnt) {
  for (int64_t tb = t0; tb < t1; tb += SORT_BATCH) {
    int id[SORT_BATCH];
    load_choices(p, tb, t1, lane, id);
#pragma unroll
    for (int u = 0; u < SORT_BATCH; ++u) {
      if (id[u] >= 0) cnt[id[u]] += 1;  // a token's experts differ: no two lanes meet
      __syncwarp();
    }
  }
}

// Sorted place of every pair of this block's tokens.  A token chooses an
// expert at most once, so the place of a pair within its expert is the number
// of earlier tokens with that expert: run[w][e] starts at the first place of
// warp w's tokens and goes up by one for each of them.
//   s_cnt [warps][Ep]  rows of each expert in each warp's tokens (in), running places (out)
//   s_base [Ep]        first place of this block's rows of each expert
__device__ void assign_places(const RouteParams& p, int32_t* s_cnt, const int32_t* s_base, int64_t t0, int64_t t1,
                              int warp, int lane) {
  for (int e = threadIdx.x; e < p.E; e += ROUTE_THREADS) {
    int at = s_base[e];
#pragma unroll
    for (int w = 0; w < ROUTE_WARPS; ++w) {
      const int c = s_cnt[w * p.Ep + e];
      s_cnt[w * p.Ep + e] = at;
      at += c;
    }
  }
  __syncthreads();
  int32_t* run = s_cnt + warp * p.Ep;
  for (int64_t tb = t0; tb < t1; tb += SORT_BATCH) {
    int id[SORT_BATCH];
    load_choices(p, tb, t1, lane, id);
#pragma unroll
    for (int u = 0; u < SORT_BATCH; ++u) {
      int at = -1;
      if (id[u] >= 0) {
        at = run[id[u]];
        run[id[u]] = at + 1;
        p.rows[at] = (int32_t)(tb + u);
      }
      if (lane < p.k && tb + u < t1) p.pos[(tb + u) * p.k + lane] = at;
      __syncwarp();
    }
  }
}

// Exclusive sums of s_tot[0..E) into s_base and, from one block, into
// offsets [E + 1]; warp 0 works, all threads meet.
__device__ int scan_experts(const RouteParams& p, const int32_t* s_tot, int32_t* s_base, int32_t* s_total, bool write) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int carry = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      const int v = e < p.E ? s_tot[e] : 0;
      int inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      if (e < p.E) {
        s_base[e] = carry + inc - v;
        if (write) p.offsets[e] = carry + inc - v;
      }
      carry += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) {
      *s_total = carry;
      if (write) p.offsets[p.E] = carry;
    }
  }
  __syncthreads();
  return *s_total;
}

// L lanes a token, PER logits a lane (expert sub + L * i), 32 / L tokens a warp
// at a time.  k rounds find the largest key below the round's before: PER
// compares a lane and log2(L) exchanges, for all the warp's tokens at once.
// (A warp a token with two redux.sync a round took 25 us for 16384 tokens, 128
// experts and k 8: that instruction issues every 16 clocks or so.)
template <int DT, int PER, int L>
__global__ void __launch_bounds__(ROUTE_THREADS) route_topk_kernel(RouteParams p) {
  using Key = RouteKey<DT>;
  using KT = typename Key::T;
  constexpr int TOK = 32 / L;
  extern __shared__ int32_t s_route[];
  int32_t* s_cnt = s_route;                       // [warps][Ep]
  int32_t* s_tot = s_cnt + ROUTE_WARPS * p.Ep;    // [Ep]
  int32_t* s_base = s_tot + p.Ep;                 // [Ep]
  KT* s_win = reinterpret_cast<KT*>(s_base + p.Ep);  // [warps][TOK][32]: the chosen keys
  __shared__ int32_t s_total;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & (L - 1);
  for (int i = threadIdx.x; i < (ROUTE_WARPS + 1) * p.Ep; i += ROUTE_THREADS) s_cnt[i] = 0;
  __syncthreads();
  pdl_wait();
  const int64_t per_warp = p.tokens / ROUTE_WARPS;
  const int64_t t0 = min((int64_t)blockIdx.x * p.tokens + warp * per_warp, p.T);
  const int64_t t1 = min(t0 + per_warp, p.T);
  const typename Elem<DT>::T* x = reinterpret_cast<const typename Elem<DT>::T*>(p.logits);
  const KT none = Key::make(NEG_INF, 0) | 0xFFFFu;  // no key of -inf is above
  KT* win = s_win + (warp * TOK + lane / L) * 32;
  for (int64_t tb = t0; tb < t1; tb += TOK) {
    const int64_t t = tb + lane / L;
    const bool in = t < t1;
    float v[PER];
    KT key[PER];
    bool nan = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = sub + L * i;
      v[i] = in && e < p.E ? Elem<DT>::to_f(x[t * p.ld + e]) : NEG_INF;
      nan |= v[i] != v[i];
      key[i] = Key::make(v[i], e);
    }
    KT last = ~(KT)0;
    for (int j = 0; j < p.k; ++j) {
      KT best = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const KT c = key[i] < last ? key[i] : 0;
        best = c > best ? c : best;
      }
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) {
        const KT c = __shfl_xor_sync(0xffffffffu, best, o);
        best = c > best ? c : best;
      }
      last = best;
      if (sub == 0) win[j] = best;
    }
    __syncwarp();
    nan = __any_sync(0xffffffffu >> (32 - L) << (lane & ~(L - 1)), nan);
    // weights: e / sum; slots sub, sub + L, ... in this lane
    const bool any = win[0] > none;
    const float first = Key::value(win[0]);
    const float top = p.sigmoid ? log_sigmoid(first) : first;
    float sum = 0.0f;
    if (!p.sigmoid && !p.renorm) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (sub + L * i < p.E) sum += expf(v[i] - top);
    } else if (p.renorm) {
      // s_j / sum s = softmax of the chosen log-sigmoids: no 0 / 0 far below zero
      for (int j = sub; j < p.k; j += L)
        if (win[j] > none) sum += expf((p.sigmoid ? log_sigmoid(Key::value(win[j])) : Key::value(win[j])) - top);
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (in) {
      for (int j = sub; j < p.k; j += L) {
        const KT c = win[j];
        const bool chosen = any && c > none;
        const float y = Key::value(c);
        float w = 1.0f / (1.0f + expf(-y));
        if (!p.sigmoid || p.renorm) w = expf((p.sigmoid ? log_sigmoid(y) : y) - top) / sum;
        if (nan && !p.sigmoid) w = NAN;
        p.ids[t * p.k + j] = chosen ? Key::expert(c) : -1;
        p.weights[t * p.k + j] = chosen ? w : 0.0f;
        if (chosen) atomicAdd(&s_tot[Key::expert(c)], 1);
      }
    }
    __syncwarp();
  }
  __syncthreads();
  pdl_launch_dependents();
  if (p.blocks > 1) {
    for (int e = threadIdx.x; e < p.Ep; e += ROUTE_THREADS) p.counts[(int64_t)blockIdx.x * p.Ep + e] = s_tot[e];
    return;
  }
  // one block holds all tokens: it sorts them too
  const int total = scan_experts(p, s_tot, s_base, &s_total, true);
  count_choices(p, t0, t1, lane, s_cnt + warp * p.Ep);
  __syncthreads();
  assign_places(p, s_cnt, s_base, t0, t1, warp, lane);
  for (int64_t i = total + threadIdx.x; i < p.T * p.k; i += ROUTE_THREADS) p.rows[i] = -1;
}

// Places of the pairs when the tokens lie in several blocks: every block adds
// up the counts of all blocks (its own first place of each expert is the sum
// over the blocks before it) and gives out its tokens' places.
__global__ void __launch_bounds__(ROUTE_THREADS) route_sort_kernel(RouteParams p) {
  extern __shared__ int32_t s_route[];
  int32_t* s_cnt = s_route;                     // [warps][Ep]
  int32_t* s_tot = s_cnt + ROUTE_WARPS * p.Ep;  // [Ep]
  int32_t* s_base = s_tot + p.Ep;               // [Ep]
  int32_t* s_pre = s_base + p.Ep;               // [Ep]
  __shared__ int32_t s_total;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < (ROUTE_WARPS + 3) * p.Ep; i += ROUTE_THREADS) s_route[i] = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const int64_t per_warp = p.tokens / ROUTE_WARPS;
  const int64_t t0 = min((int64_t)blockIdx.x * p.tokens + warp * per_warp, p.T);
  const int64_t t1 = min(t0 + per_warp, p.T);
  count_choices(p, t0, t1, lane, s_cnt + warp * p.Ep);
  int cols = 1;
  while (cols < p.Ep / 4) cols <<= 1;  // <= 128 for E <= 512
  const int col = threadIdx.x & (cols - 1), slices = ROUTE_THREADS / cols;
  if (col < p.Ep / 4) {
    int4 pre = make_int4(0, 0, 0, 0), tot = make_int4(0, 0, 0, 0);
#pragma unroll 8
    for (int b = threadIdx.x / cols; b < p.blocks; b += slices) {
      const int4 c = reinterpret_cast<const int4*>(p.counts + (int64_t)b * p.Ep)[col];
      tot.x += c.x; tot.y += c.y; tot.z += c.z; tot.w += c.w;
      if (b < (int)blockIdx.x) { pre.x += c.x; pre.y += c.y; pre.z += c.z; pre.w += c.w; }
    }
    atomicAdd(&s_tot[4 * col], tot.x); atomicAdd(&s_tot[4 * col + 1], tot.y);
    atomicAdd(&s_tot[4 * col + 2], tot.z); atomicAdd(&s_tot[4 * col + 3], tot.w);
    atomicAdd(&s_pre[4 * col], pre.x); atomicAdd(&s_pre[4 * col + 1], pre.y);
    atomicAdd(&s_pre[4 * col + 2], pre.z); atomicAdd(&s_pre[4 * col + 3], pre.w);
  }
  __syncthreads();
  const int total = scan_experts(p, s_tot, s_base, &s_total, blockIdx.x == 0);
  for (int e = threadIdx.x; e < p.E; e += ROUTE_THREADS) s_base[e] += s_pre[e];
  __syncthreads();
  assign_places(p, s_cnt, s_base, t0, t1, warp, lane);
  for (int64_t i = total + (int64_t)blockIdx.x * ROUTE_THREADS + threadIdx.x; i < p.T * p.k;
       i += (int64_t)gridDim.x * ROUTE_THREADS)
    p.rows[i] = -1;
}

void route_plan(int64_t T, int64_t& tokens, int64_t& blocks) {
  tokens = (T + ROUTE_BLOCKS - 1) / ROUTE_BLOCKS;
  tokens = (tokens + ROUTE_WARPS - 1) / ROUTE_WARPS * ROUTE_WARPS;
  if (tokens == 0) tokens = ROUTE_WARPS;  // (T = 0: no blocks)
  blocks = (T + tokens - 1) / tokens;
}

template <int DT, int PER, int L>
int launch_topk_cfg(const RouteParams& p, cudaStream_t s) {
  const size_t smem = (size_t)(ROUTE_WARPS + 2) * p.Ep * sizeof(int32_t) +
                      (size_t)ROUTE_WARPS * (32 / L) * 32 * sizeof(typename RouteKey<DT>::T);
  auto kern = route_topk_kernel<DT, PER, L>;
  static std::atomic<uint64_t> attr_devices{0};  // shared-memory limit raised once per device
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  cudaError_t e;
  if (!(attr_devices.load() & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(route)");
    attr_devices.fetch_or(bit);
  }
  e = launch_pdl(kern, dim3((unsigned)p.blocks), dim3(ROUTE_THREADS), smem, s, p);
  return e == cudaSuccess ? QLIN_OK : cuda_fail(e, "route launch");
}
template <int DT>
int launch_topk(const RouteParams& p, cudaStream_t s) {
  if (p.E <= 32) return launch_topk_cfg<DT, 4, 8>(p, s);
  if (p.E <= 64) return launch_topk_cfg<DT, 8, 8>(p, s);
  if (p.E <= 128) return launch_topk_cfg<DT, 16, 8>(p, s);
  if (p.E <= 256) return launch_topk_cfg<DT, 16, 16>(p, s);
  return launch_topk_cfg<DT, 16, 32>(p, s);
}

// ---------------------------------------------------------------------------
// combine
// ---------------------------------------------------------------------------

struct CombineParams {
  const void* y;
  int64_t R, N, ldy;
  const float* weights;
  const int32_t* pos;
  int64_t T;
  int k;
  const void* residual;  // [T, ld_res] or null
  int64_t ld_res;
  void* out;             // [T, N]
  int64_t chunks;        // blocks a token
};

constexpr int COMBINE_THREADS = 128;

// One thread per CH chunks of VEC columns of a token, COMBINE_THREADS chunks
// apart: a float32 sum in slot order, rounded once.  HBM bound: every row of y
// that a token chose is read once; BATCH of them are on their way at a time.
template <int DT, int VEC, int CH, int BATCH>
__global__ void __launch_bounds__(COMBINE_THREADS) combine_kernel(CombineParams p) {
  using T = typename Elem<DT>::T;
  union alignas(sizeof(T) * VEC) Chunk {
    uint4 whole;  // VEC > 1: 16 bytes, moved at once
    T v[VEC];
    __device__ Chunk() {}
    __device__ void load(const void* from) {
      if constexpr (VEC == 1) v[0] = *static_cast<const T*>(from);
      else whole = __ldcs(static_cast<const uint4*>(from));  // read once
    }
    __device__ void store(void* to) const {
      if constexpr (VEC == 1) *static_cast<T*>(to) = v[0];
      else *static_cast<uint4*>(to) = whole;
    }
  };
  pdl_wait();
  pdl_launch_dependents();
  const int64_t t = blockIdx.x / p.chunks;
  const int64_t col0 = (blockIdx.x % p.chunks) * (COMBINE_THREADS * CH * VEC) + threadIdx.x * VEC;
  const auto column = [&](int c) { return col0 + c * (COMBINE_THREADS * VEC); };
  Chunk res[CH];
  if (p.residual != nullptr) {  // on its way while the rows are added up
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (column(c) < p.N)
        res[c].load(reinterpret_cast<const T*>(p.residual) + t * p.ld_res + column(c));
  }
  float acc[CH][VEC];
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[c][i] = 0.0f;
  for (int j0 = 0; j0 < p.k; j0 += BATCH) {
    int at[BATCH];
    float w[BATCH];
    Chunk v[BATCH][CH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      at[u] = j0 + u < p.k ? __ldg(p.pos + t * p.k + j0 + u) : -1;
      w[u] = j0 + u < p.k ? __ldg(p.weights + t * p.k + j0 + u) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (at[u] >= 0 && at[u] < p.R) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
          if (column(c) < p.N)
            v[u][c].load(reinterpret_cast<const T*>(p.y) + at[u] * p.ldy + column(c));
      }
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (at[u] >= 0 && at[u] < p.R) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
          if (column(c) < p.N)
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[c][i] = __fmaf_rn(w[u], Elem<DT>::to_f(v[u][c].v[i]), acc[c][i]);
      }
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if (column(c) >= p.N) continue;
    Chunk o;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      o.v[i] = Elem<DT>::from_f(p.residual != nullptr ? acc[c][i] + Elem<DT>::to_f(res[c].v[i]) : acc[c][i]);
    o.store(reinterpret_cast<T*>(p.out) + t * p.N + column(c));
  }
}

template <int DT, int VEC, int CH, int BATCH>
int launch_combine_cfg(CombineParams p, cudaStream_t s) {
  constexpr int64_t per = COMBINE_THREADS * CH * VEC;
  p.chunks = (p.N + per - 1) / per;
  if (p.chunks * p.T > INT32_MAX) return fail(QLIN_ERR_UNSUPPORTED, "combine: too many tokens");
  const cudaError_t e =
      launch_pdl(combine_kernel<DT, VEC, CH, BATCH>, dim3((unsigned)(p.chunks * p.T)), dim3(COMBINE_THREADS), 0, s, p);
  return e == cudaSuccess ? QLIN_OK : cuda_fail(e, "combine launch");
}
template <int DT>
int launch_combine_dt(const CombineParams& p, bool vec, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(typename Elem<DT>::T);
  if (!vec) return launch_combine_cfg<DT, 1, 8, 4>(p, s);
  // Few rows a token: two chunks a thread, else its loads are too few (4096
  // tokens of 4096 bf16, k 2 and a residual: 20.6 us, 6.5 TB/s; with one chunk
  // 27.8).  With more rows a token one chunk has enough (k 8: 50.6 us, with two
  // 56).
  if (p.k <= 2) return launch_combine_cfg<DT, VEC, 2, 2>(p, s);
  return launch_combine_cfg<DT, VEC, 1, 4>(p, s);
}

}  // namespace

size_t route_workspace_bytes(int64_t T, int64_t E) {
  int64_t tokens, blocks;
  route_plan(T, tokens, blocks);
  return blocks > 1 ? (size_t)blocks * ((E + 3) / 4 * 4) * sizeof(int32_t) : 0;
}

int launch_route(int dt, const void* logits, int64_t ld, int64_t T, int64_t E, int top_k, int sigmoid, int renorm,
                 int32_t* ids, float* weights, int32_t* offsets, int32_t* rows, int32_t* pos, void* workspace,
                 cudaStream_t stream) {
  RouteParams p{};
  p.logits = logits;
  p.ld = ld;
  p.T = T;
  p.E = (int)E;
  p.Ep = (int)((E + 3) / 4 * 4);
  p.k = top_k;
  p.sigmoid = sigmoid;
  p.renorm = renorm;
  int64_t blocks;
  route_plan(T, p.tokens, blocks);
  p.blocks = (int)blocks;
  p.ids = ids;
  p.weights = weights;
  p.offsets = offsets;
  p.rows = rows;
  p.pos = pos;
  p.counts = static_cast<int32_t*>(workspace);
  int rc = dt == DT_BF16 ? launch_topk<DT_BF16>(p, stream)
                         : (dt == DT_F16 ? launch_topk<DT_F16>(p, stream) : launch_topk<DT_F32>(p, stream));
  if (rc || p.blocks <= 1) return rc;
  const cudaError_t e = launch_pdl(route_sort_kernel, dim3((unsigned)p.blocks), dim3(ROUTE_THREADS),
                                   (size_t)(ROUTE_WARPS + 3) * p.Ep * sizeof(int32_t), stream, p);
  return e == cudaSuccess ? QLIN_OK : cuda_fail(e, "route sort launch");
}

int launch_combine(int dt, const void* y, int64_t R, int64_t N, int64_t ldy, const float* weights, const int32_t* pos,
                   int64_t T, int top_k, const void* residual, int64_t ld_res, void* out, cudaStream_t stream) {
  CombineParams p{y, R, N, ldy, weights, pos, T, top_k, residual, ld_res, out, 0};
  const int vec = dt == DT_F32 ? 4 : 8;
  const auto al = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  const bool ok = N % vec == 0 && ldy % vec == 0 && al(y) && al(out) &&
                  (residual == nullptr || (ld_res % vec == 0 && al(residual)));
  if (dt == DT_BF16) return launch_combine_dt<DT_BF16>(p, ok, stream);
  if (dt == DT_F16) return launch_combine_dt<DT_F16>(p, ok, stream);
  return launch_combine_dt<DT_F32>(p, ok, stream);
}

}  // namespace qlin
