// Routing of tokens to experts and the weighted sum back: the plan of a
// mixture-of-experts layer whose products run in grouped.cu (int8 weights)
// and matvec.cu (4-bit weights).
//
//   route    logits [T, E] -> the k best experts of every token and their
//            weights, and the (token, slot) pairs sorted by expert;
//   combine  out[t] = sum_j weight[t, j] * y[pos[t, j]] (+ residual[t]).
#include <cfloat>
#include <cmath>

#include "../../include/qlinear_b200.h"
#include "common.cuh"
#include "internal.h"

namespace qlin {
namespace {

constexpr int ROUTE_THREADS = 256;
constexpr int ROUTE_WARPS = ROUTE_THREADS / 32;
constexpr int ROUTE_MIN_TOKENS = 64;   // tokens of a block: 8 a warp at least
constexpr int ROUTE_MAX_BLOCKS = 296;  // two a SM: the second kernel reads every block's counts
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

// Floats in the order of their values as unsigned numbers; 0 is below all.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// log(1 / (1 + exp(-v))) without overflow on either side
__device__ __forceinline__ float log_sigmoid(float v) { return fminf(v, 0.0f) - log1pf(expf(-fabsf(v))); }

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
  for (int64_t t = t0; t < t1; ++t) {
    if (lane < p.k) {
      const int id = p.ids[t * p.k + lane];
      int at = -1;
      if (id >= 0) {
        at = run[id];
        run[id] = at + 1;
        p.rows[at] = (int32_t)t;
      }
      p.pos[t * p.k + lane] = at;
    }
    __syncwarp();
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

// One warp per token: lane l holds logits l, l + 32, ...; k rounds of the
// warp's maximum (the lowest index where values tie), each two warp-wide
// reductions, leave slot j's expert and logit in lane j.
template <int DT, int PER>
__global__ void __launch_bounds__(ROUTE_THREADS) route_topk_kernel(RouteParams p) {
  extern __shared__ int32_t s_route[];
  int32_t* s_cnt = s_route;                       // [warps][Ep]
  int32_t* s_tot = s_cnt + ROUTE_WARPS * p.Ep;    // [Ep]
  int32_t* s_base = s_tot + p.Ep;                 // [Ep]
  __shared__ int32_t s_total;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < ROUTE_WARPS * p.Ep; i += ROUTE_THREADS) s_cnt[i] = 0;
  __syncthreads();
  pdl_wait();
  const int64_t per_warp = p.tokens / ROUTE_WARPS;
  const int64_t t0 = min((int64_t)blockIdx.x * p.tokens + warp * per_warp, p.T);
  const int64_t t1 = min(t0 + per_warp, p.T);
  const typename Elem<DT>::T* x = reinterpret_cast<const typename Elem<DT>::T*>(p.logits);
  int32_t* cnt = s_cnt + warp * p.Ep;
  for (int64_t t = t0; t < t1; ++t) {
    float v[PER];
    uint32_t key[PER];
    bool nan = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane + 32 * i;
      v[i] = e < p.E ? Elem<DT>::to_f(x[t * p.ld + e]) : NEG_INF;
      const bool bad = v[i] != v[i];
      nan |= bad;
      key[i] = ordered(bad ? NEG_INF : v[i] + 0.0f);  // -0 and +0 tie
    }
    const uint32_t none = ordered(NEG_INF);
    int my_id = -1;
    float my_v = NEG_INF;
    for (int j = 0; j < p.k; ++j) {
      uint32_t best = key[0];
      int at = 0;
#pragma unroll
      for (int i = 1; i < PER; ++i)
        if (key[i] > best) { best = key[i]; at = i; }
      const uint32_t m = __reduce_max_sync(0xffffffffu, best);
      if (m <= none) break;  // the rest may not be chosen
      const uint32_t id = __reduce_min_sync(0xffffffffu, best == m ? (uint32_t)(lane + 32 * at) : 0xffffffffu);
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if ((uint32_t)(lane + 32 * i) == id) key[i] = 0u;
      if (lane == j) { my_id = (int)id; my_v = unordered(m); }
    }
    const bool chosen = my_id >= 0;
    float w = 0.0f;
    if (p.sigmoid) {
      if (p.renorm) {  // s_j / sum s = softmax of the chosen log-sigmoids: no 0 / 0 far below zero
        const float l = log_sigmoid(my_v);
        const float ref = __shfl_sync(0xffffffffu, l, 0);
        const float e = chosen ? expf(l - ref) : 0.0f;
        w = e / warp_sum(e);
      } else {
        w = 1.0f / (1.0f + expf(-my_v));
      }
    } else {
      const float top = __shfl_sync(0xffffffffu, my_v, 0);
      const float e = chosen ? expf(my_v - top) : 0.0f;
      float part = e;
      if (!p.renorm) {
        part = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (lane + 32 * i < p.E) part += expf(v[i] - top);
      }
      w = e / warp_sum(part);
      if (__any_sync(0xffffffffu, nan)) w = NAN;
    }
    if (lane < p.k) {
      p.ids[t * p.k + lane] = my_id;
      p.weights[t * p.k + lane] = chosen ? w : 0.0f;
      if (chosen) cnt[my_id] += 1;  // a token's experts differ: no two lanes meet
    }
    __syncwarp();
  }
  __syncthreads();
  pdl_launch_dependents();
  for (int e = threadIdx.x; e < p.Ep; e += ROUTE_THREADS) {
    int c = 0;
#pragma unroll
    for (int w = 0; w < ROUTE_WARPS; ++w) c += s_cnt[w * p.Ep + e];
    if (p.blocks > 1) p.counts[(int64_t)blockIdx.x * p.Ep + e] = c;
    else s_tot[e] = c;
  }
  if (p.blocks > 1) return;
  // one block holds all tokens: it sorts them too
  __syncthreads();
  const int total = scan_experts(p, s_tot, s_base, &s_total, true);
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
  int32_t* cnt = s_cnt + warp * p.Ep;
  for (int64_t t = t0; t < t1; ++t) {
    if (lane < p.k) {
      const int id = p.ids[t * p.k + lane];
      if (id >= 0) cnt[id] += 1;
    }
    __syncwarp();
  }
  int cols = 1;
  while (cols < p.Ep / 4) cols <<= 1;  // <= 128 for E <= 512
  const int col = threadIdx.x & (cols - 1), slices = ROUTE_THREADS / cols;
  if (col < p.Ep / 4) {
    int4 pre = make_int4(0, 0, 0, 0), tot = make_int4(0, 0, 0, 0);
#pragma unroll 4
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
  tokens = (T + ROUTE_MAX_BLOCKS - 1) / ROUTE_MAX_BLOCKS;
  tokens = (tokens + ROUTE_WARPS - 1) / ROUTE_WARPS * ROUTE_WARPS;
  if (tokens < ROUTE_MIN_TOKENS) tokens = ROUTE_MIN_TOKENS;
  blocks = (T + tokens - 1) / tokens;
}

template <int DT>
int launch_topk(const RouteParams& p, cudaStream_t s) {
  const size_t smem = (size_t)(ROUTE_WARPS + 2) * p.Ep * sizeof(int32_t);
  const dim3 grid((unsigned)p.blocks), block(ROUTE_THREADS);
  cudaError_t e;
  if (p.E <= 32) e = launch_pdl(route_topk_kernel<DT, 1>, grid, block, smem, s, p);
  else if (p.E <= 64) e = launch_pdl(route_topk_kernel<DT, 2>, grid, block, smem, s, p);
  else if (p.E <= 128) e = launch_pdl(route_topk_kernel<DT, 4>, grid, block, smem, s, p);
  else if (p.E <= 256) e = launch_pdl(route_topk_kernel<DT, 8>, grid, block, smem, s, p);
  else e = launch_pdl(route_topk_kernel<DT, 16>, grid, block, smem, s, p);
  return e == cudaSuccess ? QLIN_OK : cuda_fail(e, "route launch");
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

// One thread per VEC columns of a token: a float32 sum in slot order, rounded
// once.  HBM bound: every row of y that a token chose is read once.
template <int DT, int VEC>
__global__ void __launch_bounds__(128) combine_kernel(CombineParams p) {
  using T = typename Elem<DT>::T;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t t = blockIdx.x / p.chunks;
  const int64_t col = ((blockIdx.x % p.chunks) * 128 + threadIdx.x) * VEC;
  if (col >= p.N) return;
  const T* y = reinterpret_cast<const T*>(p.y) + col;
  float acc[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
  for (int j = 0; j < p.k; ++j) {
    const int at = p.pos[t * p.k + j];
    if (at < 0 || at >= p.R) continue;
    const float w = p.weights[t * p.k + j];
    alignas(16) T v[VEC];
    if constexpr (VEC == 1) v[0] = y[at * p.ldy];
    else *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(y + at * p.ldy));
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = __fmaf_rn(w, Elem<DT>::to_f(v[i]), acc[i]);
  }
  alignas(16) T v[VEC];
  if (p.residual != nullptr) {
    const T* r = reinterpret_cast<const T*>(p.residual) + t * p.ld_res + col;
    if constexpr (VEC == 1) v[0] = r[0];
    else *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(r));
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] += Elem<DT>::to_f(v[i]);
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = Elem<DT>::from_f(acc[i]);
  T* o = reinterpret_cast<T*>(p.out) + t * p.N + col;
  if constexpr (VEC == 1) o[0] = v[0];
  else *reinterpret_cast<uint4*>(o) = *reinterpret_cast<uint4*>(v);
}

template <int DT>
int launch_combine_dt(CombineParams p, bool vec, cudaStream_t s) {
  constexpr int VEC = 16 / sizeof(typename Elem<DT>::T);
  const int64_t per = 128 * (vec ? VEC : 1);
  p.chunks = (p.N + per - 1) / per;
  if (p.chunks * p.T > INT32_MAX) return fail(QLIN_ERR_UNSUPPORTED, "combine: too many tokens");
  const dim3 grid((unsigned)(p.chunks * p.T));
  const cudaError_t e = vec ? launch_pdl(combine_kernel<DT, VEC>, grid, dim3(128), 0, s, p)
                            : launch_pdl(combine_kernel<DT, 1>, grid, dim3(128), 0, s, p);
  return e == cudaSuccess ? QLIN_OK : cuda_fail(e, "combine launch");
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
