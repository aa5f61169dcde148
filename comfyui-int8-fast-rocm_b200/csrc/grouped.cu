// Grouped W8A8 product: rows sorted by expert, each expert's rows times its
// own int8 weights.
//   y[r, n] = dt(dt(float(sum_k a[src(r), k] * w[e, n, k]) * xs[src(r)] * ws[e, n]) + bias[e, n])
// for the rows r of expert e, offsets[e] <= r < offsets[e + 1]; src(r) is
// a_rows[r], or r.  The rounding sequence is that of qlin_gemm_w8a8, so an
// expert's rows are bit-equal to that GEMM on them.
#include "../../include/qlinear_b200.h"
#include "common.cuh"
#include "internal.h"

namespace qlin {
namespace {

struct GroupedParams {
  const int8_t* a;        // [Ra, K]
  const float* a_scale;   // [Ra]
  int64_t Ra;
  const int8_t* w;        // [E, N, K]
  const float* w_scale;   // [E, N]
  const int32_t* offsets; // [E + 1]
  int64_t E;
  const int32_t* a_rows;  // [R] or null
  const void* bias;       // [E, N] in the output dtype, or null
  void* out;              // [R, N]
  int64_t R, N, K;
};

// The simplest right form: one warp per output, four products an instruction.
template <int DT>
__global__ void __launch_bounds__(256) grouped_simple_kernel(GroupedParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t o = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (o >= p.R * p.N) return;
  const int64_t r = o / p.N, n = o % p.N;
  int64_t e = -1, begin = max(0, p.offsets[0]);
  if (r >= begin) {
    for (int64_t i = 0; i < p.E; ++i) {
      const int64_t end = max(begin, (int64_t)p.offsets[i + 1]);
      if (r < end) { e = i; break; }
      begin = end;
    }
  }
  using EO = Elem<DT>;
  typename EO::T* out = reinterpret_cast<typename EO::T*>(p.out) + o;
  if (e < 0) {
    if (lane == 0) *out = EO::from_f(0.0f);
    return;
  }
  const int64_t src = p.a_rows != nullptr ? (int64_t)p.a_rows[r] : r;
  const bool ok = src >= 0 && src < p.Ra;
  int acc = 0;
  if (ok)
    for (int64_t k = lane * 4; k < p.K; k += 128)
      acc = __dp4a(*reinterpret_cast<const int*>(p.a + src * p.K + k),
                   *reinterpret_cast<const int*>(p.w + (e * p.N + n) * p.K + k), acc);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, i);
  if (lane == 0) {
    const float xs = ok ? p.a_scale[src] : 0.0f;
    float y = EO::round(__fmul_rn(__fmul_rn(__int2float_rn(acc), xs), p.w_scale[e * p.N + n]));
    if (p.bias != nullptr) y = __fadd_rn(y, EO::to_f(reinterpret_cast<const typename EO::T*>(p.bias)[e * p.N + n]));
    *out = EO::from_f(y);
  }
}

}  // namespace

int launch_grouped(const int8_t* a, const float* a_scale, int64_t Ra, const int8_t* w, const float* w_scale,
                   const int32_t* offsets, int64_t E, const int32_t* a_rows, const void* bias, void* out, int out_dt,
                   int64_t R, int64_t N, int64_t K, cudaStream_t stream) {
  const GroupedParams p{a, a_scale, Ra, w, w_scale, offsets, E, a_rows, bias, out, R, N, K};
  const int64_t blocks = (R * N + 7) / 8;
  if (blocks > INT32_MAX) return fail(QLIN_ERR_UNSUPPORTED, "grouped GEMM: too many outputs");
  const dim3 grid((unsigned)blocks), block(256);
  cudaError_t e;
  if (out_dt == DT_BF16) e = launch_pdl(grouped_simple_kernel<DT_BF16>, grid, block, 0, stream, p);
  else if (out_dt == DT_F16) e = launch_pdl(grouped_simple_kernel<DT_F16>, grid, block, 0, stream, p);
  else e = launch_pdl(grouped_simple_kernel<DT_F32>, grid, block, 0, stream, p);
  return e == cudaSuccess ? QLIN_OK : cuda_fail(e, "grouped GEMM launch");
}

}  // namespace qlin
