// Matrix-vector products with packed 4-bit weights for few rows:
//   y[r, n] = dt(sum_g s[n, g] * (sum_{k in g} x[src(r), k] * q[n, k]) + bias[n])
// with signed nibbles q (low nibble = even k), float32 sums and one rounding.
// Unlike the W4A8 / W4A4 GEMMs the activations are not quantised.  With
// offsets [E + 1] the rows are sorted by expert and each uses its expert's
// weights.
#include "../../include/qlinear_b200.h"
#include "common.cuh"
#include "internal.h"

namespace qlin {
namespace {

struct MatvecParams {
  const void* x;
  int64_t Rx, ldx;
  const uint8_t* w;       // [E, N, K / 2]
  const void* scale;      // [E, N, groups]
  int scale_dt;
  int groups;             // scales a row: K / 128, or 1
  const int32_t* offsets; // [E + 1] or null (one expert, all rows)
  int64_t E;
  const int32_t* x_rows;  // [R] or null
  const void* bias;       // [E, N] or null
  void* out;              // [R, N]
  int64_t R, N, K;
};

// The simplest right form: one warp per output.
template <int DT>
__global__ void __launch_bounds__(256) matvec_simple_kernel(MatvecParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t o = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (o >= p.R * p.N) return;
  const int64_t r = o / p.N, n = o % p.N;
  int64_t e = 0;
  if (p.offsets != nullptr) {
    int64_t begin = max(0, p.offsets[0]);
    e = -1;
    if (r >= begin) {
      for (int64_t i = 0; i < p.E; ++i) {
        const int64_t end = max(begin, (int64_t)p.offsets[i + 1]);
        if (r < end) { e = i; break; }
        begin = end;
      }
    }
  }
  typename Elem<DT>::T* out = reinterpret_cast<typename Elem<DT>::T*>(p.out) + o;
  if (e < 0) {
    if (lane == 0) *out = Elem<DT>::from_f(0.0f);
    return;
  }
  const int64_t src = p.x_rows != nullptr ? (int64_t)p.x_rows[r] : r;
  const int64_t row = e * p.N + n;
  float acc = 0.0f;
  if (src >= 0 && src < p.Rx) {
    const typename Elem<DT>::T* x = reinterpret_cast<const typename Elem<DT>::T*>(p.x) + src * p.ldx;
    const int64_t glen = p.K / p.groups;
    for (int g = 0; g < p.groups; ++g) {
      float part = 0.0f;
      for (int64_t b = g * glen / 2 + lane; b < (g + 1) * glen / 2; b += 32) {
        const int c = (int)p.w[row * (p.K / 2) + b];
        part = __fmaf_rn(Elem<DT>::to_f(x[2 * b]), (float)(((c & 15) ^ 8) - 8), part);
        part = __fmaf_rn(Elem<DT>::to_f(x[2 * b + 1]), (float)((c >> 4 ^ 8) - 8), part);
      }
      const int64_t si = row * p.groups + g;
      const float s = p.scale_dt == DT_F32 ? reinterpret_cast<const float*>(p.scale)[si]
                                           : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.scale)[si]);
      acc = __fmaf_rn(part, s, acc);
    }
  }
#pragma unroll
  for (int o2 = 16; o2 > 0; o2 >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o2);
  if (lane == 0) {
    if (p.bias != nullptr) acc += Elem<DT>::to_f(reinterpret_cast<const typename Elem<DT>::T*>(p.bias)[row]);
    *out = Elem<DT>::from_f(acc);
  }
}

}  // namespace

int launch_matvec_w4(int dt, const void* x, int64_t Rx, int64_t ldx, const uint8_t* w, const void* scale, int scale_dt,
                     int groups, const int32_t* offsets, int64_t E, const int32_t* x_rows, const void* bias, void* out,
                     int64_t R, int64_t N, int64_t K, cudaStream_t stream) {
  const MatvecParams p{x, Rx, ldx, w, scale, scale_dt, groups, offsets, E, x_rows, bias, out, R, N, K};
  const int64_t blocks = (R * N + 7) / 8;
  if (blocks > INT32_MAX) return fail(QLIN_ERR_UNSUPPORTED, "matvec_w4: too many outputs");
  const dim3 grid((unsigned)blocks), block(256);
  cudaError_t e;
  if (dt == DT_BF16) e = launch_pdl(matvec_simple_kernel<DT_BF16>, grid, block, 0, stream, p);
  else if (dt == DT_F16) e = launch_pdl(matvec_simple_kernel<DT_F16>, grid, block, 0, stream, p);
  else e = launch_pdl(matvec_simple_kernel<DT_F32>, grid, block, 0, stream, p);
  return e == cudaSuccess ? QLIN_OK : cuda_fail(e, "matvec_w4 launch");
}

}  // namespace qlin
