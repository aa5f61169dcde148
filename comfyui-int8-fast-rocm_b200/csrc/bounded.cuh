// Bounded mbarrier waits for a translation unit that includes this once: its
// own error word and wait limit, read and set through the two host functions.
// Error bits as the dense GEMM's: 1 a pipeline wait ran out, 4 in-flight work
// did not drain within the limit either.
#pragma once

#include "common.cuh"
#include "internal.h"

namespace qlin {
namespace {

__device__ uint32_t g_tu_error_bits = 0;
__device__ uint64_t g_tu_wait_limit_ns = 2000000000ull;

// False (after setting the error word and *abort) if the phase did not
// complete within the limit, or another role of the CTA gave up before.
__device__ __forceinline__ bool wait_bounded(uint64_t* bar, uint32_t parity, volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t limit = *reinterpret_cast<volatile uint64_t*>(&g_tu_wait_limit_ns);
  const uint64_t t0 = globaltimer_ns();
  uint32_t iter = 0;
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((++iter & 63u) == 0) {
      if (*abort) return false;
      if (globaltimer_ns() - t0 > limit) {
        atomicOr(&g_tu_error_bits, 1u);
        *abort = 1;
        return false;
      }
    }
  }
}

// The same by all lanes of a warp, which go by one verdict: a wait that runs
// out must not part lanes that meet at shuffles and votes later on.
__device__ __forceinline__ bool wait_bounded_warp(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, wait_bounded(bar, parity, abort));
}

// Waits (whatever the abort flag says) for asynchronous work issued earlier,
// twice the limit at most: a role that owes the barrier arrivals may first
// have to run out its own wait.
__device__ __forceinline__ void wait_drain(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return;
  const uint64_t limit = 2 * *reinterpret_cast<volatile uint64_t*>(&g_tu_wait_limit_ns);
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer_ns() - t0 > limit) {
      atomicOr(&g_tu_error_bits, 4u);
      return;
    }
  }
}

// A count that another role sets (from -1) when it leaves its loop, which it
// does within the limit of its own last wait; -1 if it has not by twice that.
__device__ __forceinline__ int wait_value(const volatile int* value) {
  const uint64_t limit = 2 * *reinterpret_cast<volatile uint64_t*>(&g_tu_wait_limit_ns);
  const uint64_t t0 = globaltimer_ns();
  int v;
  while ((v = *value) < 0) {
    if (globaltimer_ns() - t0 > limit) {
      atomicOr(&g_tu_error_bits, 4u);
      break;
    }
  }
  return v;
}

int set_tu_wait_limit(uint64_t ns) {
  const cudaError_t e = cudaMemcpyToSymbol(g_tu_wait_limit_ns, &ns, sizeof(ns));
  return e == cudaSuccess ? QLIN_OK : cuda_fail(e, "set wait limit");
}

int read_tu_error(cudaStream_t stream, uint32_t* bits) {
  uint32_t h = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&h, g_tu_error_bits, sizeof(uint32_t), 0, cudaMemcpyDeviceToHost, stream);
  if (e != cudaSuccess) return cuda_fail(e, "read error word");
  const uint32_t zero = 0;
  e = cudaMemcpyToSymbolAsync(g_tu_error_bits, &zero, sizeof(uint32_t), 0, cudaMemcpyHostToDevice, stream);
  if (e != cudaSuccess) return cuda_fail(e, "clear error word");
  e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess) return cuda_fail(e, "sync");
  *bits = h;
  return QLIN_OK;
}

// Stages of a ring that a producer filled (bit s) and their last phases: it
// waits for those fills before it leaves its role.
struct Armed {
  uint32_t stages = 0, parity = 0;
  __device__ __forceinline__ void note(int stage, uint32_t phase) {
    stages |= 1u << stage;
    parity = (parity & ~(1u << stage)) | (phase << stage);
  }
  __device__ __forceinline__ void drain(uint64_t* full) const {
    for (int i = 0; i < 32; ++i)
      if (stages >> i & 1u) wait_drain(&full[i], parity >> i & 1u);
  }
};

// Ascending bounds in [0, R] of the experts' rows, whatever the offsets hold:
// begin[e] for e = 0 .. E holds the offset clamped to [0, R] on entry, and at
// least the one before on return; cum[e] the sum of items(rows) over the
// experts before e.  One warp.
template <class F>
__device__ __forceinline__ void expert_bounds(int* begin, int* cum, int E, int lane, F items) {
  int top = 0, total = 0;
  for (int e0 = 0; e0 <= E; e0 += 32) {
    const int e = e0 + lane;
    int b = e <= E ? begin[e] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= o) b = max(b, u);
    }
    b = max(b, top);
    int before = __shfl_up_sync(0xffffffffu, b, 1);
    if (lane == 0) before = e0 == 0 ? b : top;
    int n = e <= E ? items(b - before) : 0;  // of expert e - 1
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += u;
    }
    if (e <= E) {
      begin[e] = b;
      cum[e] = total + n;
    }
    top = __shfl_sync(0xffffffffu, b, 31);
    total += __shfl_sync(0xffffffffu, n, 31);
  }
}

// Zeros in [b0, b1) bytes of a 16-byte aligned buffer, both even, by thread
// `thread` of `count`.
__device__ void zero_bytes(void* out, int64_t b0, int64_t b1, int64_t thread, int64_t count) {
  char* o = static_cast<char*>(out);
  const int64_t v0 = min((b0 + 15) & ~int64_t(15), b1), v1 = max(b1 & ~int64_t(15), v0);
  for (int64_t i = v0 + 16 * thread; i < v1; i += 16 * count)
    *reinterpret_cast<uint4*>(o + i) = make_uint4(0u, 0u, 0u, 0u);
  for (int64_t i = b0 + 2 * thread; i < v0; i += 2 * count) *reinterpret_cast<uint16_t*>(o + i) = 0;
  for (int64_t i = v1 + 2 * thread; i < b1; i += 2 * count) *reinterpret_cast<uint16_t*>(o + i) = 0;
}

}  // namespace
}  // namespace qlin
