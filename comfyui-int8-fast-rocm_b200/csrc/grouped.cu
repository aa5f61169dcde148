// Grouped W8A8 product: rows sorted by expert, each expert's rows times its
// own int8 weights.
//   y[r, n] = dt(dt(float(sum_k a[src(r), k] * w[e, n, k]) * xs[src(r)] * ws[e, n]) + bias[e, n])
// for the rows r of expert e, offsets[e] <= r < offsets[e + 1]; src(r) is
// a_rows[r], or r.  The rounding sequence is that of qlin_gemm_w8a8, so an
// expert's rows are bit-equal to that GEMM on them.
//
// A persistent kernel on CTA pairs.  The operands' roles are the reverse of
// the dense GEMM's: 256 weight rows are the M side of the tcgen05.mma and the
// rows of the expert its N side, whose width is set per instruction (32 to
// 256 in steps of 32).  A tile therefore costs what its rows cost, from one
// row (the weights' bytes bound it) to 256 (the tensor cores do), and the
// ragged end of each expert wastes less than 32 columns of one tile instead
// of up to 255 rows.
//
//   warp 0      producer: 128 bytes of K a stage of this CTA's 128 weight rows
//               and of its half of the tile's rows, one TMA box each, into a
//               6-stage ring
//   warp 1      TMEM and the pair's MMA issuer (leader CTA)
//   warps 2-9   epilogue: lane = weight row, column = row of the expert
//
// Gathered rows are copied into their order first (gather_kernel): a TMA
// instruction costs the producer about the same whatever it moves, and at 9
// or 33 of them a stage (16-row boxes, tile::gather4) they bound the kernel:
// 8192 rows, 8 experts, N 12288, K 4096: 341 us with boxes of 64 and 16 rows,
// 432 us with 16, 927 us with gather4, the copy costs 14.
//
// Every wait is bounded; on a timeout the kernel sets the error word, waits
// for its copies in flight, releases TMEM and returns.
#include <atomic>

#include "../../include/qlinear_b200.h"
#include "common.cuh"
#include "internal.h"

namespace qlin {
namespace {

__device__ uint32_t g_grouped_error_bits = 0;             // as the dense GEMM's: 1 timed out, 4 not drained
__device__ uint64_t g_grouped_wait_limit_ns = 2000000000ull;

__device__ __forceinline__ bool wait_bounded(uint64_t* bar, uint32_t parity, volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t limit = *reinterpret_cast<volatile uint64_t*>(&g_grouped_wait_limit_ns);
  const uint64_t t0 = globaltimer_ns();
  uint32_t iter = 0;
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((++iter & 63u) == 0) {
      if (*abort) return false;
      if (globaltimer_ns() - t0 > limit) {
        atomicOr(&g_grouped_error_bits, 1u);
        *abort = 1;
        return false;
      }
    }
  }
}
__device__ __forceinline__ void wait_drain(uint64_t* bar, uint32_t parity) {
  const uint64_t limit = *reinterpret_cast<volatile uint64_t*>(&g_grouped_wait_limit_ns);
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer_ns() - t0 > limit) {
      atomicOr(&g_grouped_error_bits, 4u);
      return;
    }
  }
}

constexpr int BM = 128;         // weight rows a CTA, 256 a pair
constexpr int BK = 128;         // bytes of K a stage
constexpr int BT = 256;         // rows of an expert a tile at most
constexpr int BOXES = 4;        // the activations' TMA boxes: 16, 32, 64 and 128 rows
constexpr int STAGES = 6;
constexpr int SLAB = BM * BK;   // 16 KB: a stage of either operand in one CTA
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 32 * (2 + EPI_WARPS);
constexpr int MAX_EXPERTS = QLIN_MAX_EXPERTS;
constexpr uint32_t TMEM_COLS = 512;  // two accumulators of 256 columns

struct GroupedParams {
  const float* a_scale;    // [R]
  const float* w_scale;    // [E, N]
  const int32_t* offsets;  // [E + 1]
  int E;
  const void* bias;        // [E, N] in the output dtype, or null
  void* out;               // [R, N]
  int R, N, K;
};

struct Smem {  // behind the operand ring
  uint64_t full[STAGES], empty[STAGES], tfull[2], tempty[2], drain;
  uint32_t tmem_slot;
  int abort_flag;
  alignas(16) float xs[2][BT];       // activation scales of a tile's rows
  int begin[MAX_EXPERTS + 1];        // first row of each expert, ascending within [0, R]
  int cum[MAX_EXPERTS + 1];          // tiles before each expert's
};
constexpr int SMEM_BYTES = 1024 + 2 * STAGES * SLAB + (int)sizeof(Smem);
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");

// A tile's place: expert, first weight row of the pair, first row and number
// of rows.  Tiles are numbered expert by expert, weight blocks outside and
// row blocks inside, so that pairs that run together share weights in L2.
struct Tile {
  int e, n0, row0, rows, width;
};
__device__ __forceinline__ Tile locate(const Smem* s, int tile, int& e) {
  while (s->cum[e + 1] <= tile) ++e;  // the caller's tiles ascend
  Tile t;
  t.e = e;
  const int m = s->begin[e + 1] - s->begin[e];
  const int blocks = (m + BT - 1) / BT;
  const int step = ((m + blocks - 1) / blocks + 31) & ~31;  // equal row blocks
  const int j = tile - s->cum[e];
  t.n0 = j / blocks * (2 * BM);
  const int r = j % blocks * step;
  t.row0 = s->begin[e] + r;
  t.rows = min(step, m - r);
  t.width = (t.rows + 31) & ~31;  // columns of the MMA
  return t;
}

__device__ __forceinline__ void epilogue_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(32 * EPI_WARPS) : "memory"); }

// Zeros in [b0, b1) bytes of the (16-byte aligned) output, both even, by `count` threads.
__device__ void zero_bytes(void* out, int64_t b0, int64_t b1, int64_t thread, int64_t count) {
  char* o = static_cast<char*>(out);
  const int64_t v0 = min((b0 + 15) & ~int64_t(15), b1), v1 = max(b1 & ~int64_t(15), v0);
  for (int64_t i = v0 + 16 * thread; i < v1; i += 16 * count)
    *reinterpret_cast<uint4*>(o + i) = make_uint4(0u, 0u, 0u, 0u);
  for (int64_t i = b0 + 2 * thread; i < v0; i += 2 * count) *reinterpret_cast<uint16_t*>(o + i) = 0;
  for (int64_t i = v1 + 2 * thread; i < b1; i += 2 * count) *reinterpret_cast<uint16_t*>(o + i) = 0;
}

// 32 columns (rows of the expert) of one accumulator: this thread has weight
// row n of all of them.  16-bit results are exchanged between neighbouring
// lanes so that each store writes two columns of one output row.
template <int DT>
__device__ __forceinline__ void store_chunk(const GroupedParams& p, const uint32_t (&r)[32], const float* xs, float ws,
                                            float bias, bool has_bias, int64_t row, int rows, int n, int lane) {
  using EO = Elem<DT>;
  using T = typename EO::T;
  float y[32];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 x = reinterpret_cast<const float4*>(xs)[i];
    y[4 * i] = __fmul_rn(__fmul_rn(__int2float_rn((int)r[4 * i]), x.x), ws);
    y[4 * i + 1] = __fmul_rn(__fmul_rn(__int2float_rn((int)r[4 * i + 1]), x.y), ws);
    y[4 * i + 2] = __fmul_rn(__fmul_rn(__int2float_rn((int)r[4 * i + 2]), x.z), ws);
    y[4 * i + 3] = __fmul_rn(__fmul_rn(__int2float_rn((int)r[4 * i + 3]), x.w), ws);
  }
  if (has_bias) {
#pragma unroll
    for (int j = 0; j < 32; ++j) y[j] = __fadd_rn(EO::round(y[j]), bias);
  }
  T* out = reinterpret_cast<T*>(p.out) + row * p.N;
  if (DT == DT_F32 || (p.N & 1)) {
    if (n < p.N) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < rows) out[(int64_t)j * p.N + n] = EO::from_f(y[j]);
    }
    return;
  }
  uint32_t* words = reinterpret_cast<uint32_t*>(out) + (n >> 1);
  const int64_t pitch = p.N >> 1;
  const int odd = lane & 1;
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    uint32_t own;
    if constexpr (DT == DT_F16) {
      const __half2 h = __floats2half2_rn(y[j], y[j + 1]);
      own = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(y[j], y[j + 1]);
      own = *reinterpret_cast<const uint32_t*>(&h);
    }
    const uint32_t other = __shfl_xor_sync(0xffffffffu, own, 1);
    const uint32_t w = odd ? __byte_perm(other, own, 0x7632) : __byte_perm(own, other, 0x5410);
    if (j + odd < rows && n < p.N) words[(j + odd) * pitch] = w;
  }
}

struct RowMaps {
  CUtensorMap box[BOXES];  // the activations in boxes of 16 << i rows
};

template <int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    grouped_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ RowMaps tmX, GroupedParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sW = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sX = sW + STAGES * SLAB;
  Smem* s = reinterpret_cast<Smem*>(sX + STAGES * SLAB);
  volatile int* abort_flag = &s->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&s->full[i], 1);
      mbar_init(&s->empty[i], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&s->tfull[b], 1);
      mbar_init(&s->tempty[b], 2 * EPI_WARPS);
    }
    mbar_init(&s->drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(&s->tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // barriers of both CTAs initialised, TMEM allocated
  tc_fence_after();
  const uint32_t tmem_base = s->tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  // Row ranges and tile numbers of the experts, whatever the offsets hold.
  for (int e = threadIdx.x; e <= p.E; e += THREADS) s->begin[e] = min(max(p.offsets[e], 0), p.R);
  __syncthreads();
  const int num_n = (p.N + 2 * BM - 1) / (2 * BM);
  if (warp == 0) {
    int top = 0, tiles = 0;
    for (int e0 = 0; e0 <= p.E; e0 += 32) {
      const int e = e0 + lane;
      int b = e <= p.E ? s->begin[e] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) b = max(b, u);
      }
      b = max(b, top);
      int before = __shfl_up_sync(0xffffffffu, b, 1);
      if (lane == 0) before = e0 == 0 ? b : top;
      int n = e <= p.E ? (b - before + BT - 1) / BT * num_n : 0;  // tiles of expert e - 1
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += u;
      }
      if (e <= p.E) {
        s->begin[e] = b;
        s->cum[e] = tiles + n;
      }
      top = __shfl_sync(0xffffffffu, b, 31);
      tiles += __shfl_sync(0xffffffffu, n, 31);
    }
  }
  __syncthreads();
  const int num_tiles = s->cum[p.E];
  const int num_kb = (p.K + BK - 1) / BK;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (warp == 0) {
    // ---------------- producer (both CTAs) ----------------
    if (lane == 0) {
      tma_prefetch_desc(&tmW);
      for (int i = 0; i < BOXES; ++i) tma_prefetch_desc(&tmX.box[i]);
      int stage = 0, e = 0;
      uint32_t phase = 0, armed = 0, parity = 0;  // of the stages filled so far
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step) {
        const Tile t = locate(s, tile, e);
        const int half = t.width >> 1;
        const int wrow = t.e * p.N + t.n0 + (int)rank * BM, xrow = t.row0 + (int)rank * half;
        // the smallest box that holds this CTA's rows (the MMA reads no more of them)
        int box = 0;
        while ((16 << box) < half) ++box;
        const CUtensorMap* tmx = &tmX.box[box];
        const uint32_t bytes = 2 * (SLAB + (16 << box) * BK);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!wait_bounded(&s->empty[stage], phase ^ 1, abort_flag)) { ok = false; break; }
          const uint32_t fb = mapa_shared(smem_u32(&s->full[stage]), 0);
          if (leader) mbar_arrive_expect_tx(&s->full[stage], bytes);
          tma_load_2d_pair(sW + stage * SLAB, &tmW, fb, kb * BK, wrow);
          tma_load_2d_pair(sX + stage * SLAB, tmx, fb, kb * BK, xrow);
          armed |= 1u << stage;
          parity = (parity & ~(1u << stage)) | (phase << stage);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // no load still writing shared memory at exit (both CTAs' loads are
      // counted by the leader; the peer waits for it at the last cluster barrier)
      if (leader)
        for (int i = 0; i < STAGES; ++i)
          if (armed >> i & 1u) wait_drain(&s->full[i], parity >> i & 1u);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (leader CTA) ----------------
    if (leader && lane == 0) {
      int stage = 0, acc = 0, e = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool issued = false, ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += step) {
        const Tile t = locate(s, tile, e);
        const uint32_t idesc = umma_idesc_i8(2 * BM, t.width);
        if (!wait_bounded(&s->tempty[acc], acc_phase ^ 1, abort_flag)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + acc * BT;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!wait_bounded(&s->full[stage], phase, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint64_t wdesc = umma_desc_k_sw128(smem_u32(sW + stage * SLAB));
          const uint64_t xdesc = umma_desc_k_sw128(smem_u32(sX + stage * SLAB));
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            umma_i8_pair(d, wdesc + 2 * k, xdesc + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
          issued = true;
          umma_commit_pair(&s->empty[stage], 0x3);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        umma_commit_pair(&s->tfull[acc], 0x3);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      if (*abort_flag && issued) {  // MMAs complete before TMEM is released
        umma_commit_pair(&s->drain, 0x1);
        wait_drain(&s->drain, 0);
      }
    }
  } else {
    // ---------------- epilogue (both CTAs) ----------------
    using EO = Elem<DT>;
    const int tid = threadIdx.x - 64, quarter = warp & 3, half = (warp - 2) >> 2;
    {  // rows of no expert
      const int64_t line = (int64_t)p.N * sizeof(typename EO::T);
      const int64_t thread = (int64_t)blockIdx.x * 32 * EPI_WARPS + tid, count = (int64_t)gridDim.x * 32 * EPI_WARPS;
      if (s->begin[0] > 0) zero_bytes(p.out, 0, s->begin[0] * line, thread, count);
      if (s->begin[p.E] < p.R) zero_bytes(p.out, s->begin[p.E] * line, p.R * line, thread, count);
    }
    int acc = 0, e = 0;
    uint32_t acc_phase = 0;
    const bool has_bias = p.bias != nullptr;
    for (int tile = first; tile < num_tiles; tile += step) {
      const Tile t = locate(s, tile, e);
      // this tile's scales and bias, while its products are computed
      const int n = t.n0 + (int)rank * BM + quarter * 32 + lane;
      float ws = 0.0f, bias = 0.0f, xs = 0.0f;
      if (n < p.N) {
        const int64_t at = (int64_t)t.e * p.N + n;
        ws = __ldg(p.w_scale + at);
        if (has_bias) bias = EO::to_f(reinterpret_cast<const typename EO::T*>(p.bias)[at]);
      }
      if (tid < t.rows) xs = __ldg(p.a_scale + t.row0 + tid);
      s->xs[acc][tid] = xs;
      wait_bounded(&s->tfull[acc], acc_phase, abort_flag);
      epilogue_barrier();
      if (*abort_flag) break;
      tc_fence_after();
      for (int c = half * 32; c < t.rows; c += 64) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(tmem_base + acc * BT + c + ((uint32_t)(quarter * 32) << 16), r);
        tmem_ld_wait_regs(r);
        store_chunk<DT>(p, r, &s->xs[acc][c], ws, bias, has_bias, t.row0 + c, t.rows - c, n, lane);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&s->tempty[acc]), 0));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
  }

  tc_fence_before();
  cluster_sync();  // all MMAs done and all remote arrivals delivered
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// Rows a[rows[r]] and their scales in the order of r, zeros for an index
// outside [0, Ra); a block takes `per` rows, a thread 16 bytes at a time.
constexpr int GATHER_THREADS = 256;
__global__ void __launch_bounds__(GATHER_THREADS)
    gather_kernel(const int8_t* __restrict__ a, const float* __restrict__ a_scale, int64_t Ra,
                  const int32_t* __restrict__ rows, int64_t R, int K16, int per, int8_t* __restrict__ out,
                  float* __restrict__ out_scale) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t r0 = (int64_t)blockIdx.x * per;
  const int count = (int)min((int64_t)per, R - r0);
  const uint4* src = reinterpret_cast<const uint4*>(a);
  uint4* dst = reinterpret_cast<uint4*>(out) + r0 * K16;
  const int total = count * K16;
#pragma unroll 4
  for (int i = threadIdx.x; i < total; i += GATHER_THREADS) {
    const int64_t from = rows[r0 + i / K16];
    dst[i] = from >= 0 && from < Ra ? src[from * K16 + i % K16] : make_uint4(0u, 0u, 0u, 0u);
  }
  for (int i = threadIdx.x; i < count; i += GATHER_THREADS) {
    const int64_t from = rows[r0 + i];
    out_scale[r0 + i] = from >= 0 && from < Ra ? a_scale[from] : 0.0f;
  }
}

template <int DT>
int launch_dt(const CUtensorMap& tw, const RowMaps& tx, const GroupedParams& p, int clusters, cudaStream_t stream) {
  auto kern = grouped_kernel<DT>;
  static std::atomic<uint64_t> attr_devices{0};  // shared-memory limit raised once per device
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  cudaError_t e;
  if (!(attr_devices.load() & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(grouped)");
    attr_devices.fetch_or(bit);
  }
  e = launch_pdl(kern, dim3(2 * clusters), dim3(THREADS), SMEM_BYTES, stream, tw, tx, p);
  return e == cudaSuccess ? QLIN_OK : cuda_fail(e, "grouped GEMM launch");
}

size_t gather_scale_offset(int64_t R, int64_t K) { return ((size_t)R * K + 15) & ~size_t(15); }

}  // namespace

size_t grouped_workspace_bytes(int64_t R, int64_t K) { return gather_scale_offset(R, K) + (size_t)R * sizeof(float); }

int launch_grouped(const int8_t* a, const float* a_scale, int64_t Ra, const int8_t* w, const float* w_scale,
                   const int32_t* offsets, int64_t E, const int32_t* a_rows, const void* bias, void* out, int out_dt,
                   int64_t R, int64_t N, int64_t K, void* workspace, cudaStream_t stream) {
  const int sms = device_sm_count();
  if (sms < 2) return fail(QLIN_ERR_NO_DEVICE, "no CUDA device");
  if (a_rows != nullptr) {
    int8_t* sorted = static_cast<int8_t*>(workspace);
    float* scale = reinterpret_cast<float*>(sorted + gather_scale_offset(R, K));
    // about 16 KB a block: four 16-byte copies in flight a thread
    const int per = (int)(K >= 16384 ? 1 : 16384 / K);
    const cudaError_t e = launch_pdl(gather_kernel, dim3((unsigned)((R + per - 1) / per)), dim3(GATHER_THREADS), 0,
                                     stream, a, a_scale, Ra, a_rows, R, (int)(K / 16), per, sorted, scale);
    if (e != cudaSuccess) return cuda_fail(e, "grouped GEMM gather launch");
    a = sorted;
    a_scale = scale;
  }
  CUtensorMap tw;
  RowMaps tx;
  int rc = encode_rows_tmap(&tw, w, (uint64_t)K, (uint64_t)(E * N), BK, BM);
  for (int i = 0; i < BOXES && !rc; ++i) rc = encode_rows_tmap(&tx.box[i], a, (uint64_t)K, (uint64_t)R, BK, 16 << i);
  if (rc) return rc;
  const GroupedParams p{a_scale, w_scale, offsets, (int)E, bias, out, (int)R, (int)N, (int)K};
  // tiles at most: every expert adds one partly filled row block to R / 256
  const int64_t tiles = (R / BT + (E < R ? E : R)) * ((N + 2 * BM - 1) / (2 * BM));
  const int clusters = (int)(tiles < sms / 2 ? tiles : sms / 2);
  if (out_dt == DT_BF16) return launch_dt<DT_BF16>(tw, tx, p, clusters, stream);
  if (out_dt == DT_F16) return launch_dt<DT_F16>(tw, tx, p, clusters, stream);
  return launch_dt<DT_F32>(tw, tx, p, clusters, stream);
}

int set_grouped_wait_limit(uint64_t ns) {
  const cudaError_t e = cudaMemcpyToSymbol(g_grouped_wait_limit_ns, &ns, sizeof(ns));
  return e == cudaSuccess ? QLIN_OK : cuda_fail(e, "set grouped GEMM wait limit");
}

int read_grouped_error(cudaStream_t stream, uint32_t* bits) {
  uint32_t h = 0;
  cudaError_t e =
      cudaMemcpyFromSymbolAsync(&h, g_grouped_error_bits, sizeof(uint32_t), 0, cudaMemcpyDeviceToHost, stream);
  if (e != cudaSuccess) return cuda_fail(e, "read grouped GEMM error word");
  const uint32_t zero = 0;
  e = cudaMemcpyToSymbolAsync(g_grouped_error_bits, &zero, sizeof(uint32_t), 0, cudaMemcpyHostToDevice, stream);
  if (e != cudaSuccess) return cuda_fail(e, "clear grouped GEMM error word");
  e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess) return cuda_fail(e, "sync");
  *bits = h;
  return QLIN_OK;
}

}  // namespace qlin
