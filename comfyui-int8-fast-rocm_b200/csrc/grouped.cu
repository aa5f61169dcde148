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
//   warp 0      producer: this CTA's 128 weight rows and its half of the tile's
//               rows, one TMA box each a stage, into a ring of 3 stages of 256
//               bytes of K (6 of 128 where K is no multiple of 128)
//   warp 1      TMEM and the pair's MMA issuer (leader CTA)
//   warps 2-9   epilogue: lane = weight row, column = row of the expert
//
// What bounds it: with many rows the feed of the tensor cores.  8192 rows, 8
// experts, N 12288, K 4096 take 289-311 us on different GPUs (2.65-2.85
// POP/s); one expert of 8192 rows takes 260-275, where the dense GEMM takes
// 261-270.  Weights that are read for the first time cost 9% of that, the
// epilogue's stores 8% (a copy of the kernel without each); at K 1536 the
// stores cost a fifth.  With few rows the weights' bytes: 24 experts with
// rows, N 2048, K 4096, 202 MB in 39 us (5.1 TB/s), 41.6 with gathered rows.
//
// A TMA instruction costs the producer about the same whatever it moves, so
// each operand comes in one box a stage (the case of 8192 rows: 290 us with
// 256-byte stages, 301 with 128, 341 with rows in boxes of 64 and 16, 432 in
// boxes of 16), and gathered rows are copied into their order first
// (gather_kernel: no measurable cost there; by tile::gather4 927 us).
//
// Tried and not kept: L2 prefetches of the weights (297 us), row blocks of
// equal widths (no change: the pairs share what bounds them), two
// neighbouring columns a thread through tcgen05.ld.16x256b instead of lane
// exchanges (K 1536: 3% slower, its stores are half as long).
//
// Every wait is bounded; on a timeout the kernel sets the error word, waits
// for its copies in flight, releases TMEM and returns.
#include <atomic>

#include "../../include/qlinear_b200.h"
#include "bounded.cuh"

namespace qlin {
namespace {

constexpr int BM = 128;         // weight rows a CTA, 256 a pair
constexpr int BK = 128;         // bytes of K a stage
constexpr int BT = 256;         // rows of an expert a tile at most
constexpr int BOXES = 4;        // the activations' TMA boxes: 16, 32, 64 and 128 rows
constexpr int MAX_STAGES = 6;
constexpr int SLAB = BM * BK;   // 16 KB: a stage of either operand in one CTA
constexpr int EPI_WARPS = 8;    // two a quarter of the TMEM lanes (12 and 16 measured no gain)
constexpr int CHUNK = 16;       // columns an epilogue warp takes at a time (32: 3% slower at K 1536)
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
  int early;               // the kernel before this one is gather_kernel
  // Self-test: the stage, counted from 0, that both producers of a pair leave
  // out (stall_rank 2), or before which that of one CTA waits in vain; else -1.
  int stall, stall_rank;
};

struct Smem {  // behind the operand ring
  uint64_t full[MAX_STAGES], empty[MAX_STAGES], tfull[2], tempty[2], drain, never;
  uint32_t tmem_slot;
  int abort_flag;
  int other_fills;                   // stages that the other CTA's producer filled, once its loop has ended; -1 before
  int ready[2];                      // whether an accumulator was complete in time: what all epilogue threads go by
  alignas(16) float xs[2][BT];       // activation scales of a tile's rows
  int begin[MAX_EXPERTS + 1];        // first row of each expert, ascending within [0, R]
  int cum[MAX_EXPERTS + 1];          // tiles before each expert's
};
constexpr int SMEM_BYTES = 1024 + 2 * MAX_STAGES * SLAB + (int)sizeof(Smem);
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

// The smallest TMA box that holds a CTA's rows of the tile (the MMA reads no more of them).
__device__ __forceinline__ int box_of(const Tile& t) {
  int box = 0;
  while ((32 << box) < t.width) ++box;
  return box;
}

// *at = v in CTA `rank` of the cluster.
__device__ __forceinline__ void store_cluster(const int* at, uint32_t rank, int v) {
  asm volatile("st.relaxed.cluster.shared::cluster.u32 [%0], %1;" ::"r"(mapa_shared(smem_u32(at), rank)), "r"(v) : "memory");
}

__device__ __forceinline__ void epilogue_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(32 * EPI_WARPS) : "memory"); }

// 32 lanes x 16 columns of 32-bit TMEM -> 16 registers, waited for.
__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// Two values rounded to the 16-bit dtype, the first in the low half.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == DT_F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <int DT>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (DT == DT_F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// CHUNK columns (rows of the expert) of one accumulator: this thread has
// weight row n of all of them; out: element [first row, 0].  16-bit results
// are exchanged between neighbouring lanes so that a store writes two columns
// of one output row (a warp: two segments of 64 bytes).
template <int DT>
__device__ __forceinline__ void store_chunk(const uint32_t (&r)[CHUNK], const float* xs, float ws, float bias,
                                            bool has_bias, typename Elem<DT>::T* out, int64_t N, int rows, int n,
                                            int lane) {
  using EO = Elem<DT>;
  float y[CHUNK];
#pragma unroll
  for (int i = 0; i < CHUNK / 4; ++i) {
    const float4 x = reinterpret_cast<const float4*>(xs)[i];
    y[4 * i] = __fmul_rn(__fmul_rn(__int2float_rn((int)r[4 * i]), x.x), ws);
    y[4 * i + 1] = __fmul_rn(__fmul_rn(__int2float_rn((int)r[4 * i + 1]), x.y), ws);
    y[4 * i + 2] = __fmul_rn(__fmul_rn(__int2float_rn((int)r[4 * i + 2]), x.z), ws);
    y[4 * i + 3] = __fmul_rn(__fmul_rn(__int2float_rn((int)r[4 * i + 3]), x.w), ws);
  }
  if constexpr (DT == DT_F32) {
    if (n >= N) return;
#pragma unroll
    for (int j = 0; j < CHUNK; ++j)
      if (j < rows) out[j * N + n] = has_bias ? __fadd_rn(y[j], bias) : y[j];
  } else {
    uint32_t w[CHUNK / 2];  // rows 2i and 2i + 1
#pragma unroll
    for (int i = 0; i < CHUNK / 2; ++i) {
      w[i] = pack2<DT>(y[2 * i], y[2 * i + 1]);
      if (has_bias) {
        const float2 v = unpack2<DT>(w[i]);
        w[i] = pack2<DT>(__fadd_rn(v.x, bias), __fadd_rn(v.y, bias));
      }
    }
    if (N & 1) {  // output rows off a word: one value a store
      if (n >= N) return;
      uint16_t* o = reinterpret_cast<uint16_t*>(out) + n;
#pragma unroll
      for (int j = 0; j < CHUNK; ++j)
        if (j < rows) o[j * N] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
      return;
    }
    const int odd = lane & 1;
    uint32_t* o = reinterpret_cast<uint32_t*>(out) + odd * (N >> 1) + (n >> 1);
#pragma unroll
    for (int i = 0; i < CHUNK / 2; ++i) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, w[i], 1);
      const uint32_t v = odd ? __byte_perm(other, w[i], 0x7632) : __byte_perm(w[i], other, 0x5410);
      if (2 * i + odd < rows && n < N) *o = v;
      o += N;
    }
  }
}

struct RowMaps {
  CUtensorMap box[BOXES];  // the activations in boxes of 16 << i rows
};

// SL slabs of 128 bytes of K a stage: 2 where rows are whole slabs (one TMA
// box then covers both), else 1.
template <int DT, int SL>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    grouped_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ RowMaps tmX, GroupedParams p) {
  constexpr int STAGES = MAX_STAGES / SL;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sW = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sX = sW + MAX_STAGES * SLAB;
  Smem* s = reinterpret_cast<Smem*>(sX + MAX_STAGES * SLAB);
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
    mbar_init(&s->never, 1);
    *abort_flag = 0;
    s->other_fills = -1;
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
  // gather_kernel waits for the kernels before it, then lets this one start:
  // only the rows' order (a, a_scale) is still to come, and the weights are on
  // their way before it
  if (!p.early) pdl_wait();
  pdl_launch_dependents();

  // Row ranges and tile numbers of the experts, whatever the offsets hold.
  for (int e = threadIdx.x; e <= p.E; e += THREADS) s->begin[e] = min(max(p.offsets[e], 0), p.R);
  __syncthreads();
  const int num_n = (p.N + 2 * BM - 1) / (2 * BM);
  if (warp == 0)
    expert_bounds(s->begin, s->cum, p.E, lane, [=](int rows) { return (rows + BT - 1) / BT * num_n; });
  __syncthreads();
  const int num_tiles = s->cum[p.E];
  const int num_kb = (p.K + SL * BK - 1) / (SL * BK);
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (warp == 0) {
    // ---------------- producer (both CTAs) ----------------
    if (lane == 0) {
      tma_prefetch_desc(&tmW);
      for (int i = 0; i < BOXES; ++i) tma_prefetch_desc(&tmX.box[i]);
      int stage = 0, e = 0, fills = 0;
      uint32_t phase = 0;
      Armed armed;
      const int skip = p.stall_rank == 2 ? p.stall : -1, vain = p.stall_rank == (int)rank ? p.stall : -1;
      // After a wait that ran out, the stages that the other producer filled:
      // both end with as many, since the leader arms and awaits the loads of
      // both, and no load may outlive the kernel.
      int until = INT32_MAX;
      int ahead = 0;  // stages whose weights were asked for before the rows could be
      auto load_w = [&](int st, const Tile& t, int kb) {
        const uint32_t fb = mapa_shared(smem_u32(&s->full[st]), 0);
        if (leader) mbar_arrive_expect_tx(&s->full[st], 2 * SL * (SLAB + (16 << box_of(t)) * BK));
        const int row = t.e * p.N + t.n0 + (int)rank * BM;
        if constexpr (SL == 1) tma_load_2d_pair(sW + st * SLAB, &tmW, fb, kb * BK, row);
        else tma_load_3d_pair(sW + st * SL * SLAB, &tmW, fb, 0, row, kb * SL);
      };
      if (p.early) {
        int ea = 0;
        for (int tile = first; tile < num_tiles && ahead < STAGES; tile += step) {
          const Tile t = locate(s, tile, ea);
          for (int kb = 0; kb < num_kb && ahead < STAGES; ++kb) load_w(ahead++, t, kb);
        }
        pdl_wait();
      }
      for (int tile = first; tile < num_tiles && fills < until; tile += step) {
        const Tile t = locate(s, tile, e);
        const int xrow = t.row0 + (int)rank * (t.width >> 1);
        const CUtensorMap* tmx = &tmX.box[box_of(t)];
        for (int kb = 0; kb < num_kb; ++kb) {
          if (until == INT32_MAX && !(fills != vain ? wait_bounded(&s->empty[stage], phase ^ 1, abort_flag)
                                                    : wait_bounded(&s->never, 0, abort_flag))) {
            store_cluster(&s->other_fills, rank ^ 1, fills);
            store_cluster(&s->abort_flag, rank ^ 1, 1);
            until = max(fills, wait_value(&s->other_fills));
          }
          if (fills == until) break;
          // (behind a wait that ran out: the other CTA's producer saw the stage
          // empty, and one commit empties it in both)
          if (fills++ != skip) {
            if (ahead > 0) --ahead;
            else load_w(stage, t, kb);
            const uint32_t fb = mapa_shared(smem_u32(&s->full[stage]), 0);
            if constexpr (SL == 1) tma_load_2d_pair(sX + stage * SLAB, tmx, fb, kb * BK, xrow);
            else tma_load_3d_pair(sX + stage * SL * SLAB, tmx, fb, 0, xrow, kb * SL);
            armed.note(stage, phase);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (until == INT32_MAX) store_cluster(&s->other_fills, rank ^ 1, fills);
      // no load still writing shared memory at exit (both CTAs' loads are
      // counted by the leader; the peer waits for it at the last cluster barrier)
      if (leader) armed.drain(s->full);
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
        const uint32_t xslab = (16u << box_of(t)) * BK;  // from one slab of the rows to the next
        if (!wait_bounded(&s->tempty[acc], acc_phase ^ 1, abort_flag)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + acc * BT;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!wait_bounded(&s->full[stage], phase, abort_flag)) { ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < SL; ++h) {
            const uint64_t wdesc = umma_desc_k_sw128(smem_u32(sW + (stage * SL + h) * SLAB));
            const uint64_t xdesc = umma_desc_k_sw128(smem_u32(sX + stage * SL * SLAB) + h * xslab);
#pragma unroll
            for (int k = 0; k < BK / 32; ++k)
              umma_i8_pair(d, wdesc + 2 * k, xdesc + 2 * k, idesc, (kb | h | k) != 0 ? 1u : 0u);
          }
          issued = true;
          umma_commit_pair(&s->empty[stage], 0x3);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        umma_commit_pair(&s->tfull[acc], 0x3);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      // MMAs complete before TMEM is released, also when the epilogue gives up
      // after this loop has ended
      if (issued) {
        umma_commit_pair(&s->drain, 0x1);
        wait_drain(&s->drain, 0);
      }
    }
  } else {
    // ---------------- epilogue (both CTAs) ----------------
    using EO = Elem<DT>;
    using T = typename EO::T;
    const int tid = threadIdx.x - 64, quarter = warp & 3, part = (warp - 2) >> 2;
    if (p.early) pdl_wait();  // before anything is written, or a scale read
    {  // rows of no expert
      const int64_t line = (int64_t)p.N * sizeof(T);
      const int64_t thread = (int64_t)blockIdx.x * 32 * EPI_WARPS + tid, count = (int64_t)gridDim.x * 32 * EPI_WARPS;
      if (s->begin[0] > 0) zero_bytes(p.out, 0, s->begin[0] * line, thread, count);
      if (s->begin[p.E] < p.R) zero_bytes(p.out, s->begin[p.E] * line, p.R * line, thread, count);
    }
    int acc = 0, e = 0;
    uint32_t acc_phase = 0;
    const bool has_bias = p.bias != nullptr;
    // a tile's scales and bias, read while the tile before it is converted
    Tile t{};
    int n = 0;
    float ws = 0.0f, bias = 0.0f, xs = 0.0f;
    auto fetch = [&](int tile) {
      t = locate(s, tile, e);
      n = t.n0 + (int)rank * BM + quarter * 32 + lane;
      ws = bias = xs = 0.0f;
      if (n < p.N) {
        const int64_t at = (int64_t)t.e * p.N + n;
        ws = __ldg(p.w_scale + at);
        if (has_bias) bias = EO::to_f(reinterpret_cast<const T*>(p.bias)[at]);
      }
      if (tid < t.rows) xs = __ldg(p.a_scale + t.row0 + tid);
    };
    if (first < num_tiles) fetch(first);
    for (int tile = first; tile < num_tiles; tile += step) {
      const Tile now = t;
      const int col = n;
      const float wscale = ws, b = bias;
      if (tid < BT) s->xs[acc][tid] = xs;
      // one thread polls; the others sleep at the barrier
      if (tid == 0) s->ready[acc] = wait_bounded(&s->tfull[acc], acc_phase, abort_flag);
      epilogue_barrier();
      if (!s->ready[acc]) break;
      tc_fence_after();
      if (tile + step < num_tiles) fetch(tile + step);
      for (int c = part * CHUNK; c < now.rows; c += EPI_WARPS / 4 * CHUNK) {
        uint32_t r[CHUNK];
        tmem_ld_16(tmem_base + acc * BT + c + ((uint32_t)(quarter * 32) << 16), r);
        store_chunk<DT>(r, &s->xs[acc][c], wscale, b, has_bias,
                        reinterpret_cast<T*>(p.out) + (int64_t)(now.row0 + c) * p.N, p.N, now.rows - c, col, lane);
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

template <int DT, int SL>
int launch_dt(const CUtensorMap& tw, const RowMaps& tx, const GroupedParams& p, int clusters, cudaStream_t stream) {
  auto kern = grouped_kernel<DT, SL>;
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
                   int64_t R, int64_t N, int64_t K, void* workspace, cudaStream_t stream, int stall,
                   int stall_rank) {
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
  const int slabs = K % BK == 0 ? 2 : 1;
  int rc = encode_slab_tmap(&tw, w, (uint64_t)K, (uint64_t)(E * N), BK, BM, slabs);
  for (int i = 0; i < BOXES && !rc; ++i)
    rc = encode_slab_tmap(&tx.box[i], a, (uint64_t)K, (uint64_t)R, BK, 16 << i, slabs);
  if (rc) return rc;
  const GroupedParams p{a_scale, w_scale, offsets, (int)E, bias, out, (int)R, (int)N, (int)K,
                        a_rows != nullptr, stall, stall_rank};
  // tiles at most: every expert adds one partly filled row block to R / 256
  const int64_t tiles = (R / BT + (E < R ? E : R)) * ((N + 2 * BM - 1) / (2 * BM));
  const int clusters = (int)(tiles < sms / 2 ? tiles : sms / 2);
#define QLIN_GROUPED(DT)                                                                                   \
  return slabs == 2 ? launch_dt<DT, 2>(tw, tx, p, clusters, stream) : launch_dt<DT, 1>(tw, tx, p, clusters, stream)
  if (out_dt == DT_BF16) QLIN_GROUPED(DT_BF16);
  if (out_dt == DT_F16) QLIN_GROUPED(DT_F16);
  QLIN_GROUPED(DT_F32);
#undef QLIN_GROUPED
}

int set_grouped_wait_limit(uint64_t ns) { return set_tu_wait_limit(ns); }
int read_grouped_error(cudaStream_t stream, uint32_t* bits) { return read_tu_error(stream, bits); }

}  // namespace qlin
