// Matrix-vector products with packed 4-bit weights for few rows:
//   y[r, n] = dt(sum_g s[n, g] * (sum_{k in g} x[src(r), k] * q[n, k]) + bias[n])
// with signed nibbles q (low nibble = even k), float32 sums and one rounding.
// Unlike the W4A8 / W4A4 GEMMs the activations are not quantised.  With
// offsets [E + 1] the rows are sorted by expert and each uses its expert's
// weights.
//
// The weights' bytes bound it if a nibble costs next to nothing: at the HBM
// rate an SM receives 46 of them a clock.  As integers they cost 3/8 of an
// instruction each (a mask puts four into the high halves of four bytes, 16 q,
// without sign extension; as bf16 they take 11/8), so the activations become
// integers too, without losing theirs:
//
//   split_kernel   each 128 k of a row (a weight scale's group) as 32-bit
//                  integers X = x * 2^(29 - e), e the exponent of the largest
//                  of them, each in four signed base-256 digits.  A value down
//                  to 2^-6 (float32), 2^-19 (f16) or 2^-22 (bf16) of the
//                  largest is exact, a smaller one off by 2^-30 of the largest
//                  at most: less than a float32 sum of the 128 loses where the
//                  largest has a weight, and lost where its weight is 0;
//   matvec_kernel  mma.sync m16n8k32 (int8): 16 weight rows times 8 columns,
//                  the four digits of two rows.  The int32 sums of a block of
//                  128 are exact; their upper and lower two digits become a
//                  float32 each, meet the scale and are added up in float32.
//
// What bounds it: one row, N 24576, K 4096 (53.6 MB) takes 15.0 us: about 5 us
// of launches and latency, then 5.4 TB/s (N 98304 5.5 TB/s in all; a copy of the
// kernel that only loads 5.9).  With more rows the multiplying warps do, two to a
// scheduler that issue an instruction every four clocks or so (4 rows 18.4 us, 8
// rows 24.9); 16 of them, with half a stage each, are no faster, since what a
// warp does once a stage and a tile doubles.
//
// matvec_kernel is persistent, a block of threads a SM.  One warp brings the
// weights by TMA, 32 or 16 KB a stage of 32 rows or more (loads of 64 bytes a
// row straight into the lanes that need them stayed at 2 TB/s), one their
// scales, as many at a time as their alignment allows.  One brings an expert's
// activation digits, which stay in shared memory for all its row tiles.  Eight
// warps multiply, each 32 rows and one or two blocks of 128 k of a stage.  One
// adds their sums up, in a fixed order, while they go on.
#include <algorithm>
#include <atomic>

#include "../../include/qlinear_b200.h"
#include "bounded.cuh"

namespace qlin {
namespace {

constexpr int KB = 128;                // k of a block: one weight scale, one exponent
constexpr int WARPS = 8;               // that multiply
constexpr int THREADS = 32 * (WARPS + 4);
// Bytes of weights a stage, 2 or 1 blocks of 128 k a warp: with few columns
// the larger, whose fixed costs are half (the digits of eight rows leave no
// room for it).
template <int CB> constexpr int kStage = CB <= 2 ? 32768 : 16384;
// Buffers of partial sums between the multiplying warps and the one that adds them up.
template <int CB> constexpr int kParts = CB <= 2 ? 3 : 2;
constexpr int MAX_STAGES = 12;
// Room for a stage's weight scales, see scale_pitch.
template <int CB> constexpr int kScales = kStage<CB> / 32 * 3;
enum Scales { ROW, GROUP_F32, GROUP_BF16 };  // one a row (in the epilogue), or a row and block of 128 k
constexpr int MAX_EXPERTS = QLIN_MAX_EXPERTS;
constexpr int SMEM = 227 * 1024;

struct MatvecParams {
  const void* x;
  int64_t Rx, ldx;
  int64_t Rd;             // rows of digits: of the source rows, or of the result rows where they are fewer
  const uint8_t* w;       // [E, N, K / 2]
  const void* scale;      // [E, N, groups]
  int scale_bf16;
  int groups;             // scales a row: K / 128, or 1
  const int32_t* offsets; // [E + 1] or null (one expert, all rows)
  int E;
  const int32_t* x_rows;  // [R] or null
  const void* bias;       // [E, N] or null
  void* out;              // [R, N]
  int R, N, K;
  int blocks;             // of 128 k
  int early;              // the kernel before this one is split_kernel
  int own_digits;         // matvec_kernel makes the digits itself (one pass of one expert)
  int tile;               // weight rows a stage: 32 to 256
  int scale_copy;         // bytes of a copy of weight scales: 16, 8 or 4, 2 for plain loads
  int x_fours;            // rows of x begin at multiples of four values, and K is one
  int whole;              // a stage is one three-dimensional TMA box (rows are whole slabs of 128 bytes)
  int stages;
  int pass;               // rows of an expert whose digits fit, at most 2 * CB
  int stall_weights;      // self-test: the stage, counted from 0, that a block's producer leaves out; else -1
  int stall_scales;       // and the one at which the scales' warp waits in vain
  // of split_kernel, in the caller's workspace
  int8_t* digits;         // [Rd, blocks, half, digit, lane t, 16]
  float* exps;            // [Rd, epitch] 2^e, negative where the row has infinities or NaN
  int epitch;             // blocks rounded up to 4
};

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

__device__ __forceinline__ float scale_at(const MatvecParams& p, int64_t i) {
  return p.scale_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.scale)[i])
                      : __ldg(reinterpret_cast<const float*>(p.scale) + i);
}
// source row of result row r, or -1: a row of zeros
__device__ __forceinline__ int64_t source_row(const MatvecParams& p, int r) {
  const int64_t src = p.x_rows != nullptr ? (int64_t)p.x_rows[r] : r;
  return src >= 0 && src < p.Rx ? src : -1;
}

// where its digits are, or -1 as above
__device__ __forceinline__ int64_t digit_row(const MatvecParams& p, int r) {
  const int64_t src = source_row(p, r);
  return src < 0 || p.Rd == p.Rx ? src : r;
}

// ---------------------------------------------------------------------------
// activations -> digits
// ---------------------------------------------------------------------------

// Lane l of a warp has k 4l .. 4l + 3 of a block of 128.
template <int DT>
__device__ __forceinline__ void load_x4(const MatvecParams& p, int64_t src, int b, int lane, float (&v)[4]) {
  using T = typename Elem<DT>::T;
  struct alignas(4 * sizeof(T)) Four { T v[4]; };
  const int k = b * KB + 4 * lane;
  const T* x = reinterpret_cast<const T*>(p.x) + src * p.ldx + k;
  if (p.x_fours) {
    Four f;
    if (src >= 0 && k < p.K) f = *reinterpret_cast<const Four*>(x);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = src >= 0 && k < p.K ? Elem<DT>::to_f(f.v[i]) : 0.0f;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = src >= 0 && k + i < p.K ? Elem<DT>::to_f(x[i]) : 0.0f;
  }
}
// The digits of UN blocks to out[u] [half][digit][lane t][16 bytes], 2^e to
// *exp[u]; which of the blocks (bit u) have infinities or NaN (which add
// nothing here, see odd_terms).  The matrix instruction meets a word of eight
// nibbles as its even and its odd ones, so the digits of k 0 2 4 6 and of
// 1 3 5 7 of each eight lie together; lane t of the product reads words 4t ..
// 4t + 3 of a block, two at a time.
template <int UN>
__device__ __forceinline__ uint32_t make_digits(float (&v)[UN][4], int lane, void* const (&out)[UN],
                                                float* const (&exp)[UN]) {
  uint32_t big[UN], odd = 0;
#pragma unroll
  for (int u = 0; u < UN; ++u) {
    big[u] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t m = __float_as_uint(v[u][i]) & 0x7FFFFFFFu;
      if (m >= 0x7F800000u) {
        odd |= 1u << u;
        v[u][i] = 0.0f;
        m = 0;
      }
      big[u] = max(big[u], m);
    }
  }
#pragma unroll
  for (int u = 0; u < UN; ++u) big[u] = __reduce_max_sync(0xffffffffu, big[u]);
  const int word = lane >> 1;  // of eight k: the even lane stores its even ones, the odd lane its odd ones
  const int at = (word >> 1 & 1) * 256 + (word >> 2) * 16 + (word & 1) * 8 + (lane & 1) * 4;
  const uint32_t mine = lane & 1 ? 0x7531u : 0x6420u, theirs = lane & 1 ? 0x6420u : 0x7531u;
  const uint32_t low = lane & 1 ? 0x1054u : 0x5410u, high = lane & 1 ? 0x3276u : 0x7632u;
#pragma unroll
  for (int u = 0; u < UN; ++u) {
    const int e = max((int)(big[u] >> 23), 1) - 127;  // |x| < 2^(e + 1)
    // 2^(29 - e) in two factors, each a float
    const float f1 = pow2((29 - e) >> 1), f2 = pow2(29 - e - ((29 - e) >> 1));
    uint32_t d[4];  // a k's signed digits: X + 128 (1 + 256 + 65536) has them 128 up as its bytes
#pragma unroll
    for (int i = 0; i < 4; ++i)
      d[i] = (uint32_t)(__float2int_rn(__fmul_rn(__fmul_rn(v[u][i], f1), f2)) + 0x00808080) ^ 0x00808080u;
    const uint32_t a = __byte_perm(d[0], d[1], 0x5140), b = __byte_perm(d[2], d[3], 0x5140);
    const uint32_t c = __byte_perm(d[0], d[1], 0x7362), f = __byte_perm(d[2], d[3], 0x7362);
    const uint32_t q[4] = {__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(c, f, 0x5410),
                           __byte_perm(c, f, 0x7632)};  // digit q of the four k
    uint32_t* to = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(out[u]) + at);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {  // two digits an exchange
      const uint32_t keep = __byte_perm(q[i], q[i + 1], mine);
      const uint32_t other = __shfl_xor_sync(0xffffffffu, __byte_perm(q[i], q[i + 1], theirs), 1);
      to[i * 16] = __byte_perm(keep, other, low);
      to[(i + 1) * 16] = __byte_perm(keep, other, high);
    }
    if (lane == 0) *exp[u] = pow2(e);
  }
  return __reduce_or_sync(0xffffffffu, odd);
}

// One block a row, a warp 128 k at a time.
template <int DT>
__global__ void __launch_bounds__(1024) split_kernel(MatvecParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t r = blockIdx.x, src = p.Rd == p.Rx ? r : source_row(p, (int)r);
  bool odd = false;
  for (int b = warp; b < p.blocks; b += blockDim.x >> 5) {
    float v[1][4];
    load_x4<DT>(p, src, b, lane, v[0]);
    odd |= make_digits<1>(v, lane, {p.digits + (r * p.blocks + b) * (4 * KB)}, {p.exps + r * p.epitch + b}) != 0;
  }
  if (__syncthreads_or(odd))
    for (int b = threadIdx.x; b < p.blocks; b += blockDim.x) p.exps[r * p.epitch + b] *= -1.0f;
}

// What the infinities and NaN of a row add to one output.
template <int DT>
__device__ float odd_terms(const MatvecParams& p, int64_t src, int64_t row) {
  const typename Elem<DT>::T* x = reinterpret_cast<const typename Elem<DT>::T*>(p.x) + src * p.ldx;
  float v = 0.0f;
  for (int k = 0; k < p.K; ++k) {
    const float f = Elem<DT>::to_f(x[k]);
    if (fabsf(f) <= 3.402823466e38f) continue;
    const int c = p.w[row * (p.K >> 1) + (k >> 1)] >> (4 * (k & 1)) & 15;
    v += __fmul_rn(f, __fmul_rn((float)((c ^ 8) - 8), p.groups > 1 ? scale_at(p, row * p.groups + k / KB) : 1.0f));
  }
  return v;
}

// ---------------------------------------------------------------------------
// digits x weights
// ---------------------------------------------------------------------------

__device__ __forceinline__ void mma16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct Smem {  // behind the ring, the digits, the partial sums and the scales
  uint64_t full[MAX_STAGES], empty[MAX_STAGES], pfull[3], pempty[3], xfull, xempty, never;
  int abort_flag;
  int fills;                   // stages the producer filled, once it has left its loop; -1 before
  uint32_t odd;                // own_digits: rows with infinities or NaN
  int first_items, first_pass, first_n0;  // this block of threads' items: how many, and where they begin
  int begin[MAX_EXPERTS + 1];  // first row of each expert, ascending within [0, R]
  int cum[MAX_EXPERTS + 1];    // passes before each expert's
};

// An item of work: one row tile of one pass (up to p.pass rows of an expert).
// Items are numbered pass by pass, and a block of threads has consecutive
// ones, so that it changes its digits seldom.
struct Item {
  int left;                // items of this block from here on
  int pass, e, r0, rows, n0;
  __device__ __forceinline__ void find(const MatvecParams& p, const Smem* s) {
    while (s->cum[e + 1] <= pass) ++e;  // passes ascend
    const int r = (pass - s->cum[e]) * p.pass;
    r0 = s->begin[e] + r;
    rows = min(p.pass, s->begin[e + 1] - r0);
  }
  // Once a block of threads: the divisions took each warp a microsecond.
  static __device__ __forceinline__ void share_out(const MatvecParams& p, Smem* s) {
    const uint32_t tiles = (uint32_t)(p.N + p.tile - 1) / (uint32_t)p.tile, items = (uint32_t)s->cum[p.E] * tiles;
    const uint32_t each = items / gridDim.x, more = items - each * gridDim.x;  // (items fit an int: see launch_cfg)
    const uint32_t first = blockIdx.x * each + min(blockIdx.x, more), pass = first / tiles;
    s->first_items = (int)(each + (blockIdx.x < more));
    s->first_pass = (int)pass;
    s->first_n0 = (int)(first - pass * tiles) * p.tile;
  }
  __device__ __forceinline__ void start(const MatvecParams& p, const Smem* s) {
    left = s->first_items;
    pass = s->first_pass;
    n0 = s->first_n0;
    e = 0;
    if (left > 0) find(p, s);
  }
  __device__ __forceinline__ void next(const MatvecParams& p, const Smem* s) {
    --left;
    n0 += p.tile;
    if (n0 >= p.N) {
      n0 = 0;
      ++pass;
      if (left > 0) find(p, s);
    }
  }
};

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
// The barrier counts this thread once its copies are complete.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Bytes from one row's weight scales of a stage to the next row's: the eight
// rows that a warp reads at once lie in different banks.  tile * pitch is at
// most 3072 with 32 KB of weights a stage, half of that with 16.
__host__ __device__ constexpr int scale_pitch(int bytes) { return bytes > 16 ? bytes + 16 : bytes; }

__device__ __forceinline__ void tma_load_3d(void* dst, const void* tmap, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Everything read before pdl_wait was complete before split_kernel let this
// kernel start (it waits for the kernels before it first).
// CB: blocks of 8 columns, two rows each.
template <int DT, int CB, Scales SC>
__global__ void __launch_bounds__(THREADS, 1) matvec_kernel(const __grid_constant__ CUtensorMap tmW, MatvecParams p) {
  using T = typename Elem<DT>::T;
  constexpr int STAGE = kStage<CB>, BLK = STAGE / 16384;  // blocks of 128 k a warp and stage
  constexpr int PARTS = kParts<CB>;
  constexpr int PITCH = 2 * CB + 1;                       // of a warp's partial sums [32 rows][PITCH]
  constexpr int PART = 32 * PITCH;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* xdig = ring + p.stages * STAGE;                            // [pass][blocks][512]
  float* xexp = reinterpret_cast<float*>(xdig + (int64_t)p.pass * p.blocks * (4 * KB));  // [pass][epitch]
  float* part = xexp + p.pass * p.epitch;                             // [PARTS][WARPS][PART]
  constexpr bool GROUPS = SC != ROW;
  constexpr int SB = SC == GROUP_BF16 ? 2 : 4;                        // bytes of a scale
  uint8_t* scales = reinterpret_cast<uint8_t*>(part + PARTS * WARPS * PART);  // [stages][kScales]
  Smem* s = reinterpret_cast<Smem*>(scales + (GROUPS ? p.stages * kScales<CB> : 0));
  volatile int* abort_flag = &s->abort_flag;
  volatile int* fills_at_end = &s->fills;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&s->full[i], GROUPS ? 33 : 1);
      mbar_init(&s->empty[i], WARPS);
    }
    for (int i = 0; i < PARTS; ++i) {
      mbar_init(&s->pfull[i], WARPS);
      mbar_init(&s->pempty[i], 1);
    }
    mbar_init(&s->xfull, p.own_digits ? WARPS : 1);
    mbar_init(&s->xempty, WARPS + 1);
    mbar_init(&s->never, 1);
    *abort_flag = 0;
    *fills_at_end = -1;
    s->odd = 0u;
    fence_mbar_init();
  }
  pdl_launch_dependents();
  if (!p.early) pdl_wait();
  struct alignas(4 * sizeof(T)) Four { T v[4]; };  // a lane's values of a block
  if (p.own_digits && warp < WARPS) {
    // The values, where their digits will be, asked for before the first
    // weights: behind those a load waits until the ring is full (2 us).
#pragma unroll 1
    for (int i = warp; i < p.R * p.blocks; i += WARPS) {
      const int r = i / p.blocks, k = (i - r * p.blocks) * KB + 4 * lane;
      const int64_t src = source_row(p, r);
      const T* from = reinterpret_cast<const T*>(p.x) + src * p.ldx + k;
      Four* to = reinterpret_cast<Four*>(xdig + (int64_t)i * (4 * KB)) + lane;
      if (p.x_fours && src >= 0 && k < p.K) {
        cp_async<4 * sizeof(T)>(smem_u32(to), from);
      } else {
        for (int j = 0; j < 4; ++j) to->v[j] = src >= 0 && k + j < p.K ? from[j] : Elem<DT>::from_f(0.0f);
      }
    }
  }
  if (p.offsets != nullptr) {
    for (int e = threadIdx.x; e <= p.E; e += THREADS) s->begin[e] = min(max(p.offsets[e], 0), p.R);
  } else if (threadIdx.x < 2) {
    s->begin[threadIdx.x] = threadIdx.x ? p.R : 0;
  }
  __syncthreads();
  if (warp == 0) {
    expert_bounds(s->begin, s->cum, p.E, lane, [&](int rows) { return (rows + p.pass - 1) / p.pass; });
    __syncwarp();
    if (lane == 0) Item::share_out(p, s);
  }
  __syncthreads();
  const int slabs = STAGE / (128 * p.tile);                    // of 128 bytes a row and stage
  const int steps = (p.blocks + 2 * slabs - 1) / (2 * slabs);  // stages of a tile
  const int row_groups = p.tile >> 5;                          // of 32 rows
  const int share = WARPS / row_groups;                        // warps of a row group

  if (warp == WARPS) {
    // ---------------- weights ----------------
    if (lane == 0) {
      tma_prefetch_desc(&tmW);
      int stage = 0, fills = 0;
      uint32_t phase = 0;
      Armed armed;
      bool ok = true;
      Item it;
      for (it.start(p, s); it.left > 0 && ok; it.next(p, s)) {
        const int row = it.e * p.N + it.n0;
        for (int st = 0; st < steps; ++st) {
          if (!wait_bounded(&s->empty[stage], phase ^ 1, abort_flag)) { ok = false; break; }
          if (fills++ != p.stall_weights) {
            mbar_arrive_expect_tx(&s->full[stage], STAGE);
            uint8_t* d = ring + stage * STAGE;
            if (p.whole) {
              tma_load_3d(d, &tmW, &s->full[stage], 0, row, st * slabs);
            } else {
              for (int i = 0; i < slabs; ++i)  // (behind K: zeros)
                tma_load_2d(d + i * 128 * p.tile, &tmW, &s->full[stage], (st * slabs + i) * 128, row);
            }
            armed.note(stage, phase);
          }
          if (++stage == p.stages) { stage = 0; phase ^= 1; }
        }
      }
      *fills_at_end = fills;
      armed.drain(s->full);  // no load still writing shared memory at exit
    }
  } else if (warp == WARPS + 1) {
    // ---------------- digits and exponents of a pass's rows ----------------
    if (p.early) pdl_wait();
    int now = -1;
    uint32_t loads = 0;
    Item it;
    for (it.start(p, s); it.left > 0 && !p.own_digits; it.next(p, s)) {
      if (it.pass == now) continue;
      now = it.pass;
      bool ok = true;
      if (lane == 0 && loads > 0) ok = wait_bounded(&s->xempty, (loads - 1) & 1, abort_flag);
      if (!__shfl_sync(0xffffffffu, (int)ok, 0)) break;
      const int64_t src = lane < it.rows ? digit_row(p, it.r0 + lane) : -1;
      const uint32_t live = __ballot_sync(0xffffffffu, src >= 0);
      if (lane < it.rows && src < 0) {  // a row of zeros: whatever its digits are
        for (int i = 0; i < p.epitch; ++i) xexp[lane * p.epitch + i] = 0.0f;
        fence_proxy_async_smem();  // a later pass's bulk copy writes here
      }
      __syncwarp();
      const uint32_t dbytes = (uint32_t)p.blocks * (4 * KB), ebytes = (uint32_t)p.epitch * 4;
      if (lane == 0) mbar_arrive_expect_tx(&s->xfull, (uint32_t)__popc(live) * (dbytes + ebytes));
      __syncwarp();
      if (src >= 0) {
        bulk_load(xdig + (int64_t)lane * dbytes, p.digits + src * dbytes, dbytes, &s->xfull);
        bulk_load(xexp + lane * p.epitch, p.exps + src * p.epitch, ebytes, &s->xfull);
      }
      ++loads;
    }
    if (lane == 0 && loads > 0) wait_drain(&s->xfull, (loads - 1) & 1);
  } else if (warp == WARPS + 3) {
    // ---------------- weight scales ----------------
    // Of a stage's rows in turn, a lane each.  (In the multiplying warps, one
    // word a row and block, these copies took a sixth of their time and a
    // quarter of the shared-memory cycles.)
    if constexpr (GROUPS) {
      const int per = 2 * slabs, bytes = per * SB, pitch = scale_pitch(bytes);
      int stage = 0, fills = 0;
      uint32_t phase = 0;
      bool ok = true;
      Item it;
      for (it.start(p, s); it.left > 0 && ok; it.next(p, s))
        for (int st = 0; st < steps; ++st) {
          if (!wait_bounded_warp(fills != p.stall_scales ? &s->empty[stage] : &s->never,
                                 fills != p.stall_scales ? phase ^ 1 : 0, abort_flag)) {
            ok = false;
            break;
          }
          const int here = min(per, p.blocks - st * per) * SB;  // (behind K: whatever is there)
          for (int r = lane; r < p.tile; r += 32) {
            const int64_t first = ((int64_t)it.e * p.N + min(it.n0 + r, p.N - 1)) * p.groups + st * per;
            const uint8_t* from = static_cast<const uint8_t*>(p.scale) + first * SB;
            uint8_t* to = scales + stage * kScales<CB> + r * pitch;
            if (p.scale_copy == 16) {
              for (int i = 0; i < here; i += 16) cp_async<16>(smem_u32(to + i), from + i);
            } else if (p.scale_copy == 8) {
              for (int i = 0; i < here; i += 8) cp_async<8>(smem_u32(to + i), from + i);
            } else if (p.scale_copy == 4) {
              for (int i = 0; i < here; i += 4) cp_async<4>(smem_u32(to + i), from + i);
            } else {
              for (int i = 0; i < here; i += 2)
                *reinterpret_cast<uint16_t*>(to + i) = __ldg(reinterpret_cast<const uint16_t*>(from + i));
            }
          }
          if (p.scale_copy > 2) cp_async_arrive(&s->full[stage]);
          else mbar_arrive(&s->full[stage]);
          ++fills;
          if (++stage == p.stages) { stage = 0; phase ^= 1; }
        }
      if (!ok) {
        // The producer waits for its loads at the barriers that this warp
        // arrives at too: it gets the arrivals of the stages filled since.
        for (const int n = wait_value(fills_at_end); fills < n; ++fills) {
          mbar_arrive(&s->full[stage]);
          if (++stage == p.stages) stage = 0;
        }
      }
      cp_async_wait_all();  // no copy still writing shared memory at exit
    }
  } else if (warp == WARPS + 2) {
    // ---------------- outputs ----------------
    if (p.early) pdl_wait();  // before anything is written
    {  // rows of no expert
      const int64_t line = (int64_t)p.N * sizeof(T);
      const int64_t thread = (int64_t)blockIdx.x * 32 + lane, count = (int64_t)gridDim.x * 32;
      if (s->begin[0] > 0) zero_bytes(p.out, 0, s->begin[0] * line, thread, count);
      if (s->begin[p.E] < p.R) zero_bytes(p.out, s->begin[p.E] * line, p.R * line, thread, count);
    }
    // bias and scale of this lane's column of each 32 of an item, read while the
    // sums of the one before it are added up
    constexpr int MAXG = 8;
    T next_bias[MAXG];
    float next_scale[MAXG];
    Item ahead;
    ahead.start(p, s);
    auto fetch = [&]() {
#pragma unroll
      for (int j = 0; j < MAXG; ++j)
        if (j < row_groups && ahead.left > 0) {
          const int64_t at = (int64_t)ahead.e * p.N + min(ahead.n0 + 32 * j + lane, p.N - 1);
          if (p.bias != nullptr) next_bias[j] = reinterpret_cast<const T*>(p.bias)[at];
          if constexpr (!GROUPS) next_scale[j] = scale_at(p, at);
        }
    };
    fetch();
    int buf = 0, now = -1;
    uint32_t phase = 0, odd = 0;  // rows of the pass with infinities or NaN
    while (ahead.left > 0) {
      const Item it = ahead;
      float bias[MAXG], row_scale[MAXG];
#pragma unroll
      for (int j = 0; j < MAXG; ++j) {
        bias[j] = p.bias != nullptr && j < row_groups ? Elem<DT>::to_f(next_bias[j]) : 0.0f;
        row_scale[j] = next_scale[j];
      }
      ahead.next(p, s);
      fetch();
      if (!wait_bounded_warp(&s->pfull[buf], phase, abort_flag)) break;
      if (it.pass != now) {
        now = it.pass;
        odd = s->odd | __ballot_sync(0xffffffffu, lane < it.rows && xexp[min(lane, it.rows - 1) * p.epitch] < 0.0f);
        if (lane == 0) mbar_arrive(&s->xempty);  // done with the exponents
      }
#pragma unroll
      for (int j = 0; j < MAXG; ++j) {
        const int n = it.n0 + 32 * j + lane;
        if (j < row_groups && n < p.N) {
          const int64_t at = (int64_t)it.e * p.N + n;
#pragma unroll
          for (int r = 0; r < 2 * CB; ++r) {
            if (r >= it.rows) break;
            const float* q = part + (buf * WARPS + j) * PART + lane * PITCH + r;
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < WARPS; ++k)
              if (k < share) v += q[k * row_groups * PART];
            if (odd >> r & 1u) v += odd_terms<DT>(p, source_row(p, it.r0 + r), at);
            if constexpr (!GROUPS) v *= row_scale[j];
            if (p.bias != nullptr) v += bias[j];
            reinterpret_cast<T*>(p.out)[(int64_t)(it.r0 + r) * p.N + n] = Elem<DT>::from_f(v);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s->pempty[buf]);
      if (++buf == PARTS) { buf = 0; phase ^= 1; }
    }
  } else {
    // ---------------- products ----------------
    const int g = lane >> 2, t = lane & 3;
    const int rg = warp & (row_groups - 1);           // this warp's row group,
    const int bi = warp / row_groups * BLK;           // and its first block of a stage
    // lane group g has rows r = g/2 + 4 (g%2) and r + 8 of each 16: rows 4
    // apart lie in different halves of the 128-byte swizzle's banks
    const int row = (g >> 1) + 4 * (g & 1);
    uint32_t woff[BLK];
#pragma unroll
    for (int k = 0; k < BLK; ++k)
      woff[k] = (uint32_t)(((bi + k) >> 1) * 128 * p.tile + (rg * 32 + row) * 128 + (((((bi + k) & 1) * 4 + t) ^ row) * 16));
    // 16 q times digit d of X = x 2^(29 - e): lanes of odd t have the upper two digits
    const float unit = (t & 1) ? pow2(16 - 33) : pow2(-33);
    // rows behind the last of a pass repeat it (their sums are not stored)
    auto xrow = [&](int c, int odd_half, int rows) { return min(2 * c + odd_half, rows - 1); };

    const int pitch = scale_pitch(2 * slabs * SB);
    const uint8_t* my_scales = scales + (rg * 32 + row) * pitch + bi * SB;  // of row `row`; the others are 8 pitches apart
    if (p.own_digits) {
      cp_async_wait_all();
      __syncwarp();
#pragma unroll 1  // (code that runs once waits for its instructions)
      for (int i = warp; i < p.R * p.blocks; i += WARPS) {
        const int r = i / p.blocks;
        uint8_t* block = xdig + (int64_t)i * (4 * KB);
        const Four f = reinterpret_cast<const Four*>(block)[lane];
        float v[1][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[0][j] = Elem<DT>::to_f(f.v[j]);
        __syncwarp();  // read by all before the digits take their place
        if (make_digits<1>(v, lane, {block}, {xexp + r * p.epitch + i - r * p.blocks}) && lane == 0)
          atomicOr(&s->odd, 1u << r);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s->xfull);
    }
    int stage = 0, now = -1, buf = 0;
    uint32_t phase = 0, loads = 0, pphase = 0;
    // 0 once a wait of this lane ran out: it then goes on with whatever the
    // stages hold, so that all lanes meet below, and the warp's verdict is taken
    // once an item.  Bit 0: lane 0, which arrives for the warp.  (8 rows of N
    // 24576, K 4096: 24.8 us, with a vote a stage 26.0.)
    int arrives = lane == 0 ? 3 : 2;
    Item it;
    for (it.start(p, s); it.left > 0; it.next(p, s)) {
      if (it.pass != now) {
        if (now >= 0) {  // this warp is done with the digits of the pass before
          __syncwarp();
          if (lane == 0) mbar_arrive(&s->xempty);
        }
        now = it.pass;
        if (!wait_bounded(&s->xfull, loads & 1, abort_flag)) arrives = 0;
        ++loads;
      }
      const uint8_t* xd[CB];
      const float* xe[CB];
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        xd[c] = xdig + (int64_t)xrow(c, g >> 2, it.rows) * p.blocks * (4 * KB) + (g & 3) * 64 + t * 16;
        xe[c] = xexp + xrow(c, t >> 1, it.rows) * p.epitch;
      }
      float sum[2][CB][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < CB; ++c) sum[i][c][0] = sum[i][c][1] = 0.0f;
#pragma unroll 1
      for (int st = 0; st < steps; ++st) {
        const int b0 = st * 2 * slabs + bi;
        if (!wait_bounded(&s->full[stage], phase, abort_flag)) arrives = 0;
#pragma unroll
        for (int k = 0; k < BLK; ++k) {
          // Behind K the weights are 0, and the last block's digits and exponent
          // serve; a branch here would keep the two blocks of a warp one behind
          // the other.
          const int b = min(b0 + k, p.blocks - 1);
          float ws[2][2] = {{1.0f, 1.0f}, {1.0f, 1.0f}};
          if constexpr (GROUPS) {
            const uint8_t* from = my_scales + stage * kScales<CB> + k * SB;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint8_t* f = from + 8 * j * pitch;
              const float v = SC == GROUP_BF16 ? __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(f) << 16)
                                               : *reinterpret_cast<const float*>(f);
              ws[j >> 1][j & 1] = b0 + k < p.blocks ? v : 0.0f;
            }
          }
          const uint8_t* d = ring + stage * STAGE + woff[k];
          uint4 w[2][2];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) w[i][h] = *reinterpret_cast<const uint4*>(d + (16 * i + 8 * h) * 128);
          int acc[2][CB][4];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int c = 0; c < CB; ++c)
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[i][c][j] = 0;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint4 xv[CB];
#pragma unroll
            for (int c = 0; c < CB; ++c) xv[c] = *reinterpret_cast<const uint4*>(xd[c] + b * (4 * KB) + half * 256);
#pragma unroll
            for (int q = 0; q < 2; ++q) {  // a word of eight k a lane
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint32_t a[2][2];  // [row half][even, odd k]: 16 times the nibble
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const uint32_t u = half == 0 ? (q == 0 ? w[i][h].x : w[i][h].y) : (q == 0 ? w[i][h].z : w[i][h].w);
                  a[h][0] = (u << 4) & 0xF0F0F0F0u;
                  a[h][1] = u & 0xF0F0F0F0u;
                }
#pragma unroll
                for (int c = 0; c < CB; ++c)
                  mma16832(acc[i][c], a[0][0], a[1][0], a[0][1], a[1][1], q ? xv[c].z : xv[c].x, q ? xv[c].w : xv[c].y);
              }
            }
          }
#pragma unroll
          for (int c = 0; c < CB; ++c) {
            const float xs = fabsf(xe[c][b]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                // |digit sums| <= 128 * 128 * 128: both digits fit an int (the
                // unit goes to the sum, where it is exact however small the scale)
                const float v = __fmul_rn(__int2float_rn(acc[i][c][2 * h] + 256 * acc[i][c][2 * h + 1]), unit);
                sum[i][c][h] = __fmaf_rn(GROUPS ? __fmul_rn(v, ws[i][h]) : v, xs, sum[i][c][h]);
              }
          }
        }
        __syncwarp();
        if (arrives & 1) mbar_arrive(&s->empty[stage]);
        if (++stage == p.stages) { stage = 0; phase ^= 1; }
      }
      if (!wait_bounded(&s->pempty[buf], pphase ^ 1, abort_flag)) arrives = 0;
      if (!__all_sync(0xffffffffu, arrives)) break;
      float* to = part + (buf * WARPS + warp) * PART;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < CB; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float v = sum[i][c][h] + __shfl_xor_sync(0xffffffffu, sum[i][c][h], 1);
            if (!(t & 1)) to[(16 * i + 8 * h + row) * PITCH + 2 * c + (t >> 1)] = v;
          }
      __syncwarp();
      if (lane == 0) mbar_arrive(&s->pfull[buf]);
      if (++buf == PARTS) { buf = 0; pphase ^= 1; }
    }
  }
}

// The same for any K and alignment, digits and weights straight from memory: a
// block of threads 16 weight rows and 2 * CB rows of one expert at a time (grid.y:
// the experts that have rows, one after another), each warp every eighth block
// of K.  A lane reads its 16 bytes of a weight row as the aligned words that
// hold them, one block ahead.
template <int DT, int CB, bool GROUPS>
__global__ void __launch_bounds__(32 * WARPS) matvec_any_kernel(MatvecParams p) {
  using T = typename Elem<DT>::T;
  __shared__ int s_begin[MAX_EXPERTS + 1], s_cum[MAX_EXPERTS + 1];
  __shared__ float s_part[WARPS][16][2 * CB + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_wait();
  pdl_launch_dependents();
  if (p.offsets != nullptr) {
    for (int e = threadIdx.x; e <= p.E; e += 32 * WARPS) s_begin[e] = min(max(p.offsets[e], 0), p.R);
  } else if (threadIdx.x < 2) {
    s_begin[threadIdx.x] = threadIdx.x ? p.R : 0;
  }
  __syncthreads();
  if (warp == 0) expert_bounds(s_begin, s_cum, p.E, lane, [](int rows) { return rows > 0; });
  __syncthreads();
  {
    const int64_t line = (int64_t)p.N * sizeof(T), block = blockIdx.y * (int64_t)gridDim.x + blockIdx.x;
    const int64_t thread = block * 32 * WARPS + threadIdx.x, count = (int64_t)gridDim.x * gridDim.y * 32 * WARPS;
    if (s_begin[0] > 0) zero_bytes(p.out, 0, s_begin[0] * line, thread, count);
    if (s_begin[p.E] < p.R) zero_bytes(p.out, s_begin[p.E] * line, p.R * line, thread, count);
  }
  if ((int)blockIdx.y >= s_cum[p.E]) return;
  int e = 0;
  while (s_cum[e + 1] <= (int)blockIdx.y) ++e;
  const int n0 = blockIdx.x * 16, bytes = p.K >> 1;
  const float unit = (t & 1) ? pow2(16 - 33) : pow2(-33);
  const uint32_t* words[2];  // of the row, and where in the first one it begins and in which it ends
  int shift[2], last[2];
  int64_t wrow[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    wrow[h] = (int64_t)e * p.N + min(n0 + 8 * h + g, p.N - 1);
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.w + wrow[h] * bytes);
    words[h] = reinterpret_cast<const uint32_t*>(at & ~uintptr_t(3));
    shift[h] = 8 * (int)(at & 3);
    last[h] = (int)((at & 3) + bytes - 1) >> 2;
  }
  auto load = [&](int b, uint32_t (&u)[2][5]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        const int at = b * (KB / 8) + 4 * t + i;
        u[h][i] = b < p.blocks && at <= last[h] ? __ldg(words[h] + at) : 0u;  // (behind K the digits are 0)
      }
  };
  for (int r0 = s_begin[e]; r0 < s_begin[e + 1]; r0 += 2 * CB) {
    const int rows = min(2 * CB, s_begin[e + 1] - r0);
    int64_t src[CB], sum_src[CB];  // the rows whose digits this lane reads, whose sums it gets
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      src[c] = digit_row(p, r0 + min(2 * c + (g >> 2), rows - 1));
      sum_src[c] = digit_row(p, r0 + min(2 * c + (t >> 1), rows - 1));
    }
    float sum[CB][2];
#pragma unroll
    for (int c = 0; c < CB; ++c) sum[c][0] = sum[c][1] = 0.0f;
    uint32_t next[2][5];
    load(warp, next);
    for (int b = warp; b < p.blocks; b += WARPS) {
      uint32_t a[4][2][2];  // [word][row half][even, odd k]: 16 times the nibble
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w = __funnelshift_r(next[h][q], next[h][q + 1], shift[h]);
          a[q][h][0] = (w << 4) & 0xF0F0F0F0u;
          a[q][h][1] = w & 0xF0F0F0F0u;
        }
      load(b + WARPS, next);
      float ws[2] = {1.0f, 1.0f};
      if constexpr (GROUPS) {
        ws[0] = scale_at(p, wrow[0] * p.groups + b);
        ws[1] = scale_at(p, wrow[1] * p.groups + b);
      }
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        uint4 d[2];
        d[0] = d[1] = make_uint4(0u, 0u, 0u, 0u);
        if (src[c] >= 0) {
          const int8_t* from = p.digits + (src[c] * p.blocks + b) * (4 * KB) + (g & 3) * 64 + t * 16;
          d[0] = *reinterpret_cast<const uint4*>(from);
          d[1] = *reinterpret_cast<const uint4*>(from + 256);
        }
        int acc[4] = {0, 0, 0, 0};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint4& v = d[q >> 1];
          mma16832(acc, a[q][0][0], a[q][1][0], a[q][0][1], a[q][1][1], (q & 1) ? v.z : v.x, (q & 1) ? v.w : v.y);
        }
        const float xs = sum_src[c] >= 0 ? fabsf(p.exps[sum_src[c] * p.epitch + b]) : 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float v = __fmul_rn(__int2float_rn(acc[2 * h] + 256 * acc[2 * h + 1]), unit);
          sum[c][h] = __fmaf_rn(GROUPS ? __fmul_rn(v, ws[h]) : v, xs, sum[c][h]);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float v = sum[c][h] + __shfl_xor_sync(0xffffffffu, sum[c][h], 1);
        if (!(t & 1)) s_part[warp][8 * h + g][2 * c + (t >> 1)] = v;
      }
    __syncthreads();
    const int n = n0 + (threadIdx.x & 15), r = threadIdx.x >> 4;
    if (r < rows && n < p.N) {
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) v += s_part[k][threadIdx.x & 15][r];
      const int64_t at = (int64_t)e * p.N + n, from = digit_row(p, r0 + r);
      if (from >= 0 && p.exps[from * p.epitch] < 0.0f) v += odd_terms<DT>(p, source_row(p, r0 + r), at);
      if constexpr (!GROUPS) v *= scale_at(p, at);
      if (p.bias != nullptr) v += Elem<DT>::to_f(reinterpret_cast<const T*>(p.bias)[at]);
      reinterpret_cast<T*>(p.out)[(int64_t)(r0 + r) * p.N + n] = Elem<DT>::from_f(v);
    }
    __syncthreads();
  }
}

// Few values: every block of threads makes the digits itself, which saves a
// launch and a workspace: a call takes 12.8 us instead of 17.4.  On the device
// (bf16, us; with split_kernel) one row gains: N 24576, K 4096 15.5 (16.3), N
// 8192, K 8192 11.4 (11.8); two rows are even: N 8192, K 4096 9.5 (9.3); more
// rows lose, which a replayed graph pays: 4 of N 8192, K 2048 9.7 (8.9), 5 of N
// 1111, K 1440 8.8 (7.2), 8 of N 8192, K 1024 10.9 (9.5).  With more values, 4
// rows of K 4096, the device loses 3 to 4 us, nearly what the call gains.
bool makes_own_digits(bool experts, int64_t R, int64_t K) { return !experts && R <= 8 && R * K <= 8192; }

template <int CB>
constexpr int fixed_bytes() {
  return 1024 + kParts<CB> * WARPS * 32 * (2 * CB + 1) * 4 + (int)sizeof(Smem);
}
// Bytes of a pass's digits and exponents that every instance has room for, beside 64 KB of weights.
constexpr int64_t kDigitRoom =
    SMEM - 65536 - 4 * 1536 - std::max({fixed_bytes<1>(), fixed_bytes<2>(), fixed_bytes<4>()});

template <int DT, int CB, Scales SC>
int launch_cfg(MatvecParams p, cudaStream_t stream) {
  const int sms = device_sm_count();
  // rows a pass: what fits beside 64 KB of weights; then as many stages as fit
  constexpr int STAGE = kStage<CB>;
  const int slabs = (p.K / 2 + 127) / 128;  // of 128 bytes a row; as few rows a tile as fill whole stages: the most tiles to share out
  p.tile = 32;
  while (p.tile < 8 * 32 && STAGE / (128 * p.tile) > slabs) p.tile *= 2;
  // With many items 64 rows, whose sums are handed over half as often (N 98304, 4
  // rows: 45 us, with 32 rows a tile 49; 32 rows of 8 experts, N 8192: 43 and
  // 45); with few, 32, which share out evenly (N 28672, K 8192: 27 us, 64 rows 30).
  const int64_t whole_passes = p.R / (2 * CB) > 0 ? p.R / (2 * CB) : 1;
  if (p.tile == 32 && whole_passes * (p.N / 32) >= 12 * (int64_t)sms) p.tile = 64;
  p.whole = p.K % 256 == 0 && STAGE > 128 * p.tile;  // one slab a stage: the map stays two-dimensional
  const int64_t room = SMEM - fixed_bytes<CB>(), per_row = (int64_t)p.blocks * (4 * KB) + p.epitch * 4;
  const int64_t stage = STAGE + (SC != ROW ? kScales<CB> : 0), fit = (room - 65536 / STAGE * stage) / per_row;
  p.pass = (int)(fit < 2 * CB ? fit : 2 * CB);
  if (p.pass > p.R) p.pass = p.R;
  const int64_t stages = (room - p.pass * per_row) / stage;
  p.stages = (int)(stages < MAX_STAGES ? stages : MAX_STAGES);
  if constexpr (SC != ROW) {  // the widest copies that all rows and stages begin at multiples of
    constexpr int SB = SC == GROUP_BF16 ? 2 : 4;
    const uintptr_t all = reinterpret_cast<uintptr_t>(p.scale) | (uintptr_t)p.groups * SB |
                          (uintptr_t)(2 * STAGE / (128 * p.tile)) * SB;
    p.scale_copy = all % 16 == 0 ? 16 : (all % 8 == 0 ? 8 : (all % 4 == 0 ? 4 : 2));
  }
  const int64_t passes = p.R / p.pass + (p.offsets == nullptr ? 1 : (p.R < p.E ? p.R : p.E));  // at most
  const int64_t items = passes * ((p.N + p.tile - 1) / p.tile);
  if (items > INT32_MAX) return fail(QLIN_ERR_UNSUPPORTED, "matvec_w4: too many outputs");
  CUtensorMap tw;
  const int rc = encode_slab_tmap(&tw, p.w, (uint64_t)p.K / 2, (uint64_t)p.E * p.N, 128, p.tile,
                                  p.whole ? STAGE / (128 * p.tile) : 1);
  if (rc) return rc;
  auto kern = matvec_kernel<DT, CB, SC>;
  static std::atomic<uint64_t> attr_devices{0};  // shared-memory limit raised once per device
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  cudaError_t e;
  if (!(attr_devices.load() & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(matvec_w4)");
    attr_devices.fetch_or(bit);
  }
  e = launch_pdl(kern, dim3((unsigned)(items < sms ? items : sms)), dim3(THREADS),
                 (size_t)(fixed_bytes<CB>() + p.pass * per_row + p.stages * stage), stream, tw, p);
  return e == cudaSuccess ? QLIN_OK : cuda_fail(e, "matvec_w4 launch");
}

template <int DT, int CB>
int launch_cb(const MatvecParams& p, cudaStream_t stream) {
  if (p.groups == 1) return launch_cfg<DT, CB, ROW>(p, stream);
  return p.scale_bf16 ? launch_cfg<DT, CB, GROUP_BF16>(p, stream) : launch_cfg<DT, CB, GROUP_F32>(p, stream);
}

template <int DT>
int launch_dt(MatvecParams p, bool aligned, cudaStream_t stream) {
  cudaError_t e;
  const int64_t per_row = (int64_t)p.blocks * (4 * KB) + p.epitch * 4;
  const bool fast = aligned && per_row <= kDigitRoom;  // (the latter: K up to about 32,000)
  p.own_digits = fast && makes_own_digits(p.offsets != nullptr, p.R, p.K);
  p.early = !p.own_digits && p.Rx > 0;
  if (p.early) {
    const int threads = 32 * (p.blocks < 32 ? p.blocks : 32);
    e = launch_pdl(split_kernel<DT>, dim3((unsigned)p.Rd), dim3(threads), 0, stream, p);
    if (e != cudaSuccess) return cuda_fail(e, "matvec_w4 split launch");
  }
  if (!fast) {
    const int64_t slots = p.offsets == nullptr ? 1 : (p.R < p.E ? p.R : p.E);
    const dim3 grid((unsigned)((p.N + 15) / 16), (unsigned)slots), block(32 * WARPS);
#define QLIN_ANY(CB)                                                                             \
  e = p.groups > 1 ? launch_pdl(matvec_any_kernel<DT, CB, true>, grid, block, 0, stream, p)      \
                   : launch_pdl(matvec_any_kernel<DT, CB, false>, grid, block, 0, stream, p)
    if (p.R <= 2 * slots) QLIN_ANY(1);
    else QLIN_ANY(4);
#undef QLIN_ANY
    return e == cudaSuccess ? QLIN_OK : cuda_fail(e, "matvec_w4 launch");
  }
  // Rows a pass by the rows an expert has on average (how they spread is known
  // on the device only): more columns than rows cost more than a second pass
  // over an expert's weights, which L2 then holds (32 rows of 8 experts, N
  // 8192, K 4096: 43 us with 4 rows a pass, 47 with 8; 16 rows 32 us with 4 rows
  // a pass, 34 with 2; 4 rows of one weight, N 24576: 19 and 24).  launch_cfg may
  // find room for fewer rows than the instance has columns for (K 8192 4 of 8,
  // 11008 3, 14336 2, above about 20,000 one), and the pass then costs what all
  // columns cost: N 4096, 4 rows 10.2 us at K 8192, 20.8 at K 11008; 8 rows 18.7
  // and 31.9.
  const int64_t sets = p.offsets == nullptr ? 1 : p.E;
  if (p.offsets == nullptr ? p.R <= 2 : p.R < 2 * sets) return launch_cb<DT, 1>(p, stream);
  if (p.R < 5 * sets) return launch_cb<DT, 2>(p, stream);
  return launch_cb<DT, 4>(p, stream);
}

bool aligned_weights(const uint8_t* w, int64_t K) { return K % 32 == 0 && (reinterpret_cast<uintptr_t>(w) & 15) == 0; }

struct Workspace {
  int64_t rows, blocks, epitch;
  size_t exps, bytes;
};
Workspace workspace_layout(int64_t R, int64_t Rx, int64_t K) {
  Workspace w;
  w.rows = R < Rx ? R : Rx;
  w.blocks = (K + KB - 1) / KB;
  w.epitch = (w.blocks + 3) & ~int64_t(3);
  w.exps = (size_t)(w.rows * w.blocks * (4 * KB));
  w.bytes = w.exps + (size_t)(w.rows * w.epitch) * sizeof(float);
  return w;
}

}  // namespace

size_t matvec_workspace_bytes(const uint8_t* w, bool experts, int64_t R, int64_t Rx, int64_t N, int64_t K) {
  if (aligned_weights(w, K) && makes_own_digits(experts, R, K)) return 0;
  return workspace_layout(R, Rx, K).bytes;
}

int launch_matvec_w4(int dt, const void* x, int64_t Rx, int64_t ldx, const uint8_t* w, const void* scale, int scale_dt,
                     int groups, const int32_t* offsets, int64_t E, const int32_t* x_rows, const void* bias, void* out,
                     int64_t R, int64_t N, int64_t K, void* workspace, cudaStream_t stream, int stall_weights,
                     int stall_scales) {
  if (device_sm_count() < 1) return fail(QLIN_ERR_NO_DEVICE, "no CUDA device");
  const Workspace l = workspace_layout(R, Rx, K);
  MatvecParams p{};
  p.x = x;
  p.Rx = Rx;
  p.Rd = l.rows;
  p.ldx = ldx;
  p.w = w;
  p.scale = scale;
  p.scale_bf16 = scale_dt == DT_BF16;
  p.groups = groups;
  p.offsets = offsets;
  p.E = (int)E;
  p.x_rows = x_rows;
  p.bias = bias;
  p.out = out;
  p.R = (int)R;
  p.N = (int)N;
  p.K = (int)K;
  p.blocks = (int)l.blocks;
  p.digits = static_cast<int8_t*>(workspace);
  p.exps = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + l.exps);
  p.epitch = (int)l.epitch;
  p.stall_weights = stall_weights;
  p.stall_scales = stall_scales;
  const int64_t four = 4 * (dt == DT_F32 ? 4 : 2);
  p.x_fours = K % 4 == 0 && ldx % 4 == 0 && reinterpret_cast<uintptr_t>(x) % four == 0;
  const bool aligned = aligned_weights(w, K);
  if (dt == DT_BF16) return launch_dt<DT_BF16>(p, aligned, stream);
  if (dt == DT_F16) return launch_dt<DT_F16>(p, aligned, stream);
  return launch_dt<DT_F32>(p, aligned, stream);
}

int set_matvec_wait_limit(uint64_t ns) { return set_tu_wait_limit(ns); }
int read_matvec_error(cudaStream_t stream, uint32_t* bits) { return read_tu_error(stream, bits); }

}  // namespace qlin
