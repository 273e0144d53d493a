// Dense 16-bit operators next to the grouped GEMMs: the gated feed-forward block of a shared or dense
// expert and the projection with its epilogue, forward and backward.
//
//   gated:  h  = act(x Wg^T) * (x Wu^T)          dg, du from dh;  dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x
//   linear: y  = act(x W^T + b) + r              dz = dy act'(z); dx = dz W;  dW = dz^T x;  db = column sums of dz
//
// Every product is one tcgen05 kernel (kind::f16, float32 accumulators in TMEM, operands staged by TMA in
// 128-byte-swizzled shared memory).  The operand whose reduction dimension is contiguous is "K-major", the other
// one "MN-major": both are read as they lie in memory, so nothing is ever transposed.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <mutex>
#include <type_traits>

#include "b200moe.h"
#include "common.cuh"

namespace b200moe {

constexpr int DENSE_BK = 64;                          // elements of the reduction per stage: one 128-byte swizzle row
constexpr int DENSE_SLAB = DENSE_BK * 128;            // an MN-major slab: 64 columns x 64 rows of the reduction
constexpr int DENSE_A_BYTES = 128 * DENSE_BK * 2;     // 128 operand rows
constexpr int DENSE_MAX_SPLIT = 8;                    // portable cluster size
constexpr int ST_DENSE_EMPTY = 401, ST_DENSE_FULL = 402, ST_DENSE_ACC = 403;

// epilogues
constexpr int DENSE_GLU = 0;     // gate and up accumulators -> activation product
constexpr int DENSE_LINEAR = 1;  // bias, activation, residual
constexpr int DENSE_STORE = 2;   // the accumulator as it is (gradients)

struct DenseParams {
  int rows, cols;            // valid rows (operand A side) and columns (operand B side) of the result
  int row_tiles, col_tiles;  // of one result; with `stacked` there are 2 * row_tiles
  int tile_cols;             // accumulator columns of a tile (per accumulator)
  int k_tiles;               // stages over the whole reduction (both chains)
  int chain_tiles;           // stages of one chain: beyond them the second pair of tensor maps is read
  int split;                 // CTAs of a cluster that share a tile's reduction
  int stages, stage_bytes;
  int reduce_offset;         // where the partial sums meet, from the start of the ring
  int reduce_in_ring;        // they meet in the ring itself
  int smem_bytes;
  int a_mn, b_mn;            // operand is MN-major
  int stacked;               // row tiles beyond row_tiles belong to the second A operand and the second output
  uint32_t idesc;
  uint32_t tmem_cols;
  int act;
  int f16;                   // 16-bit type of the operands and of 16-bit outputs
  int out_f32;
  int bias_f32;
  int vec_store;             // output rows may be written 16 bytes at a time
  void* out[2];
  void* pre[2];              // gate / up, or the pre-activation: written when not NULL
  const void* bias;
  const void* residual;
  int64_t ld_out, ld_res, ld_pre[2];
  const uint32_t* amax;      // the operands of a gradient were scaled by grad_scale of this: the result is scaled back
  int test_skip_b_loads;     // test hook: no load of operand B is issued, so every wait runs out
  uint64_t wait_limit_ns;
};

struct DenseMaps {
  CUtensorMap a[2], b[2];
};

// Instruction descriptor of kind::f16: [4,6) D = float32, [7,10) / [10,13) A / B = fp16 (0) or bf16 (1), bit 15 / 16 A / B
// MN-major, [17,23) N >> 3, [24,29) M >> 4
static uint32_t dense_idesc(int m, int n, bool f16, bool a_mn, bool b_mn) {
  const uint32_t t = f16 ? 0u : 1u;
  return (1u << 4) | (t << 7) | (t << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

// Issue by one lane of a converged warp, as predicated instructions instead of a branch around them: the operands then stay in
// uniform registers, where a branch moves every descriptor over for every instruction (four products and a commit took
// 250 cycles that way and 175 like this).
#define B200_IF_ASM(INSTR) "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t@q " INSTR "\n\t}"
template <bool kPair>
__device__ __forceinline__ void mma_f16_if(uint32_t go, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  if constexpr (kPair) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(go)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(go)
        : "memory");
  }
}
__device__ __forceinline__ void commit_if(uint32_t go, uint32_t bar) {
  asm volatile(B200_IF_ASM("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];")::"r"(go), "r"(bar) : "memory");
}
__device__ __forceinline__ void commit_pair_if(uint32_t go, uint32_t bar) {
  asm volatile(B200_IF_ASM("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%1], %2;")::"r"(go),
               "r"(bar), "h"((uint16_t)3)
               : "memory");
}
__device__ __forceinline__ void expect_tx_if(uint32_t go, uint32_t bar, uint32_t bytes) {
  asm volatile(B200_IF_ASM("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%1], %2;")::"r"(go), "r"(bar), "r"(bytes) : "memory");
}
// into the issuing CTA's own shared memory; kPair: credited to a barrier of either CTA of the pair
template <bool kPair>
__device__ __forceinline__ void load_2d_if(uint32_t go, uint32_t dst, const void* tmap, uint32_t bar, int c0, int c1) {
  if constexpr (kPair)
    asm volatile(B200_IF_ASM("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%2, {%4, %5}], [%3];")::"r"(go),
                 "r"(dst), "l"(tmap), "r"(bar), "r"(c0), "r"(c1)
                 : "memory");
  else
    asm volatile(B200_IF_ASM("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%2, {%4, %5}], [%3];")::"r"(go),
                 "r"(dst), "l"(tmap), "r"(bar), "r"(c0), "r"(c1)
                 : "memory");
}
#undef B200_IF_ASM

// 32 lanes x 16 consecutive columns -> 16 registers per thread
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// later uses of v[] stay behind the tcgen05.wait::ld that precedes this call
__device__ __forceinline__ void reg_fence16(float* v) {
  asm volatile(""
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                 "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])::"memory");
}
__device__ __forceinline__ void st_cluster_f32x4(uint32_t cluster_addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// Programmatic dependent launch: a kernel launched with the attribute may start while its predecessor on the stream
// drains, sets itself up, and waits here until the predecessor has ended and its writes are visible.  Nothing of global
// memory is touched before the wait.  The trigger lets the successor start in the same way.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Where a wait gave up, a CTA may not end, nor free its TMEM, while its copies still write its shared memory or its products still
// read it: after all warps have stopped issuing, they are waited for, whichever warp it was that gave up.  The limit is one for all waits
// of a CTA from `t0` on; the abort flag, which is set by then, does not end them.
__device__ __noinline__ void drain_wait(uint32_t bar, uint32_t parity, uint64_t t0, uint64_t limit_ns) {
#pragma unroll 1
  while (!mbar_try_wait_hint(bar, parity, kWaitHintNs) && global_timer_ns() - t0 <= limit_ns) {
  }
}
// the copies of the last `issued` stages, the latest round of each stage
__device__ __forceinline__ void drain_copies(uint32_t full_bar0, int issued, int stages, uint64_t limit_ns) {
  const uint64_t t0 = global_timer_ns();
  for (int i = max(0, issued - stages); i < issued; ++i) drain_wait(full_bar0 + 8u * (uint32_t)(i % stages), (uint32_t)(i / stages) & 1u, t0, limit_ns);
}

__device__ __forceinline__ float load16(const void* p, int64_t i, bool f16) {
  return f16 ? __half2float(reinterpret_cast<const __half*>(p)[i]) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store16(void* p, int64_t i, float v, bool f16) {
  if (f16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ float2 unpack16x2(uint32_t w, bool f16) {
  return f16 ? __half22float2(*reinterpret_cast<__half2*>(&w)) : __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w));
}

// ---------------------------------------------------------------------------------------
// Scale of an fp16 gradient operand (dz, or dg and du together): the power of two that brings its largest finite magnitude `amax`
// (the bits of a float32, kept on the device) into [2^14, 2^15).  fp16 holds 2^-24 to 65504, a gradient from float32 values or from
// products with `up` may lie anywhere; so scaled, values down to 2^-28 of the largest keep all their bits and none
// overflows.  The sums of the products are taken back by the inverse, in float32: both factors are exact.  Finding amax takes a pass of its own
// over what dz is formed from (backward pass of the gated block, 1531 x 7168, 2048: 157 -> 165 us).
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ int grad_exponent(uint32_t amax) { return amax ? min(14 - ((int)(amax >> 23) - 127), 126) : 0; }
__device__ __forceinline__ float pow2_f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ float grad_scale(const uint32_t* amax) { return amax ? pow2_f(grad_exponent(*amax)) : 1.0f; }
__device__ __forceinline__ float grad_unscale(const uint32_t* amax) { return amax ? pow2_f(-grad_exponent(*amax)) : 1.0f; }

// ---------------------------------------------------------------------------------------
// Activations.  sigmoid(v) = 1 / (1 + 2^(-v log2 e)) on the approximate exponential and reciprocal (about 2^-22
// relative each, where the exponential's argument is small; its rounding costs 2^-24 of the argument, so 4e-6 at v = -80, and below
// -87 the result is 0).  Of a 16-bit result that is a 2^-7th of a step or less; float32 results carry it as it is.
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ float sigmoid_f(float v) { return rcp_approx(1.0f + ex2_approx(v * -1.4426950408889634f)); }

// SwiGLU: gate sigmoid(gate) up.  GeGLU as the grouped GEMM defines it: gate <= 7, -7 <= up <= 7,
// (up + 1) gate sigmoid(1.702 gate).  The limits pass NaN on (a comparison, not fminf).
__device__ __forceinline__ float glu_f(float g, float u, int act) {
  if (act == B200MOE_ACT_GEGLU) {
    g = g > 7.0f ? 7.0f : g;
    u = u > 7.0f ? 7.0f : (u < -7.0f ? -7.0f : u);
    return g * sigmoid_f(1.702f * g) * (u + 1.0f);
  }
  return g * sigmoid_f(g) * u;
}
// gradients with respect to gate and up; a limited value has none
__device__ __forceinline__ void glu_grad_f(float dh, float g, float u, int act, float& dg, float& du) {
  if (act == B200MOE_ACT_GEGLU) {
    const bool g_in = !(g > 7.0f), u_in = !(u > 7.0f || u < -7.0f);
    g = g_in ? g : 7.0f;
    u = u > 7.0f ? 7.0f : (u < -7.0f ? -7.0f : u);
    const float s = sigmoid_f(1.702f * g);
    dg = g_in ? dh * (u + 1.0f) * s * (1.0f + 1.702f * g * (1.0f - s)) : 0.0f;
    du = u_in ? dh * g * s : 0.0f;
  } else {
    const float s = sigmoid_f(g);
    dg = dh * u * s * (1.0f + g * (1.0f - s));
    du = dh * g * s;
  }
}
// Distribution function of the normal distribution, erfc(-z / sqrt 2) / 2, and e^(-z^2 / 2).  With x = |z| / sqrt 2 and
// t = 1 / (1 + 0.4 x), e^(x^2) erfc(x) = t P(t); P of degree 8 is a fit over (0, 1] for the least largest relative error (reweighted
// least squares on Chebyshev nodes: 1.3e-7).  In float32 that is within 6e-7 for z >= -2 and, as the exponent's argument is rounded,
// within 1.4e-6 down to -5 and 8e-6 to the end of the range: the negative tail keeps its digits.  (Through erfcf the
// 777 x 1000 -> 2001 product took 4 us longer.)
__device__ __forceinline__ float normal_cdf_f(float z, float& e) {
  const float t = rcp_approx(fmaf(fabsf(z), 0.4f * 0.70710678118654752f, 1.0f));
  float q = 0.05026041716337204f;
  q = fmaf(q, t, -0.18289488554000854f);
  q = fmaf(q, t, 0.16907517611980438f);
  q = fmaf(q, t, -0.005599260330200195f);
  q = fmaf(q, t, 0.14142775535583496f);
  q = fmaf(q, t, 0.16854286193847656f);
  q = fmaf(q, t, 0.2078426033258438f);
  q = fmaf(q, t, 0.22566960752010345f);
  q = fmaf(q, t, 0.22567586600780487f);
  e = ex2_approx(z * z * -0.72134752044448171f);
  const float tail = 0.5f * t * q * e;
  return z > 0.0f ? 1.0f - tail : tail;
}
__device__ __forceinline__ float act_f(float z, int act) {
  switch (act) {
    case B200MOE_ACT_RELU: return z < 0.0f ? 0.0f : z;
    case B200MOE_ACT_SILU: return z * sigmoid_f(z);
    case B200MOE_ACT_GELU: {
      float e;
      return z * normal_cdf_f(z, e);
    }
    default: return z;
  }
}
__device__ __forceinline__ float act_grad_f(float z, int act) {
  switch (act) {
    case B200MOE_ACT_RELU: return z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
    case B200MOE_ACT_SILU: {
      const float s = sigmoid_f(z);
      return s * (1.0f + z * (1.0f - s));
    }
    case B200MOE_ACT_GELU: {
      float e;
      const float cdf = normal_cdf_f(z, e);
      return fmaf(z * 0.3989422804014327f, e, cdf);
    }
    default: return 1.0f;
  }
}

// the activation on kN values: one uniform branch, so that v[] stays in registers
template <int kN>
__device__ __forceinline__ void act_values(float* v, int act) {
  if (act == B200MOE_ACT_RELU) {
#pragma unroll
    for (int q = 0; q < kN; ++q) v[q] = act_f(v[q], B200MOE_ACT_RELU);
  } else if (act == B200MOE_ACT_SILU) {
#pragma unroll
    for (int q = 0; q < kN; ++q) v[q] = act_f(v[q], B200MOE_ACT_SILU);
  } else if (act == B200MOE_ACT_GELU) {
#pragma unroll
    for (int q = 0; q < kN; ++q) v[q] = act_f(v[q], B200MOE_ACT_GELU);
  }
}

// ---------------------------------------------------------------------------------------
// One tile per CTA.  The tile's reduction may be shared by the CTAs of a cluster: each walks its part of the
// k-tiles, sends its partial sums to the owners of the columns through distributed shared memory, and every CTA
// finishes its share of the columns.  Sums are added in the order of the ranks, so a result does not depend on timing.
//
// DENSE_GLU: the 128 operand rows of a tile are 64 rows of the gate weights and the same 64 rows of the up weights, so the
// two projections of a feature land in lanes r and r + 64 and meet in shared memory, where the partial sums go anyway.
//
// kTrans: the rows of the tile are output features and its columns are tokens, element (r, c) goes to
// out[c * ld + r] (32 lanes = 32 neighbouring features); otherwise element (r, c) goes to out[r * ld + c].
//
// kSeg: the accumulator is drained into registers every kSegTiles stages and added there with float32
// round-to-nearest.  The tensor core's own accumulation rounds towards zero: over K = 7168 that leaves a bias of
// 7e-6 of the result (measured), 4e-7 over the 512 elements of a segment.  Used for float32 outputs; a 16-bit
// output's rounding (2^-9) hides it.
//
// warps: 0 producer of A, 10 producer of B, 1 MMA issuer and TMEM owner, 2-9 epilogue (TMEM lane quarter x every other 16
// columns)
// ---------------------------------------------------------------------------------------
constexpr int DENSE_THREADS = 352;
constexpr int DENSE_WARP_B = 10;
// Two CTAs fit an SM only if registers suffice for 12 + 12 warps: the warps of both start at the same of the SM's four parts, so
// two of them hold 6 (95 registers a thread left one CTA to an SM).
constexpr int DENSE_BOUND = 384;
constexpr int DENSE_SMEM = 112 * 1024;       // per CTA, two CTAs to an SM
constexpr int DENSE_SMEM_ALONE = 225 * 1024;  // where every CTA has an SM of its own
constexpr int kSegTiles = 8;
constexpr int kSegCols = 128;

template <bool kTrans, int kEpi, bool kSeg>
__global__ void __launch_bounds__(DENSE_BOUND, kSeg ? 1 : 2) dense_tile_kernel(const __grid_constant__ DenseMaps maps, const __grid_constant__ DenseParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t s_bars[2 * 16 + 5];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ int s_issued[2];  // stages whose copies each producer has issued
  constexpr bool kGlu = kEpi == DENSE_GLU;
  constexpr int kTileRows = kGlu ? 64 : 128;
  const uint32_t ring = smem_u32(smem);
  const uint32_t bars = smem_u32(s_bars);
  const int stages = p.stages;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (16 + s); };
  auto acc_full_bar = [&](int b) { return bars + 8u * (32 + b); };
  auto acc_empty_bar = [&](int b) { return bars + 8u * (34 + b); };
  const uint32_t drain_bar = bars + 8u * 36;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WaitCtx wc = {&s_abort, p.wait_limit_ns};

  const int rank = (int)(blockIdx.x % (unsigned)p.split);
  const int tile = (int)(blockIdx.x / (unsigned)p.split);
  const int all_row_tiles = p.row_tiles * (p.stacked ? 2 : 1);
  int row_tile = tile % all_row_tiles;
  const int col_tile = tile / all_row_tiles;
  const int which = row_tile >= p.row_tiles ? 1 : 0;  // stacked: second operand and output
  row_tile -= which * p.row_tiles;
  const int C = p.tile_cols;
  const int row0 = row_tile * kTileRows, col0 = col_tile * C;
  const int kt0 = (int)((int64_t)p.k_tiles * rank / p.split), kt1 = (int)((int64_t)p.k_tiles * (rank + 1) / p.split);
  const int nk = kt1 - kt0;  // at least 1: split <= k_tiles

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full_bar(b), 1);
      mbar_init(acc_empty_bar(b), 8);
    }
    mbar_init(drain_bar, 1);
    s_abort = s_issued[0] = s_issued[1] = 0;
    fence_mbar_init();
    prefetch_tensormap(&maps.a[0]);
    prefetch_tensormap(&maps.b[0]);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&s_tmem), p.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // (waited for before the first access to another CTA's shared memory: by then every CTA of the cluster has started)
  if (p.split > 1) cluster_arrive();
  const uint32_t tmem = s_tmem;
  pdl_wait();
  pdl_trigger();

  if (warp == 0 || (!kGlu && warp == DENSE_WARP_B)) {
    // ---- producers ----------------------------------------------------------------------
    // (stage, parity and addresses run along: a division by the number of stages in this loop and the issuer's made a stage
    // cost 700 cycles whatever it held; one warp for both operands took 420.  The gated block's one warp issues both all the
    // same: 17.5 us against 18.8 for 128 tokens of 7168 -> 2 x 2048.)
    const bool side_b = warp != 0;
    const uint32_t stage_bytes = (uint32_t)p.stage_bytes, dst0 = ring + (side_b ? DENSE_A_BYTES : 0), dst_end = dst0 + (uint32_t)stages * stage_bytes;
    const bool mn = side_b ? p.b_mn != 0 : (!kGlu && p.a_mn != 0), two = !side_b || C > 64;
    const int first = side_b ? col0 : row0;
    const CUtensorMap* map = side_b ? &maps.b[0] : &maps.a[kGlu ? 0 : which];
    const CUtensorMap* map1 = side_b ? &maps.b[1] : &maps.a[1];  // of the second chain, or the up weights
    int kt = kt0, chain_left = p.chain_tiles - kt;
    if (chain_left <= 0) {
      kt -= p.chain_tiles;
      map = map1;
    }
    int kc = kt * DENSE_BK;
    uint32_t dst = dst0, fb = full_bar(0), eb = empty_bar(0), parity = 1;
    const uint32_t elected = elect_one();  // (the same lane of a full warp every time)
    const uint32_t go = side_b && p.test_skip_b_loads ? 0u : elected, go_announce = side_b ? 0u : elected;
    int issued = 0;
    for (; issued < nk; ++issued) {
      if (!__all_sync(0xffffffffu, mbar_wait(eb, parity, wc, ST_DENSE_EMPTY))) break;
      expect_tx_if(go_announce, fb, stage_bytes);
      if (mn) {
        load_2d_if<false>(go, dst, map, fb, first, kc);
        if (two) load_2d_if<false>(go, dst + DENSE_SLAB, map, fb, first + 64, kc);
      } else {
        load_2d_if<false>(go, dst, map, fb, kc, first);
        if constexpr (kGlu) {
          load_2d_if<false>(go, dst + 64 * 128, map1, fb, kc, first);
          load_2d_if<false>(p.test_skip_b_loads ? 0u : go, dst + DENSE_A_BYTES, &maps.b[0], fb, kc, col0);
        }
      }
      kc += DENSE_BK;
      if (--chain_left == 0) {
        kc = 0;
        map = map1;
      }
      dst += stage_bytes;
      fb += 8;
      eb += 8;
      if (dst == dst_end) {
        dst = dst0;
        fb = full_bar(0);
        eb = empty_bar(0);
        parity ^= 1u;
      }
    }
    if (lane == 0) s_issued[side_b] = issued;
    __syncwarp();
  } else if (warp == 1) {
    // ---- MMA issuer ---------------------------------------------------------------------
    constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);  // SBO 1024, version 1, 128-byte swizzle
    // K-major: 16 elements = 32 bytes further per MMA inside the swizzle row.  MN-major: 16 rows of 128 bytes; the
    // leading byte offset is the distance of two slabs.  (In a cluster the shared-memory address of a CTA carries its
    // rank above the 18 bits of the offset: only the 14-bit field goes into the descriptor.)
    const uint32_t a_lo0 = ((ring >> 4) & 0x3FFFu) | (p.a_mn ? (uint32_t)(DENSE_SLAB >> 4) << 16 : 1u << 16);
    const uint32_t b_lo0 = (((ring + DENSE_A_BYTES) >> 4) & 0x3FFFu) | (p.b_mn ? (uint32_t)(DENSE_SLAB >> 4) << 16 : 1u << 16);
    const uint32_t a_step = p.a_mn ? (16u * 128u) >> 4 : 2u, b_step = p.b_mn ? (16u * 128u) >> 4 : 2u;
    const uint32_t stage_step = (uint32_t)p.stage_bytes >> 4, idesc = p.idesc;
    auto desc = [](uint32_t lo) { return ((uint64_t)HI << 32) | lo; };
    bool ok = true;
    int seg = 0, in_seg = 0, stage = 0;
    uint32_t parity = 0, a_lo = a_lo0, b_lo = b_lo0;
    const uint32_t go = elect_one();
    for (int i = 0; i < nk && ok; ++i) {
      const uint32_t acc = tmem + (kSeg ? (uint32_t)((seg & 1) * C) : 0u);
      if (kSeg && in_seg == 0 && seg >= 2) {
        // the epilogue has taken the segment that used this accumulator
        if (!__all_sync(0xffffffffu, mbar_wait(acc_empty_bar(seg & 1), (uint32_t)((seg >> 1) - 1) & 1u, wc, ST_DENSE_ACC))) { ok = false; break; }
        tc_fence_after();
      }
      if (!__all_sync(0xffffffffu, mbar_wait(full_bar(stage), parity, wc, ST_DENSE_FULL))) { ok = false; break; }
      const bool seg_end = i + 1 == nk || (kSeg && in_seg == kSegTiles - 1);
#pragma unroll
      for (int j = 0; j < 4; ++j) mma_f16_if<false>(go, acc, desc(a_lo + j * a_step), desc(b_lo + j * b_step), idesc, (in_seg | j) != 0);
      commit_if(go, empty_bar(stage));
      if (seg_end) commit_if(go, acc_full_bar(kSeg ? seg & 1 : 0));
      ++in_seg;
      if (seg_end) {
        ++seg;
        if (kSeg) in_seg = 0;
      }
      a_lo += stage_step;
      b_lo += stage_step;
      if (++stage == stages) {
        stage = 0;
        parity ^= 1u;
        a_lo = a_lo0;
        b_lo = b_lo0;
      }
    }
    __syncwarp();
  }

  // ---- epilogue -------------------------------------------------------------------------
  const bool f16 = p.f16 != 0;
  const bool finisher = warp >= 2 && warp < 10;
  const int quarter = warp & 3, half = (warp - 2) >> 2;  // this warp: TMEM lanes 32 quarter .. + 31, chunks half, half + 2, ...
  const int r_in_tile = quarter * 32 + lane;
  const int valid = min(C, p.cols - col0);
  float sums[kSeg ? kSegCols / 2 : 1];
  bool ok = true;
  if (finisher) {
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    if constexpr (kSeg) {
#pragma unroll
      for (int j = 0; j < kSegCols / 2; ++j) sums[j] = 0.0f;
      const int segs = (nk + kSegTiles - 1) / kSegTiles;
      for (int sg = 0; sg < segs; ++sg) {
        if (!__all_sync(0xffffffffu, mbar_wait(acc_full_bar(sg & 1), (uint32_t)(sg >> 1) & 1u, wc, ST_DENSE_ACC))) { ok = false; break; }
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < kSegCols / 32; ++q) {
          const int c = half * 16 + q * 32;
          if (c < C) {
            float v[16];
            tmem_ld_32x16(tmem + lanes + (uint32_t)((sg & 1) * C + c), v);
            tmem_ld_wait();
            reg_fence16(v);
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[q * 16 + j] += v[j];
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty_bar(sg & 1));
      }
    } else {
      ok = __all_sync(0xffffffffu, mbar_wait(acc_full_bar(0), 0, wc, ST_DENSE_ACC));
      tc_fence_after();
    }
  }

  // this warp's chunks of 16 accumulator columns: f(first column, values)
  auto each_chunk = [&](auto f) {
    if constexpr (kSeg) {
#pragma unroll
      for (int q = 0; q < kSegCols / 32; ++q)
        if (half * 16 + q * 32 < valid) f(half * 16 + q * 32, sums + q * 16);
    } else {
      const uint32_t base = tmem + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
      for (int c = half * 16; c < valid; c += 32) {
        float v[16];
        __syncwarp();
        tmem_ld_32x16(base + c, v);
        tmem_ld_wait();
        reg_fence16(v);
        f(c, v);
      }
    }
  };
  // kTrans: kN values of feature `row` for the tokens col0 + c0 + j, of which the first `count` exist; v = the accumulator
  // (GLU: the gate's), u = the up projection's.  Every choice is a branch around a whole loop.
  const float unscale = !kGlu && finisher ? grad_unscale(p.amax) : 1.0f;
  // residual values (raw) of the same elements; their loads are issued by `fetch`, ahead of whatever v waits for
  auto fetch = [&](auto size, int row, int c0, int count, uint16_t* raw) {
    constexpr int kN = decltype(size)::value;
    if (kEpi != DENSE_LINEAR || !p.residual) return;
    const uint16_t* r = reinterpret_cast<const uint16_t*>(p.residual) + (int64_t)(col0 + c0) * p.ld_res + row;
#pragma unroll
    for (int j = 0; j < kN; ++j, r += p.ld_res)
      if (j < count) raw[j] = __ldg(r);
  };
  auto finish = [&](auto size, int row, int c0, int count, float bias, float* v, const float* u, const uint16_t* raw) {
    constexpr int kN = decltype(size)::value;
    const int64_t t0 = col0 + c0;
    auto put = [&](void* base, int64_t ld, const float* w) {
      uint16_t* d = reinterpret_cast<uint16_t*>(base) + t0 * ld + row;
      if (f16) {
#pragma unroll
        for (int j = 0; j < kN; ++j, d += ld)
          if (j < count) *d = __half_as_ushort(__float2half_rn(w[j]));
      } else {
#pragma unroll
        for (int j = 0; j < kN; ++j, d += ld)
          if (j < count) *d = __bfloat16_as_ushort(__float2bfloat16_rn(w[j]));
      }
    };
    if constexpr (kGlu) {
      if (p.pre[0]) {
        put(p.pre[0], p.ld_pre[0], v);
        put(p.pre[1], p.ld_pre[1], u);
      }
#pragma unroll
      for (int j = 0; j < kN; ++j) v[j] = glu_f(v[j], u[j], p.act);
    } else {
#pragma unroll
      for (int j = 0; j < kN; ++j) v[j] = fmaf(v[j], unscale, bias);
      if (p.pre[0]) put(p.pre[0], p.ld_pre[0], v);
      act_values<kN>(v, p.act);
      if (p.residual) {
#pragma unroll
        for (int j = 0; j < kN; ++j)
          if (j < count) v[j] += f16 ? __half2float(__ushort_as_half(raw[j])) : __bfloat162float(__ushort_as_bfloat16(raw[j]));
      }
    }
    if (p.out_f32) {
      float* d = reinterpret_cast<float*>(p.out[0]) + t0 * p.ld_out + row;
#pragma unroll
      for (int j = 0; j < kN; ++j, d += p.ld_out)
        if (j < count) *d = v[j];
    } else {
      put(p.out[0], p.ld_out, v);
    }
  };
  auto bias_at = [&](int row) -> float {
    if (kEpi != DENSE_LINEAR || !p.bias || row >= p.rows) return 0.0f;
    return p.bias_f32 ? reinterpret_cast<const float*>(p.bias)[row] : load16(p.bias, row, f16);
  };

  const int split = p.split;
  if (kGlu || split > 1) {
    // partial sums meet in shared memory, four columns of a row side by side: [rank][4 columns of the owner's slice][row][4].
    // With one CTA that is the ring, which the products have left; with several a region of its own, since another CTA's
    // products may still read its ring, or, where that would leave too few stages, the ring once all of the cluster's
    // products are done.
    const int slice4 = ((valid + split - 1) / split + 3) / 4;  // groups of 4 columns that one CTA of the cluster finishes
    const uint32_t region = ring + p.reduce_offset;
    if (split > 1) {
      __syncwarp();
      cluster_wait();  // (of the arrival at the start)
      if (p.reduce_in_ring) {
        cluster_arrive();
        cluster_wait();
      }
    }
    if (finisher && ok) {
      each_chunk([&](int c0, const float* v) {
        const uint32_t base = region + (uint32_t)((rank * slice4 * 128 + r_in_tile) * 16);
        int owner = (c0 / 4) / slice4, at = c0 / 4 - owner * slice4;
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          if (c0 + j < valid) {
            const float4 w = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            if (split == 1) st_shared_f32x4(base + (uint32_t)((c0 + j) * 512), w);
            else st_cluster_f32x4(map_to_cta(base, (uint32_t)owner) + (uint32_t)(at * 2048), w);
            if (++at == slice4) {
              at = 0;
              ++owner;
            }
          }
        }
      });
    }
    // where a wait gave up, sums are missing: the CTAs of the cluster tell one another and store nothing
    __syncwarp();
    if (split > 1) {
      if (lane < split && *wc.abort_flag) st_shared_cluster(map_to_cta(smem_u32(&s_abort), (uint32_t)lane), 1u);
      __syncwarp();
      cluster_arrive();
      cluster_wait();
    } else {
      __syncthreads();
    }
    if (finisher && !*wc.abort_flag) {
      constexpr int kGroups = 256 / kTileRows;  // groups of columns in flight
      const int t = (int)threadIdx.x - 64;
      const int r = t % kTileRows, row = row0 + r;
      if (row < p.rows) {
        const float4* part = reinterpret_cast<const float4*>(smem + p.reduce_offset) + r;
        const float bias = bias_at(row);
        for (int g = t / kTileRows; g < slice4; g += kGroups) {
          const int c = (rank * slice4 + g) * 4, count = min(4, valid - c);
          if (count <= 0) break;
          uint16_t raw[4];
          if constexpr (kTrans) fetch(std::integral_constant<int, 4>(), row, c, count, raw);
          float v[4] = {0.0f, 0.0f, 0.0f, 0.0f}, u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          for (int q = 0; q < split; ++q) {
            const float4 w = part[(q * slice4 + g) * 128];
            v[0] += w.x, v[1] += w.y, v[2] += w.z, v[3] += w.w;
            if constexpr (kGlu) {
              const float4 x = part[(q * slice4 + g) * 128 + 64];
              u[0] += x.x, u[1] += x.y, u[2] += x.z, u[3] += x.w;
            }
          }
          if constexpr (kTrans) {
            finish(std::integral_constant<int, 4>(), row, c, count, bias, v, u, raw);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (j < count) store16(p.out[which], (int64_t)row * p.ld_out + col0 + c + j, v[j] * unscale, f16);
          }
        }
      }
    }
  } else if (finisher && ok) {
    const int row = row0 + r_in_tile;
    const bool row_ok = row < p.rows;
    const float bias = bias_at(row);
    uint16_t raw[16];
    const std::integral_constant<int, 8> eight;
    const std::integral_constant<int, 16> sixteen;
    if (kTrans && row_ok && half * 16 < valid) fetch(sixteen, row, half * 16, valid - half * 16, raw);
    each_chunk([&](int c0, const float* v) {
      if (!row_ok) return;
      if constexpr (kTrans) {
        uint16_t now[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) now[j] = raw[j];
        if (c0 + 32 < valid) fetch(sixteen, row, c0 + 32, valid - c0 - 32, raw);  // this warp's next chunk
#pragma unroll
        for (int h = 0; h < 16; h += 8) {
          if (c0 + h >= valid) break;
          float w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = v[h + j];
          finish(eight, row, c0 + h, min(8, valid - c0 - h), bias, w, w, now + h);
        }
      } else {
        const int64_t o = (int64_t)row * p.ld_out + col0 + c0;
        if (p.vec_store && c0 + 16 <= valid) {
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = pack16x2_from_float(v[2 * j] * unscale, v[2 * j + 1] * unscale, f16);
          uint4* d = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out[which]) + o);
          d[0] = make_uint4(w[0], w[1], w[2], w[3]);
          d[1] = make_uint4(w[4], w[5], w[6], w[7]);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < valid) store16(p.out[which], o + j, v[j] * unscale, f16);
        }
      }
    });
  }
  tc_fence_before();
  __syncthreads();
  if (*wc.abort_flag) {
    if (warp == 0) drain_copies(full_bar(0), max(s_issued[0], s_issued[1]), stages, p.wait_limit_ns);
    if (warp == 1) {
      commit_if(elect_one(), drain_bar);  // (of all products that this lane has issued)
      drain_wait(drain_bar, 0, global_timer_ns(), p.wait_limit_ns);
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, p.tmem_cols);
  }
}

// ---------------------------------------------------------------------------------------
// Large products: a persistent kernel of CTA pairs, one pair per two SMs.  A tile is 256 x 256 (cta_group::2: each CTA
// holds 128 rows of A, 128 columns of B and the accumulator of its 128 rows), its two accumulators of 256 columns fill
// TMEM, so the epilogue of one tile runs beside the products of the next.  Where tiles of that size would leave pairs
// without work they have 128 columns (half the flops on three quarters of the bytes).  Rows are tokens (or, for a weight's gradient,
// the weight's rows), so a thread of the epilogue holds 32 neighbouring columns of one output row.
//
// DENSE_GLU: the pair's first CTA loads 128 (64) rows of the gate weights as its half of B, the second the same rows of the
// up weights: the first half of the accumulator's columns are the gate, the second half the up projection of the same features.
//
// A launch walks one or two jobs (the two gradient products of a backward pass share a launch: the tiles of the second fill
// the last wave of the first).  Tiles are dealt out in rounds; where the last round of job 0 leaves pairs idle, they
// begin job 1 `early` rounds sooner.
//
// warps: 0 producer of A, 10 producer of B (with MN-major operands a stage takes four copies per CTA, more than one warp issues
// in the time of its products), 1 MMA issuer (first CTA) and TMEM owner, 2-9 epilogue (TMEM lane quarter x column half)
// ---------------------------------------------------------------------------------------
constexpr int PAIR_THREADS = 352;
constexpr int PAIR_WARP_B = 10;
constexpr int PAIR_STAGES = 6;
constexpr int PAIR_STAGE_BYTES = 2 * DENSE_A_BYTES;
constexpr int PAIR_EPI_WARPS = 8;
constexpr int PAIR_BOX = 32 * 32 * 2;  // a block of 32 rows x 32 columns of the output
constexpr int PAIR_STAGING = PAIR_STAGES * PAIR_STAGE_BYTES;  // two blocks per epilogue warp
constexpr int PAIR_SMEM = PAIR_STAGING + PAIR_EPI_WARPS * 2 * PAIR_BOX + 1024;
constexpr int ST_PAIR_EMPTY = 411, ST_PAIR_FULL = 412, ST_PAIR_ACC_EMPTY = 413, ST_PAIR_ACC_FULL = 414;

struct PairJob {
  int rows, cols;
  int row_tiles, col_tiles;   // row_tiles of one result; twice as many with `stacked`
  int k_tiles, chain_tiles;
  int a_mn, b_mn, stacked;
  int tiles;
  int tile_cols;              // accumulator columns of a tile: 256 or 128
  int raster;                 // row tiles of a raster group: the group's rows of A stay in L2 while its columns pass
  uint32_t idesc;
  int tma_store;              // the outputs (and pre-activations) of every job have tensor maps: 16-byte aligned base and pitch
  void* out[2];
  int64_t ld_out;
};

struct PairParams {
  PairJob job[2];
  int jobs;
  int full_rounds, rest;      // job 0: every pair takes full_rounds tiles, the first `rest` pairs one more
  int early, early_tiles;     // rounds (and tiles) of job 1 that the other pairs take before all join
  int act, f16, bias_f32;
  void* pre[2];
  int64_t ld_pre[2];
  const void* bias;
  const void* residual;
  int64_t ld_res;
  int vec_res;                // residual rows may be read 16 bytes at a time
  const uint32_t* amax;       // as in DenseParams
  int test_skip_b_loads;      // test hook, as in DenseParams
  uint64_t wait_limit_ns;
};

struct PairMaps {
  DenseMaps job[2];
  CUtensorMap out[2][2];  // of each job: the outputs
  CUtensorMap pre[2];
};

struct PairTile {
  int job, row_tile, col_tile, which;
};

// the i-th tile of a pair; false when it has no more
__device__ __forceinline__ bool pair_tile(const PairParams& p, int pair, int pairs, int i, PairTile& t) {
  int idx;
  const int mine = p.full_rounds + (pair < p.rest ? 1 : 0);
  if (i < mine) {
    t.job = 0;
    idx = pair + i * pairs;
  } else {
    if (p.jobs < 2) return false;
    t.job = 1;
    i -= mine;
    const int early = p.rest > 0 && pair >= p.rest ? p.early : 0;
    if (i < early) {
      idx = i * (pairs - p.rest) + pair - p.rest;
      if (idx >= p.early_tiles) return false;
    } else {
      idx = p.early_tiles + (i - early) * pairs + pair;
      if (idx >= p.job[1].tiles) return false;
    }
  }
  const PairJob& j = p.job[t.job];
  const int rows = j.row_tiles * (j.stacked ? 2 : 1);
  const int group = idx / (j.raster * j.col_tiles);
  const int in = idx - group * j.raster * j.col_tiles;
  const int height = min(j.raster, rows - group * j.raster);
  t.col_tile = in / height;
  t.row_tile = group * j.raster + in - t.col_tile * height;
  t.which = t.row_tile >= j.row_tiles ? 1 : 0;
  t.row_tile -= t.which * j.row_tiles;
  return true;
}

__device__ __forceinline__ void tma_store_2d(const void* tmap, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(tmap), "r"(src), "r"(c0), "r"(c1) : "memory");
}
// all but the thread's latest bulk copy have finished reading shared memory
__device__ __forceinline__ void bulk_wait_read1() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }
__device__ __forceinline__ void st_shared_u32x4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// One warp's block of 32 rows x 32 columns to 16-bit memory: lane = row, v[] = its columns.  Stored from registers, every
// instruction would touch 32 lines (7000 cycles for a tile of 128 x 256, measured as 87 us for 896 tiles); so the block goes
// through shared memory (two blocks in turn, 64-byte swizzle: 16-byte writes without bank conflicts) and leaves as one bulk
// copy, or, where an output has no tensor map, row by row with neighbouring lanes on neighbouring columns.  A residual comes in
// the same way.  A launch keeps to one of the two forms: only the first waits for earlier copies that still read a block.
struct BlockWriter {
  uint32_t staging;  // this warp's two blocks
  int turn;
  int lane;
  bool f16;
  // v[] += the block of `base` at (row0, col); values beyond rows and cols are not read
  __device__ __forceinline__ void add(float* v, const void* base, int64_t ld, bool vec, int row0, int rows, int col, int cols) {
    const uint32_t block = staging + (uint32_t)(turn * PAIR_BOX);
    turn ^= 1;
    if (lane == 0) bulk_wait_read1();  // the copy before the last one used this block
    __syncwarp();
    const uint16_t* src = reinterpret_cast<const uint16_t*>(base);
    if (vec && col + 32 <= cols) {
      // 8 rows at a time, 4 lanes to a row
      uint4 w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = row0 + 8 * q + (lane >> 2);
        w[q] = make_uint4(0, 0, 0, 0);
        if (r < rows) w[q] = __ldg(reinterpret_cast<const uint4*>(src + (int64_t)r * ld + col) + (lane & 3));
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = 8 * q + (lane >> 2);
        st_shared_u32x4(block + (uint32_t)(r * 64) + ((uint32_t)((lane & 3) ^ ((r >> 1) & 3)) << 4), w[q].x, w[q].y, w[q].z, w[q].w);
      }
    } else {
      const bool in = col + lane < cols;
      const int count = min(32, rows - row0);
#pragma unroll 8
      for (int r = 0; r < 32; ++r) {
        uint16_t h = 0;
        if (in && r < count) h = src[(int64_t)(row0 + r) * ld + col + lane];
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(block + (uint32_t)(r * 64) + ((((uint32_t)lane >> 3) ^ (uint32_t)((r >> 1) & 3)) << 4) + (uint32_t)(lane & 7) * 2), "h"(h) : "memory");
      }
    }
    __syncwarp();
    const uint32_t line = block + (uint32_t)(lane * 64), swz = (uint32_t)((lane >> 1) & 3);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t w[4];
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(line + (((uint32_t)q ^ swz) << 4)) : "memory");
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack16x2(w[e], f16);
        v[8 * q + 2 * e] += f.x;
        v[8 * q + 2 * e + 1] += f.y;
      }
    }
    __syncwarp();
    if (lane == 0) bulk_commit();  // (an empty group: the block after this one was last used two groups ago)
  }
  __device__ __forceinline__ void write(const float* v, const CUtensorMap* map, void* base, int64_t ld, bool tma, int row0, int rows, int col, int cols) {
    const uint32_t block = staging + (uint32_t)(turn * PAIR_BOX);
    turn ^= 1;
    if (tma) {
      if (lane == 0) bulk_wait_read1();  // the copy before the last one used this block
    }
    __syncwarp();
    const uint32_t line = block + (uint32_t)(lane * 64), swz = (uint32_t)((lane >> 1) & 3);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float* w = v + 8 * q;
      st_shared_u32x4(line + (((uint32_t)q ^ swz) << 4), pack16x2_from_float(w[0], w[1], f16), pack16x2_from_float(w[2], w[3], f16),
                      pack16x2_from_float(w[4], w[5], f16), pack16x2_from_float(w[6], w[7], f16));
    }
    if (tma) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (row0 < rows && col < cols) tma_store_2d(map, block, col, row0);
        bulk_commit();
      }
    } else {
      __syncwarp();
      const int count = min(32, rows - row0);
      uint16_t* dst = reinterpret_cast<uint16_t*>(base) + (int64_t)row0 * ld + col + lane;
      if (col + lane < cols) {
        for (int r = 0; r < count; ++r, dst += ld) {
          const uint32_t at = block + (uint32_t)(r * 64) + ((((uint32_t)lane >> 3) ^ (uint32_t)((r >> 1) & 3)) << 4) + (uint32_t)(lane & 7) * 2;
          uint16_t h;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(at) : "memory");
          *dst = h;
        }
      }
      __syncwarp();
    }
  }
};

template <int kEpi>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
    dense_pair_kernel(const __grid_constant__ PairMaps maps, const __grid_constant__ PairParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t s_bars[2 * PAIR_STAGES + 5];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ int s_issued[4];  // first CTA's: stages whose copies each producer of the pair has issued
  const uint32_t ring = smem_u32(smem);
  const uint32_t bars = smem_u32(s_bars);
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (PAIR_STAGES + s); };
  auto acc_full_bar = [&](int b) { return bars + 8u * (2 * PAIR_STAGES + b); };
  auto acc_empty_bar = [&](int b) { return bars + 8u * (2 * PAIR_STAGES + 2 + b); };
  const uint32_t drain_bar = bars + 8u * (2 * PAIR_STAGES + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WaitCtx wc = {&s_abort, p.wait_limit_ns};
  const int rank = (int)cluster_ctarank();
  const int pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < PAIR_STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full_bar(b), 1);
      mbar_init(acc_empty_bar(b), 2 * PAIR_EPI_WARPS);
    }
    mbar_init(drain_bar, 1);
    s_abort = 0;
    fence_mbar_init();
    prefetch_tensormap(&maps.job[0].a[0]);
    prefetch_tensormap(&maps.job[0].b[0]);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&s_tmem), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive();  // both CTAs' barriers exist before either is signalled
  cluster_wait();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  pdl_wait();
  pdl_trigger();

  if (warp == 0 || warp == PAIR_WARP_B) {
    // ---- producers: this CTA's halves of A and B; every copy is credited to the first CTA's barrier --------------
    const bool side_b = warp != 0;
    const uint32_t leader_full0 = map_to_cta(full_bar(0), 0);
    const uint32_t dst0 = ring + (side_b ? DENSE_A_BYTES : 0);
    int stage = 0;
    uint32_t phase = 0;
    int issued = 0;
    bool ok = true;
    const uint32_t elected = elect_one();  // (the same lane of a full warp every time)
    const uint32_t go = side_b && p.test_skip_b_loads ? 0u : elected;
    const uint32_t go_announce = !side_b && rank == 0 ? elected : 0u;
    PairTile t;
    for (int i = 0; ok && pair_tile(p, pair, pairs, i, t); ++i) {
      const PairJob& j = p.job[t.job];
      const DenseMaps& m = maps.job[t.job];
      const int half_cols = j.tile_cols / 2;  // this CTA's columns of B
      const int first = !side_b                ? t.row_tile * 256 + rank * 128
                        : kEpi == DENSE_GLU ? t.col_tile * half_cols
                                            : t.col_tile * j.tile_cols + rank * half_cols;
      const bool mn = (side_b ? j.b_mn : j.a_mn) != 0, two = !side_b || half_cols > 64;
      const uint32_t bytes = 2u * (uint32_t)(DENSE_A_BYTES + half_cols * 128);
      const CUtensorMap* map = side_b ? &m.b[kEpi == DENSE_GLU ? rank : 0] : &m.a[t.which];
      const int k_tiles = j.k_tiles;
      int chain_left = j.chain_tiles, kc = 0;
      for (int kt = 0; kt < k_tiles; ++kt) {
        if (!__all_sync(0xffffffffu, mbar_wait(empty_bar(stage), phase ^ 1u, wc, ST_PAIR_EMPTY))) { ok = false; break; }
        const uint32_t fb = leader_full0 + 8u * stage, dst = dst0 + stage * PAIR_STAGE_BYTES;
        expect_tx_if(go_announce, full_bar(stage), bytes);
        if (mn) {
          load_2d_if<true>(go, dst, map, fb, first, kc);
          if (two) load_2d_if<true>(go, dst + DENSE_SLAB, map, fb, first + 64, kc);
        } else {
          load_2d_if<true>(go, dst, map, fb, kc, first);
        }
        ++issued;
        kc += DENSE_BK;
        if (--chain_left == 0) {
          kc = 0;
          map = side_b ? &m.b[1] : &m.a[1];
        }
        if (++stage == PAIR_STAGES) { stage = 0; phase ^= 1u; }
      }
    }
    if (lane == 0) st_shared_cluster(map_to_cta(smem_u32(&s_issued[rank * 2 + (side_b ? 1 : 0)]), 0), (uint32_t)issued);
    __syncwarp();
  } else if (warp == 1) {
    // ---- MMA issuer -------------------------------------------------------------------------------------
    if (rank == 0) {
      constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);  // SBO 1024, version 1, 128-byte swizzle
      const uint32_t a_base = (ring >> 4) & 0x3FFFu, b_base = ((ring + DENSE_A_BYTES) >> 4) & 0x3FFFu;
      auto desc = [](uint32_t lo) { return ((uint64_t)HI << 32) | lo; };
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t go = elect_one();
      PairTile t;
      for (int i = 0; ok && pair_tile(p, pair, pairs, i, t); ++i) {
        const PairJob& j = p.job[t.job];
        const uint32_t acc = tmem + (uint32_t)(i & 1) * 256u;
        const uint32_t a_lo0 = a_base | (j.a_mn ? (uint32_t)(DENSE_SLAB >> 4) << 16 : 1u << 16);
        const uint32_t b_lo0 = b_base | (j.b_mn ? (uint32_t)(DENSE_SLAB >> 4) << 16 : 1u << 16);
        const uint32_t a_step = j.a_mn ? (16u * 128u) >> 4 : 2u, b_step = j.b_mn ? (16u * 128u) >> 4 : 2u;
        const uint32_t idesc = j.idesc;
        const int k_tiles = j.k_tiles;
        if (i >= 2) {
          if (!__all_sync(0xffffffffu, mbar_wait(acc_empty_bar(i & 1), (uint32_t)((i >> 1) - 1) & 1u, wc, ST_PAIR_ACC_EMPTY))) { ok = false; break; }
          tc_fence_after();
        }
        for (int kt = 0; kt < k_tiles; ++kt) {
          bool landed = mbar_try_wait(full_bar(stage), phase);
          if (!landed) landed = mbar_wait(full_bar(stage), phase, wc, ST_PAIR_FULL);
          if (!__all_sync(0xffffffffu, landed)) { ok = false; break; }
          const uint32_t a_lo = a_lo0 + stage * (PAIR_STAGE_BYTES >> 4), b_lo = b_lo0 + stage * (PAIR_STAGE_BYTES >> 4);
#pragma unroll
          for (int q = 0; q < 4; ++q) mma_f16_if<true>(go, acc, desc(a_lo + q * a_step), desc(b_lo + q * b_step), idesc, (kt | q) != 0);
          commit_pair_if(go, empty_bar(stage));
          if (kt + 1 == k_tiles) commit_pair_if(go, acc_full_bar(i & 1));
          if (++stage == PAIR_STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else {
    // ---- epilogue ---------------------------------------------------------------------------------------
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const bool f16 = p.f16 != 0;
    const float unscale = kEpi == DENSE_STORE ? grad_unscale(p.amax) : 1.0f;
    BlockWriter writer = {ring + PAIR_STAGING + (uint32_t)((warp - 2) * 2 * PAIR_BOX), 0, lane, f16};
    PairTile t;
    for (int i = 0; pair_tile(p, pair, pairs, i, t); ++i) {
      const PairJob& j = p.job[t.job];
      const int row0 = t.row_tile * 256 + rank * 128 + quarter * 32;  // this warp's 32 rows
      const int rows = j.rows, cols = j.cols;
      const bool tma = j.tma_store != 0;
      if (!__all_sync(0xffffffffu, mbar_wait<true>(acc_full_bar(i & 1), (uint32_t)(i >> 1) & 1u, wc, ST_PAIR_ACC_FULL))) break;
      tc_fence_after();
      const uint32_t acc = tmem + (uint32_t)(i & 1) * 256u + ((uint32_t)(quarter * 32) << 16);
      const int out_cols = kEpi == DENSE_GLU ? j.tile_cols / 2 : j.tile_cols;  // output columns of the tile
      const int chunks = out_cols / 64;                                          // of 32 columns, in this warp's half
#pragma unroll 1
      for (int c = 0; c < chunks; ++c) {
        __syncwarp();
        float v[32], u[kEpi == DENSE_GLU ? 32 : 1];
        const int in_tile = (half * chunks + c) * 32;
        tmem_ld_32x32(acc + in_tile, v);
        if constexpr (kEpi == DENSE_GLU) tmem_ld_32x32(acc + out_cols + in_tile, u);
        const int col = t.col_tile * out_cols + in_tile;
        tmem_ld_wait();
        reg_fence32(v);
        if constexpr (kEpi == DENSE_GLU) reg_fence32(u);
        if (c == chunks - 1) {
          // the accumulator is in registers: the issuer may overwrite it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(map_to_cta(acc_empty_bar(i & 1), 0));
        }
        if (row0 >= rows || col >= cols) continue;  // (the whole warp)
        if constexpr (kEpi == DENSE_GLU) {
          if (p.pre[0]) {
            writer.write(v, &maps.pre[0], p.pre[0], p.ld_pre[0], tma, row0, rows, col, cols);
            writer.write(u, &maps.pre[1], p.pre[1], p.ld_pre[1], tma, row0, rows, col, cols);
          }
#pragma unroll
          for (int q = 0; q < 32; ++q) v[q] = glu_f(v[q], u[q], p.act);
        } else if constexpr (kEpi == DENSE_LINEAR) {
          if (p.bias) {
            // lane q holds the bias of column q (32 loads per lane instead cost 6 us per tile)
            const int at = min(col + lane, cols - 1);
            const float mine = p.bias_f32 ? __ldg(reinterpret_cast<const float*>(p.bias) + at) : load16(p.bias, at, f16);
#pragma unroll
            for (int q = 0; q < 32; ++q) v[q] += __shfl_sync(0xffffffffu, mine, q);
          }
          if (p.pre[0]) writer.write(v, &maps.pre[0], p.pre[0], p.ld_pre[0], tma, row0, rows, col, cols);
          act_values<32>(v, p.act);
          if (p.residual) writer.add(v, p.residual, p.ld_res, p.vec_res != 0, row0, rows, col, cols);
        } else {
#pragma unroll
          for (int q = 0; q < 32; ++q) v[q] *= unscale;
        }
        writer.write(v, &maps.out[t.job][t.which], j.out[t.which], j.ld_out, tma, row0, rows, col, cols);
      }
    }
    if (lane == 0) bulk_wait_all();  // the copies out of this CTA's shared memory
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *wc.abort_flag) st_shared_cluster(map_to_cta(smem_u32(&s_abort), (uint32_t)(rank ^ 1)), 1u);
  __syncwarp();
  cluster_arrive();  // the other CTA's arrivals and the issuer's products reach this CTA until both are here
  cluster_wait();
  if (*wc.abort_flag) {
    // (in both CTAs or in none: the copies of both are credited to the first, the products' end is told to both)
    if (warp == 0 && rank == 0) drain_copies(full_bar(0), max(max(s_issued[0], s_issued[1]), max(s_issued[2], s_issued[3])), PAIR_STAGES, p.wait_limit_ns);
    if (warp == 1) {
      if (rank == 0) commit_pair_if(elect_one(), drain_bar);
      drain_wait(drain_bar, 0, global_timer_ns(), p.wait_limit_ns);
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------
// Elementwise parts of the backward passes: one read of the incoming gradient and of the saved pre-activations, one
// write of the operand that the two gradient products share, with its rows padded to 8 values so that TMA can read it.
// ---------------------------------------------------------------------------------------
constexpr int GRAD_COLS = 256;  // columns of a block: 32 lanes x 8

// 8 neighbouring 16-bit or float32 values as they lie in memory, and as float32.  `whole`: 16-byte aligned and all there,
// otherwise the first `count` exist and zeros follow.  Loading and unpacking are apart so that every load of a step is on its way
// before the first is used (interleaved with the arithmetic, these kernels ran at 3 TB/s).
struct Raw8 {
  uint4 a, b;  // b: the second half of float32 values
};
template <bool kF32>
__device__ __forceinline__ Raw8 raw8(const void* base, int64_t i, bool whole, int count) {
  Raw8 r;
  r.a = r.b = make_uint4(0, 0, 0, 0);
  if constexpr (kF32) {
    const float* src = reinterpret_cast<const float*>(base) + i;
    if (whole) {
      r.a = __ldg(reinterpret_cast<const uint4*>(src));
      r.b = __ldg(reinterpret_cast<const uint4*>(src) + 1);
    } else {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = j < count ? __float_as_uint(src[j]) : 0u;
      r.a = make_uint4(w[0], w[1], w[2], w[3]);
      r.b = make_uint4(w[4], w[5], w[6], w[7]);
    }
  } else {
    const uint16_t* src = reinterpret_cast<const uint16_t*>(base) + i;
    if (whole) {
      r.a = __ldg(reinterpret_cast<const uint4*>(src));
    } else {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = j < count ? src[j] : 0u;
      r.a = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
    }
  }
  return r;
}
template <bool kF32, bool kF16>
__device__ __forceinline__ void values8(const Raw8& r, float* v) {
  if constexpr (kF32) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
  } else {
    const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 p = unpack16x2(w[j], kF16);
      v[2 * j] = p.x, v[2 * j + 1] = p.y;
    }
  }
}
template <bool kF16>
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack16x2_from_float(v[0], v[1], kF16), pack16x2_from_float(v[2], v[3], kF16), pack16x2_from_float(v[4], v[5], kF16),
                    pack16x2_from_float(v[6], v[7], kF16));
}

// The largest finite magnitude of a block's values goes to *amax (zero before): its bits order like the values, and a maximum does not
// depend on the order.
__device__ __forceinline__ void find_max8(const float* v, uint32_t& top) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = __float_as_uint(v[j]) & 0x7fffffffu;
    if (b < 0x7f800000u) top = max(top, b);
  }
}
__device__ __forceinline__ void publish_max(uint32_t top, uint32_t* amax) {
  __shared__ uint32_t s_top[8];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x < 32) {
    top = __reduce_max_sync(0xffffffffu, threadIdx.x < 8 ? s_top[threadIdx.x] : 0u);
    if (threadIdx.x == 0 && top) atomicMax(amax, top);
  }
}

// dg, du [m, ldo] from dh, gate, up [m, n]: 10 bytes per value, bound by HBM (4096 x 14336: 587 MB).
// They are rounded to the operands' 16 bits, as the tensor cores take both operands in one type; the rounding of each is independent, so
// the gradient products' error grows from one rounding's to two.  fp16 values are scaled (grad_scale); kFind: nothing is
// written, only their largest magnitude is found, in a launch of its own before.
template <int kAct, bool kF16, bool kFind>
__global__ void __launch_bounds__(256)
    glu_grad_kernel(const void* __restrict__ dh, const void* __restrict__ gate, const void* __restrict__ up, int64_t m, int n, int64_t ld_dh,
                    int64_t ld_gate, int64_t ld_up, void* __restrict__ dg, void* __restrict__ du, int64_t ldo, int vec, uint32_t* __restrict__ amax) {
  if (!kFind) pdl_trigger();
  const int c = (int)blockIdx.x * GRAD_COLS + (threadIdx.x & 31) * 8;
  if (!kFind && c >= n) return;
  const bool whole = vec && c + 8 <= n;
  const float scale = kF16 && !kFind ? grad_scale(amax) : 1.0f;
  uint32_t top = 0;
  for (int64_t r = c < n ? (int64_t)blockIdx.y * 8 + (threadIdx.x >> 5) : m; r < m; r += (int64_t)gridDim.y * 8) {
    const Raw8 rd = raw8<false>(dh, r * ld_dh + c, whole, n - c), rg = raw8<false>(gate, r * ld_gate + c, whole, n - c),
               ru = raw8<false>(up, r * ld_up + c, whole, n - c);
    float d[8], g[8], u[8];
    values8<false, kF16>(rd, d);
    values8<false, kF16>(rg, g);
    values8<false, kF16>(ru, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) glu_grad_f(d[j], g[j], u[j], kAct, g[j], u[j]);
    if constexpr (kFind) {
      find_max8(g, top);
      find_max8(u, top);
    } else {
      if constexpr (kF16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] *= scale, u[j] *= scale;
      }
      // (the padding columns of the last 8 are written too: they are part of the padded row)
      *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(dg) + r * ldo + c) = pack8<kF16>(g);
      *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(du) + r * ldo + c) = pack8<kF16>(u);
    }
  }
  if constexpr (kFind) publish_max(top, amax);
}

// dz [m, ldo] = dy act'(z) (dz == NULL: dy is used as it is), and the column sums of the unrounded dz over the block's
// rows: sums [gridDim.y][n].  Every sum has a fixed order: a warp's rows, then the warps, then (next kernel) the blocks.
// Rounding, scale of fp16 values and kFind as in glu_grad_kernel.
template <int kAct, bool kF16, bool kDyF32, bool kFind>
__global__ void __launch_bounds__(256)
    act_grad_kernel(const void* __restrict__ dy, const void* __restrict__ z, int64_t m, int n, int64_t ld_dy, int64_t ld_z, void* __restrict__ dz,
                    int64_t ldo, float* __restrict__ sums, int vec, int64_t rows_per_block, uint32_t* __restrict__ amax) {
  __shared__ float s_part[kFind ? 1 : 8][GRAD_COLS];
  if (!kFind) pdl_trigger();
  const float scale = kF16 && !kFind ? grad_scale(amax) : 1.0f;
  uint32_t top = 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = (int)blockIdx.x * GRAD_COLS + lane * 8;
  float acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
  const int64_t r0 = (int64_t)blockIdx.y * rows_per_block, r1 = min(m, r0 + rows_per_block);
  if (c < n) {
    const bool whole = vec && c + 8 <= n;
    constexpr int kRows = 2;  // in flight per warp
    for (int64_t r = r0 + warp; r < r1; r += 8 * kRows) {
      Raw8 rd[kRows], rz[kRows];
#pragma unroll
      for (int q = 0; q < kRows; ++q) {
        const int64_t row = min(r + 8 * q, r1 - 1);
        rd[q] = raw8<kDyF32>(dy, row * ld_dy + c, whole, n - c);
        if (kAct != B200MOE_ACT_NONE) rz[q] = raw8<false>(z, row * ld_z + c, whole, n - c);
      }
#pragma unroll
      for (int q = 0; q < kRows; ++q) {
        const int64_t row = r + 8 * q;
        if (row >= r1) break;
        float d[8];
        values8<kDyF32, kF16>(rd[q], d);
        if (kAct != B200MOE_ACT_NONE) {
          float g[8];
          values8<false, kF16>(rz[q], g);
#pragma unroll
          for (int j = 0; j < 8; ++j) d[j] *= act_grad_f(g[j], kAct);
        }
        if constexpr (kFind) {
          find_max8(d, top);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[j] += d[j];
          if constexpr (kF16) {
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] *= scale;
          }
          if (dz) *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(dz) + row * ldo + c) = pack8<kF16>(d);
        }
      }
    }
  }
  if constexpr (kFind) {
    publish_max(top, amax);
  } else if (sums) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s_part[warp][lane * 8 + j] = acc[j];
    __syncthreads();
    const int col = (int)blockIdx.x * GRAD_COLS + threadIdx.x;
    if (col < n) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) t += s_part[w][threadIdx.x];
      sums[(int64_t)blockIdx.y * n + col] = t;
    }
  }
}

// out[c] = sum over the blocks' partial sums, in order
__global__ void __launch_bounds__(256) column_sum_kernel(const float* __restrict__ sums, int blocks, int n, float* __restrict__ out) {
  pdl_trigger();
  const int c = (int)blockIdx.x * 256 + threadIdx.x;
  if (c >= n) return;
  float t = 0.0f;
  for (int b = 0; b < blocks; ++b) t += sums[(int64_t)b * n + c];
  out[c] = t;
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

static int dense_encode(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows, int f16) {
  uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows};
  uint64_t strides[1] = {(uint64_t)ld * 2};
  uint32_t box[2] = {(uint32_t)DENSE_BK, (uint32_t)box_rows};
  return encode_map(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, 2, dims, strides, box,
                    CU_TENSOR_MAP_SWIZZLE_128B);
}

// A matrix operand of a product, as it lies in memory: `outer` rows of `inner` contiguous values, pitch `ld`
struct DenseOperand {
  const void* base;
  int64_t outer, inner, ld;
};

struct DenseGemm {
  DenseOperand a[2], b[2];
  bool dual = false;          // a[0], a[1] side by side against b[0]
  bool chained = false;       // a[0] b[0] + a[1] b[1]
  bool stacked = false;       // a[0] b[0] -> out[0], a[1] b[0] -> out[1]
  bool a_mn = false, b_mn = false;
  int64_t rows = 0, cols = 0, red = 0;  // result rows and columns, length of the reduction (of one chain)
  bool trans = false;
  int epi = DENSE_STORE;
  bool segmented = false;
  // what the estimates need to know of the epilogue
  int act = B200MOE_ACT_NONE;
  bool has_residual = false, saves = false;
  bool odd_rows = false;  // some of its arrays have rows that no tensor map takes: the pair kernel writes them 2 bytes at a time
};

// A launch in clusters that may start while its predecessor drains
struct LaunchConfig {
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  LaunchConfig(unsigned grid, unsigned threads, size_t smem, int cluster, cudaStream_t stream) {
    memset(&cfg, 0, sizeof(cfg));
    memset(attr, 0, sizeof(attr));
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
  }
  LaunchConfig(const LaunchConfig&) = delete;
};

template <bool kTrans, int kEpi, bool kSeg>
static int dense_launch_tile(const DenseMaps& maps, const DenseParams& p, unsigned grid, cudaStream_t stream) {
  auto kern = dense_tile_kernel<kTrans, kEpi, kSeg>;
  static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
  int dev = 0;
  B200_CUDA_CHECK(cudaGetDevice(&dev));
  if (!(ready.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    B200_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, DENSE_SMEM_ALONE));
    B200_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    ready.fetch_or(1ull << (dev & 63));
  }
  LaunchConfig c(grid, DENSE_THREADS, (size_t)p.smem_bytes, p.split, stream);
  B200_CUDA_CHECK(cudaLaunchKernelEx(&c.cfg, kern, maps, p));
  return B200MOE_OK;
}

// ---- estimated times in nanoseconds, fitted to both kernels on products of 512 x 1024 to 14336 x 14336 at 1 to 512 tokens ----

// Time that an epilogue adds, per element and SM
static double epilogue_ns(const DenseGemm& g) {
  return 0.05 + (g.epi == DENSE_GLU ? 0.1 : 0.0) + (g.act == B200MOE_ACT_GELU ? 0.08 : (g.act == B200MOE_ACT_NONE ? 0.0 : 0.05)) + (g.has_residual ? 0.1 : 0.0) +
         (g.saves ? 0.1 : 0.0);
}
// A product's operands and result cannot pass faster than HBM's 6500 bytes / ns
static double memory_ns(const DenseGemm& g) {
  const double rows = (double)g.rows * (g.dual || g.stacked ? 2 : 1), red = (double)g.red * (g.chained ? 2 : 1);
  return 2.0 * (rows * red + (double)g.cols * red + rows * (double)g.cols) / 6500.0;
}

// Columns of the tile kernel's tiles (as many as there are, up to 128; an MN-major B comes in slabs of 64) and the CTAs that
// share a tile's reduction.  A stage takes a CTA 190 ns (the issuer's loop) or as long as its bytes take at 160 GB/s for the SM
// and 15.8 TB/s for all of L2; two CTAs run on an SM at once; joining partial sums costs more the more columns and CTAs.
// (Float32 outputs are taken for the same, but their registers leave one CTA to an SM: beyond one round of CTAs these times are
// too short for them and the ring they get is half of what they could have.  The fit had no such case.)
struct TileShape {
  int cols, split;
  int64_t tiles;
  double time;
};
// SMs that clusters of this size can occupy at once with a CTA of the tile kernel to an SM: a cluster lies within one of the chip's groups
// of SMs, whose sizes are no multiple of 4 or 8 and differ between parts (here, of 148 SMs: 33 clusters of 4, 15 of 8), so each device is
// asked once.  0: clusters of this size do not run.
static int cluster_slots(int split, const DeviceInfo* di) {
  if (split <= 2) return std::max(2, di->sm_count / 2 * 2);
  static std::atomic<int> known[64][2];
  int dev = 0, clusters = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  std::atomic<int>& slots = known[dev & 63][split == 8];
  if (slots.load(std::memory_order_relaxed) == 0) {
    auto kern = dense_tile_kernel<true, DENSE_LINEAR, false>;
    LaunchConfig c((unsigned)(split * di->sm_count), DENSE_THREADS, DENSE_SMEM_ALONE, split, nullptr);
    c.cfg.numAttrs = 1;  // (the cluster's size alone)
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, DENSE_SMEM_ALONE) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&clusters, kern, &c.cfg) != cudaSuccess) {
      (void)cudaGetLastError();
      clusters = 0;
    }
    slots.store(clusters > 0 ? clusters * split : -1, std::memory_order_relaxed);
  }
  return std::max(0, slots.load(std::memory_order_relaxed));
}
static TileShape tile_shape(const DenseGemm& g, const DeviceInfo* di) {
  const int64_t tile_rows = g.dual ? 64 : 128;
  const int64_t rows = (g.rows + tile_rows - 1) / tile_rows * (g.stacked ? 2 : 1);
  const int64_t stages = (g.red + DENSE_BK - 1) / DENSE_BK * (g.chained ? 2 : 1);
  const int least = g.b_mn ? 64 : 16;
  TileShape best = {0, 0, 0, 0.0};
  for (int c = 128; c >= least; c /= 2) {
    if (c > least && c / 2 >= g.cols) continue;  // half as many hold them all
    const int64_t tiles = rows * ((g.cols + c - 1) / c);
    const double bytes = DENSE_A_BYTES + c * 128;
    for (int split = 1; split <= DENSE_MAX_SPLIT && split * 4 <= std::max<int64_t>(4, stages); split *= 2) {
      const int64_t ctas = tiles * split, slots = cluster_slots(split, di);
      if (slots < split) continue;
      const int64_t per_sm = (ctas + slots - 1) / slots;
      const double together = per_sm > 1 ? 2.0 : 1.0, rounds = per_sm > 1 ? (double)((per_sm + 1) / 2) : 1.0;
      const double stage = std::max({190.0, together * bytes / 160.0, together * bytes * (double)std::min<int64_t>(ctas, di->sm_count) / 15800.0});
      const double load = std::max(rounds * (double)((stages + split - 1) / split) * stage, memory_ns(g));
      const double join = split > 1 || g.dual ? 1000.0 + 350.0 * split + 25.0 * c : 2000.0 + 8.0 * c;
      const double finish = join + epilogue_ns(g) * 128.0 * c / split * together;
      const double time = 3000.0 + load + finish * (rounds > 1.0 ? 1.4 * rounds : 1.0);
      if (best.cols == 0 || time < best.time) best = {c, split, tiles, time};
    }
  }
  return best;
}

// Shared part of every product: tiles, tensor maps, launch.  `p` arrives with its epilogue fields set.
static int dense_gemm(const DenseGemm& g, DenseParams& p, DeviceInfo* di, cudaStream_t stream) {
  p.rows = (int)g.rows;
  p.cols = (int)g.cols;
  p.a_mn = g.a_mn;
  p.b_mn = g.b_mn;
  p.stacked = g.stacked;
  const int tile_rows = g.dual ? 64 : 128;
  p.row_tiles = (int)((g.rows + tile_rows - 1) / tile_rows);
  p.chain_tiles = (int)((g.red + DENSE_BK - 1) / DENSE_BK);
  p.k_tiles = p.chain_tiles * (g.chained ? 2 : 1);
  TileShape shape = tile_shape(g, di);
  const int C = shape.cols;
  p.tile_cols = C;
  p.split = shape.split;
  p.col_tiles = (int)((g.cols + C - 1) / C);
  const int64_t tiles = shape.tiles;
  p.stage_bytes = DENSE_A_BYTES + C * 128;
  // (a slice of columns per CTA, rounded up to 4)
  const int reduce_bytes = p.split > 1 ? p.split * (((C + p.split - 1) / p.split + 3) / 4 * 4) * 512 : 0;
  // (the loads of a CTA come after about 1.4 us at 80 GB/s and SM: 110 KB in flight, so a CTA alone on its SM takes it all)
  p.smem_bytes = tiles * p.split <= cluster_slots(p.split, di) ? DENSE_SMEM_ALONE : DENSE_SMEM;
  p.reduce_in_ring = p.split > 1 && C == 128 && p.smem_bytes == DENSE_SMEM;
  p.stages = std::min(16, (p.smem_bytes - 1024 - (p.reduce_in_ring ? 0 : reduce_bytes)) / p.stage_bytes);
  p.reduce_offset = p.split > 1 && !p.reduce_in_ring ? p.stages * p.stage_bytes : 0;
  const int cols = C * (g.segmented ? 2 : 1);
  p.tmem_cols = cols <= 32 ? 32 : (cols <= 64 ? 64 : (cols <= 128 ? 128 : 256));
  p.idesc = dense_idesc(128, C, p.f16 != 0, g.a_mn, g.b_mn);
  if (tiles * p.split > 0x7fffffff) return fail(B200MOE_E_SHAPE, "the product has too many tiles");

  DenseMaps maps;
  memset(&maps, 0, sizeof(maps));
  const int na = (g.dual || g.chained || g.stacked) ? 2 : 1, nb = g.chained ? 2 : 1;
  for (int i = 0; i < na; ++i) {
    int rc = dense_encode(&maps.a[i], g.a[i].base, g.a[i].outer, g.a[i].inner, g.a[i].ld, g.a_mn || g.dual ? 64 : 128, p.f16);
    if (rc) return rc;
  }
  for (int i = 0; i < nb; ++i) {
    int rc = dense_encode(&maps.b[i], g.b[i].base, g.b[i].outer, g.b[i].inner, g.b[i].ld, g.b_mn ? 64 : C, p.f16);
    if (rc) return rc;
  }
  const unsigned grid = (unsigned)(tiles * p.split);
  if (g.epi == DENSE_GLU) return dense_launch_tile<true, DENSE_GLU, false>(maps, p, grid, stream);
  if (g.trans && g.segmented) return dense_launch_tile<true, DENSE_LINEAR, true>(maps, p, grid, stream);
  if (g.trans) return dense_launch_tile<true, DENSE_LINEAR, false>(maps, p, grid, stream);
  return dense_launch_tile<false, DENSE_STORE, false>(maps, p, grid, stream);
}

// a matrix that the pair kernel writes in blocks of 32 x 32
static int dense_encode_block(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int f16) {
  uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows};
  uint64_t strides[1] = {(uint64_t)ld * 2};
  uint32_t box[2] = {32, 32};
  return encode_map(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
}

template <int kEpi>
static int dense_launch_pair(const PairMaps& maps, const PairParams& p, int pairs, cudaStream_t stream) {
  auto kern = dense_pair_kernel<kEpi>;
  static std::atomic<uint64_t> ready{0};  // devices whose attribute is set
  int dev = 0;
  B200_CUDA_CHECK(cudaGetDevice(&dev));
  if (!(ready.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    B200_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PAIR_SMEM));
    ready.fetch_or(1ull << (dev & 63));
  }
  LaunchConfig c((unsigned)(2 * pairs), PAIR_THREADS, PAIR_SMEM, 2, stream);
  B200_CUDA_CHECK(cudaLaunchKernelEx(&c.cfg, kern, maps, p));
  return B200MOE_OK;
}

// The pair kernel's launch with tiles of `tile_cols` columns.  A stage of a 256 x 256 tile takes 285 ns (512 cycles of the tensor
// cores), one of a 256 x 128 tile 180 ns (the issuer's loop); a tile's epilogue takes as long as 5 stages and hides behind
// the next tile's, the last one's does not; start and end cost 6 us.
static int64_t pair_tiles(const DenseGemm& g, int tile_cols) {
  const int cols = g.dual ? tile_cols / 2 : tile_cols;
  return ((g.rows + 255) / 256) * (g.stacked ? 2 : 1) * ((g.cols + cols - 1) / cols);
}
static int64_t pair_stages(const DenseGemm& g) { return (g.red + DENSE_BK - 1) / DENSE_BK * (g.chained ? 2 : 1); }
static double pair_time(const DenseGemm* g, int jobs, int tile_cols, int pairs) {
  const double stage = tile_cols == 256 ? 285.0 : 180.0;
  double longest = 0.0, all = 0.0, memory = 0.0, last = 0.0;
  int64_t tiles = 0;
  for (int i = 0; i < jobs; ++i) {
    const double finish = (epilogue_ns(g[i]) - 0.05 + (g[i].odd_rows ? 0.1 : 0.0)) * 128.0 * tile_cols;
    const double products = stage * (double)std::max<int64_t>(5, pair_stages(g[i]));
    const double t = std::max(products, finish);
    longest = std::max(longest, t);
    last = std::max(last, std::min(products, finish));
    all += t * (double)pair_tiles(g[i], tile_cols);
    tiles += pair_tiles(g[i], tile_cols);
    memory += memory_ns(g[i]);
  }
  const double shared = jobs == 1 ? longest * (double)((tiles + pairs - 1) / pairs) : std::max(longest, all / pairs * 1.05);
  return 6000.0 + std::max(shared, memory) + last;
}
static int pair_cols(const DenseGemm* g, int jobs, const DeviceInfo* di, double* time = nullptr) {
  const double wide = pair_time(g, jobs, 256, di->sm_count / 2), narrow = pair_time(g, jobs, 128, di->sm_count / 2);
  if (time) *time = std::min(wide, narrow);
  return narrow < wide ? 128 : 256;
}

// One launch of the pair kernel over one or two products of the same epilogue; operand A's rows are the result's rows.
// `p` arrives with its epilogue fields and each job's outputs and pitch set.
static int dense_pair_gemm(const DenseGemm* g, int jobs, PairParams& p, DeviceInfo* di, cudaStream_t stream) {
  PairMaps maps;
  memset(&maps, 0, sizeof(maps));
  p.jobs = jobs;
  const int tile_cols = pair_cols(g, jobs, di);
  bool tma_store = true;
  for (int i = 0; i < jobs; ++i) tma_store = tma_store && p.job[i].ld_out % 8 == 0 && aligned16(p.job[i].out[0]) && aligned16(p.job[i].out[1]);
  for (int q = 0; q < 2; ++q) tma_store = tma_store && (!p.pre[q] || (aligned16(p.pre[q]) && p.ld_pre[q] % 8 == 0));
  for (int i = 0; i < jobs; ++i) {
    PairJob& j = p.job[i];
    j.rows = (int)g[i].rows;
    j.cols = (int)g[i].cols;
    j.tile_cols = tile_cols;
    j.row_tiles = (int)((g[i].rows + 255) / 256);
    const int out_cols = g[i].dual ? tile_cols / 2 : tile_cols;
    j.col_tiles = (int)((g[i].cols + out_cols - 1) / out_cols);
    j.chain_tiles = (int)((g[i].red + DENSE_BK - 1) / DENSE_BK);
    j.k_tiles = (int)pair_stages(g[i]);
    j.a_mn = g[i].a_mn;
    j.b_mn = g[i].b_mn;
    j.stacked = g[i].stacked;
    const int64_t tiles = pair_tiles(g[i], tile_cols);
    if (tiles > 0x3fffffff) return fail(B200MOE_E_SHAPE, "the product has too many tiles");
    j.tiles = (int)tiles;
    // (8 and 16 row tiles to a group are alike within 2 %; 8 for the plain products, 16 for the gated block measured best)
    j.raster = g[i].dual ? 16 : 8;
    j.idesc = dense_idesc(256, tile_cols, p.f16 != 0, g[i].a_mn, g[i].b_mn);
    const int na = (g[i].chained || g[i].stacked) ? 2 : 1, nb = (g[i].chained || g[i].dual) ? 2 : 1, no = j.stacked ? 2 : 1;
    for (int q = 0; q < na; ++q) {
      int rc = dense_encode(&maps.job[i].a[q], g[i].a[q].base, g[i].a[q].outer, g[i].a[q].inner, g[i].a[q].ld, g[i].a_mn ? 64 : 128, p.f16);
      if (rc) return rc;
    }
    for (int q = 0; q < nb; ++q) {
      int rc = dense_encode(&maps.job[i].b[q], g[i].b[q].base, g[i].b[q].outer, g[i].b[q].inner, g[i].b[q].ld, g[i].b_mn ? 64 : tile_cols / 2, p.f16);
      if (rc) return rc;
    }
    j.tma_store = tma_store;
    if (tma_store) {
      for (int q = 0; q < no; ++q) {
        int rc = dense_encode_block(&maps.out[i][q], j.out[q], j.rows, j.cols, j.ld_out, p.f16);
        if (rc) return rc;
      }
      for (int q = 0; q < 2 && p.pre[q]; ++q) {
        int rc = dense_encode_block(&maps.pre[q], p.pre[q], j.rows, j.cols, p.ld_pre[q], p.f16);
        if (rc) return rc;
      }
    }
  }
  // time of a tile in stages; below 5 its epilogue takes longer than its products
  auto cost = [&](int i) { return std::max(5, p.job[i].k_tiles); };
  if (jobs > 1 && cost(1) > cost(0)) {  // long tiles first, the short ones fill the rest
    std::swap(p.job[0], p.job[1]);
    std::swap(maps.job[0], maps.job[1]);
    std::swap(maps.out[0], maps.out[1]);
  }
  const int64_t total = (int64_t)p.job[0].tiles + (jobs > 1 ? p.job[1].tiles : 0);
  const int pairs = (int)std::max<int64_t>(1, std::min<int64_t>(di->sm_count / 2, total));
  p.full_rounds = p.job[0].tiles / pairs;
  p.rest = p.job[0].tiles % pairs;
  p.early = p.early_tiles = 0;
  if (jobs > 1 && p.rest > 0) {
    // a tile of job 0 lasts as long as this many of job 1
    p.early = std::max(1, (cost(0) + cost(1) / 2) / cost(1));
    p.early_tiles = (int)std::min<int64_t>(p.job[1].tiles, (int64_t)p.early * (pairs - p.rest));
  }
  if (g[0].epi == DENSE_GLU) return dense_launch_pair<DENSE_GLU>(maps, p, pairs, stream);
  if (g[0].epi == DENSE_LINEAR) return dense_launch_pair<DENSE_LINEAR>(maps, p, pairs, stream);
  return dense_launch_pair<DENSE_STORE>(maps, p, pairs, stream);
}

static void pair_params(PairParams& p, const b200moe_dense_args* a) {
  memset(&p, 0, sizeof(p));
  p.test_skip_b_loads = (a->flags & B200MOE_FLAG_TEST_SKIP_B_LOADS) != 0;
  p.f16 = a->dtype == B200MOE_DTYPE_F16;
  p.act = a->act;
  p.wait_limit_ns = a->wait_limit_ms > 0 ? (uint64_t)a->wait_limit_ms * 1000000ull : kWaitLimitNs;
}

// a TMA operand: 16-byte aligned base and pitch
static int check_operand(const char* op, const char* name, const void* p, int64_t ld, int64_t inner) {
  if (!p) return fail(B200MOE_E_NULL, "%s: %s is required", op, name);
  if (ld < inner) return fail(B200MOE_E_SHAPE, "%s: the pitch of %s is below its row length", op, name);
  if (!aligned16(p) || ld % 8 != 0) return fail(B200MOE_E_ALIGN, "%s: %s must start on a 16-byte boundary and have a pitch of a multiple of 8", op, name);
  return B200MOE_OK;
}

static int dense_check_common(const char* op, const b200moe_dense_args* a, bool gated, DeviceInfo** di) {
  if (!a) return fail(B200MOE_E_NULL, "args is NULL");
  if (a->m < 0 || a->n < 1 || a->k < 1 || a->m > 0x7ffffff0 || a->n > 0x3ffffff0 || a->k > 0x3ffffff0)
    return fail(B200MOE_E_SHAPE, "%s: m, n, k = %lld, %lld, %lld out of range", op, (long long)a->m, (long long)a->n, (long long)a->k);
  if (a->k % 8 != 0) return fail(B200MOE_E_SHAPE, "%s: k = %lld must be a multiple of 8", op, (long long)a->k);
  if (a->dtype != B200MOE_DTYPE_BF16 && a->dtype != B200MOE_DTYPE_F16) return fail(B200MOE_E_UNSUPPORTED, "%s: dtype %d", op, a->dtype);
  if (gated ? (a->act != B200MOE_ACT_SWIGLU && a->act != B200MOE_ACT_GEGLU)
            : (a->act != B200MOE_ACT_NONE && a->act != B200MOE_ACT_RELU && a->act != B200MOE_ACT_SILU && a->act != B200MOE_ACT_GELU))
    return fail(B200MOE_E_UNSUPPORTED, "%s: act %d", op, a->act);
  if (a->wait_limit_ms < 0) return fail(B200MOE_E_SHAPE, "%s: wait_limit_ms must not be negative", op);
  int rc = check_operand(op, gated ? "w_gate" : "weight", a->w0, a->ld_w0, a->k);
  if (!rc && gated) rc = check_operand(op, "w_up", a->w1, a->ld_w1, a->k);
  if (!rc && a->m > 0) rc = check_operand(op, "x", a->x, a->ld_x, a->k);
  if (rc) return rc;
  rc = get_device_info(di);
  if (rc) return rc;
  if ((*di)->cc_major != 10) return fail(B200MOE_E_DEVICE, "%s: needs an sm_100 device, found compute capability %d.x", op, (*di)->cc_major);
  return B200MOE_OK;
}

static void dense_params(DenseParams& p, const b200moe_dense_args* a) {
  memset(&p, 0, sizeof(p));
  p.test_skip_b_loads = (a->flags & B200MOE_FLAG_TEST_SKIP_B_LOADS) != 0;
  p.f16 = a->dtype == B200MOE_DTYPE_F16;
  p.act = a->act;
  p.wait_limit_ns = a->wait_limit_ms > 0 ? (uint64_t)a->wait_limit_ms * 1000000ull : kWaitLimitNs;
}

static int dense_forward(const char* op, const b200moe_dense_args* a, bool gated, cudaStream_t stream) {
  DeviceInfo* di = nullptr;
  int rc = dense_check_common(op, a, gated, &di);
  if (rc) return rc;
  if (a->m == 0) return B200MOE_OK;
  if (!a->y) return fail(B200MOE_E_NULL, "%s: the output is required", op);
  if (a->ld_y < a->n || (a->pre0 && a->ld_pre0 < a->n) || (a->pre1 && a->ld_pre1 < a->n)) return fail(B200MOE_E_SHAPE, "%s: an output's pitch is below n", op);
  if (a->residual && a->ld_residual < 0) return fail(B200MOE_E_SHAPE, "%s: the residual's pitch must not be negative", op);
  if (gated && (a->pre0 == nullptr) != (a->pre1 == nullptr)) return fail(B200MOE_E_NULL, "%s: gate and up go together", op);
  if (gated ? a->y_dtype != a->dtype : (a->y_dtype != a->dtype && a->y_dtype != B200MOE_DTYPE_F32))
    return fail(B200MOE_E_UNSUPPORTED, "%s: output dtype %d", op, a->y_dtype);
  if (a->bias && a->bias_dtype != a->dtype && a->bias_dtype != B200MOE_DTYPE_F32) return fail(B200MOE_E_UNSUPPORTED, "%s: bias dtype %d", op, a->bias_dtype);
  DenseParams p;
  dense_params(p, a);
  p.out[0] = a->y;
  p.ld_out = a->ld_y;
  p.pre[0] = a->pre0;
  p.pre[1] = a->pre1;
  p.ld_pre[0] = a->ld_pre0;
  p.ld_pre[1] = a->ld_pre1;
  DenseGemm g;
  g.a[0] = {a->w0, a->n, a->k, a->ld_w0};
  g.b[0] = {a->x, a->m, a->k, a->ld_x};
  g.rows = a->n;
  g.cols = a->m;
  g.red = a->k;
  g.trans = true;
  if (gated) {
    g.a[1] = {a->w1, a->n, a->k, a->ld_w1};
    g.dual = true;
    g.epi = DENSE_GLU;
  } else {
    g.epi = DENSE_LINEAR;
    p.bias = a->bias;
    p.bias_f32 = a->bias_dtype == B200MOE_DTYPE_F32;
    p.residual = a->residual;
    p.ld_res = a->ld_residual;
    p.out_f32 = a->y_dtype == B200MOE_DTYPE_F32;
    g.segmented = p.out_f32 != 0;
    g.act = a->act;
    g.has_residual = a->residual != nullptr;
  }
  g.saves = a->pre0 != nullptr;
  g.odd_rows = a->ld_y % 8 != 0 || !aligned16(a->y) || (a->residual && (a->ld_residual % 8 != 0 || !aligned16(a->residual))) ||
               (a->pre0 && (a->ld_pre0 % 8 != 0 || !aligned16(a->pre0))) || (a->pre1 && (a->ld_pre1 % 8 != 0 || !aligned16(a->pre1)));
  if (a->y_dtype != B200MOE_DTYPE_F32) {
    DenseGemm w;
    w.a[0] = {a->x, a->m, a->k, a->ld_x};
    w.b[0] = {a->w0, a->n, a->k, a->ld_w0};
    w.b[1] = {a->w1, a->n, a->k, a->ld_w1};
    w.dual = gated;
    w.epi = gated ? DENSE_GLU : DENSE_LINEAR;
    w.rows = a->m;
    w.cols = a->n;
    w.red = a->k;
    w.act = g.act;
    w.has_residual = g.has_residual;
    w.saves = g.saves;
    w.odd_rows = g.odd_rows;
    double time = 0.0;
    pair_cols(&w, 1, di, &time);
    if (time < tile_shape(g, di).time) {
      PairParams q;
      pair_params(q, a);
      q.job[0].out[0] = a->y;
      q.job[0].ld_out = a->ld_y;
      q.pre[0] = a->pre0;
      q.pre[1] = a->pre1;
      q.ld_pre[0] = a->ld_pre0;
      q.ld_pre[1] = a->ld_pre1;
      if (!gated) {
        q.bias = a->bias;
        q.bias_f32 = a->bias_dtype == B200MOE_DTYPE_F32;
        q.residual = a->residual;
        q.ld_res = a->ld_residual;
        q.vec_res = aligned16(a->residual) && a->ld_residual % 8 == 0;
      }
      return dense_pair_gemm(&w, 1, q, di, stream);
    }
  }
  return dense_gemm(g, p, di, stream);
}

template <int kAct>
static auto act_grad_of(bool f16, bool dy_f32, bool find) {
  if (find) return dy_f32 ? act_grad_kernel<kAct, true, true, true> : act_grad_kernel<kAct, true, false, true>;
  return f16 ? (dy_f32 ? act_grad_kernel<kAct, true, true, false> : act_grad_kernel<kAct, true, false, false>)
             : (dy_f32 ? act_grad_kernel<kAct, false, true, false> : act_grad_kernel<kAct, false, false, false>);
}

// Blocks of a launch that walks its rows: eight to an SM of a whole chip.  (No device decides it: the workspace's size is asked for before
// there is one, and the order of the column sums does not depend on the device either.)
constexpr int GRAD_BLOCKS = 148 * 8;
// blocks along the rows of act_grad_kernel, and the rows of each
static int grad_row_blocks(int64_t m, int64_t n, int64_t* rows_per_block) {
  const int64_t col_blocks = (n + GRAD_COLS - 1) / GRAD_COLS;
  // (up to 128 rows one block: its sums are the result, and no second kernel is needed)
  int64_t blocks = m <= 128 ? 1 : std::max<int64_t>(1, std::min<int64_t>((m + 31) / 32, GRAD_BLOCKS / std::max<int64_t>(1, col_blocks)));
  *rows_per_block = (m + blocks - 1) / std::max<int64_t>(1, blocks);
  return (int)((m + *rows_per_block - 1) / *rows_per_block);
}

static int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

// dx = sum of dz_i w_i and dw_i = dz_i^T x: one launch of the pair kernel, or a launch each of the kernel that suits it where
// those are estimated to take less time (a weight gradient of few tiles over many tokens shares its reduction in the tile kernel)
static int dense_grad_products(const b200moe_dense_args* a, int count, const void* const* dz, int64_t ld_dz, const uint32_t* amax, DeviceInfo* di,
                               cudaStream_t stream) {
  PairParams q;
  pair_params(q, a);
  q.amax = amax;
  DenseGemm pair[2], tile[2];
  int jobs = 0;
  if (a->dx) {
    // rows = tokens; for the tile kernel rows = the k features of x, columns = tokens.  w [n, k] is MN-major.
    DenseGemm &x = pair[jobs], &t = tile[jobs];
    for (int i = 0; i < count; ++i) {
      x.a[i] = t.b[i] = {dz[i], a->m, a->n, ld_dz};
      x.b[i] = t.a[i] = {i ? a->w1 : a->w0, a->n, a->k, i ? a->ld_w1 : a->ld_w0};
    }
    x.chained = t.chained = count == 2;
    x.b_mn = t.a_mn = true;
    x.rows = t.cols = a->m;
    x.cols = t.rows = a->k;
    x.red = t.red = a->n;
    t.trans = true;
    t.epi = DENSE_LINEAR;
    q.job[jobs].out[0] = a->dx;
    q.job[jobs++].ld_out = a->k;
  }
  if (a->dw0) {
    DenseGemm& w = pair[jobs];
    for (int i = 0; i < count; ++i) w.a[i] = {dz[i], a->m, a->n, ld_dz};
    w.b[0] = {a->x, a->m, a->k, a->ld_x};
    w.stacked = count == 2;
    w.a_mn = w.b_mn = true;
    w.rows = a->n;
    w.cols = a->k;
    w.red = a->m;
    tile[jobs] = w;
    q.job[jobs].out[0] = a->dw0;
    q.job[jobs].out[1] = a->dw1;
    q.job[jobs++].ld_out = a->k;
  }
  if (jobs == 0) return B200MOE_OK;
  double joint = 0.0, apart = 0.0, pair_ns[2] = {0.0, 0.0}, tile_ns[2] = {0.0, 0.0};
  pair_cols(pair, jobs, di, &joint);
  for (int i = 0; i < jobs; ++i) {
    pair_cols(&pair[i], 1, di, &pair_ns[i]);
    tile_ns[i] = tile_shape(tile[i], di).time;
    apart += std::min(pair_ns[i], tile_ns[i]) - (i > 0 ? 2000.0 : 0.0);  // (the second launch starts while the first drains)
  }
  if (joint <= apart) return dense_pair_gemm(pair, jobs, q, di, stream);
  for (int i = 0; i < jobs; ++i) {
    if (pair_ns[i] <= tile_ns[i]) {
      PairParams one = q;
      one.job[0] = q.job[i];
      const int rc = dense_pair_gemm(&pair[i], 1, one, di, stream);
      if (rc) return rc;
      continue;
    }
    DenseParams p;
    dense_params(p, a);
    p.amax = amax;
    p.act = B200MOE_ACT_NONE;
    p.out[0] = q.job[i].out[0];
    p.out[1] = q.job[i].out[1];
    p.ld_out = a->k;
    p.vec_store = aligned16(p.out[0]) && aligned16(p.out[1]);
    const int rc = dense_gemm(tile[i], p, di, stream);
    if (rc) return rc;
  }
  return B200MOE_OK;
}

static int zero_outputs(const b200moe_dense_args* a, bool gated, cudaStream_t stream) {
  // no tokens: the weights' gradients are zero
  if (a->dw0) B200_CUDA_CHECK(cudaMemsetAsync(a->dw0, 0, (size_t)a->n * a->k * 2, stream));
  if (gated && a->dw1) B200_CUDA_CHECK(cudaMemsetAsync(a->dw1, 0, (size_t)a->n * a->k * 2, stream));
  if (!gated && a->dbias) B200_CUDA_CHECK(cudaMemsetAsync(a->dbias, 0, (size_t)a->n * 4, stream));
  return B200MOE_OK;
}

// dz (or dg and du), the partial column sums of the linear form, and in the last 256 bytes the largest magnitude of fp16 values
constexpr int64_t AMAX_BYTES = 256;
static int64_t dense_workspace(int64_t m, int64_t n, bool gated, bool f16) {
  const int64_t ldo = (n + 7) / 8 * 8;
  if (m <= 0) return 0;
  if (gated) return 2 * round256(m * ldo * 2) + (f16 ? AMAX_BYTES : 0);
  int64_t rows_per_block;
  return round256(m * ldo * 2) + round256((int64_t)grad_row_blocks(m, n, &rows_per_block) * n * 4) + AMAX_BYTES;
}
static uint32_t* amax_word(const b200moe_dense_args* a, bool gated, bool f16) {
  return reinterpret_cast<uint32_t*>((uint8_t*)a->workspace + dense_workspace(a->m, a->n, gated, f16) - AMAX_BYTES);
}

}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_gated_ffn(const b200moe_dense_args* a, void* stream) { return dense_forward("gated_ffn", a, true, (cudaStream_t)stream); }

extern "C" int b200moe_linear(const b200moe_dense_args* a, void* stream) { return dense_forward("linear", a, false, (cudaStream_t)stream); }

extern "C" int64_t b200moe_dense_workspace_bytes(int64_t m, int64_t n, int32_t form) {
  return dense_workspace(m, n, (form & 1) != 0, (form & B200MOE_DENSE_WORKSPACE_F16) != 0);
}

extern "C" int b200moe_gated_ffn_backward(const b200moe_dense_args* a, void* stream_v) {
  const char* op = "gated_ffn_backward";
  cudaStream_t stream = (cudaStream_t)stream_v;
  DeviceInfo* di = nullptr;
  int rc = dense_check_common(op, a, true, &di);
  if (rc) return rc;
  if ((a->dw0 == nullptr) != (a->dw1 == nullptr)) return fail(B200MOE_E_NULL, "%s: the two weights' gradients go together", op);
  if (a->m == 0) return zero_outputs(a, true, stream);
  if (!a->dy || !a->pre0 || !a->pre1) return fail(B200MOE_E_NULL, "%s: dh, gate and up are required", op);
  if (a->ld_dy < a->n || a->ld_pre0 < a->n || a->ld_pre1 < a->n) return fail(B200MOE_E_SHAPE, "%s: a pitch is below n", op);
  const int64_t ldo = (a->n + 7) / 8 * 8;
  const bool f16 = a->dtype == B200MOE_DTYPE_F16, geglu = a->act == B200MOE_ACT_GEGLU;
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < dense_workspace(a->m, a->n, true, f16))
    return fail(B200MOE_E_WORKSPACE, "%s: needs %lld bytes of 16-byte aligned workspace", op, (long long)dense_workspace(a->m, a->n, true, f16));
  void* dg = a->workspace;
  void* du = (uint8_t*)a->workspace + round256(a->m * ldo * 2);
  const int vec = aligned16(a->dy) && aligned16(a->pre0) && aligned16(a->pre1) && a->ld_dy % 8 == 0 && a->ld_pre0 % 8 == 0 && a->ld_pre1 % 8 == 0;
  const unsigned col_blocks = (unsigned)((a->n + GRAD_COLS - 1) / GRAD_COLS);
  const int64_t row_blocks = (a->m + 7) / 8;
  uint32_t* amax = f16 ? amax_word(a, true, true) : nullptr;
  if (f16) {
    const dim3 grid(col_blocks, (unsigned)std::max<int64_t>(1, std::min<int64_t>(row_blocks, GRAD_BLOCKS / col_blocks)));
    const auto find = geglu ? glu_grad_kernel<B200MOE_ACT_GEGLU, true, true> : glu_grad_kernel<B200MOE_ACT_SWIGLU, true, true>;
    B200_CUDA_CHECK(cudaMemsetAsync(amax, 0, sizeof(uint32_t), stream));
    find<<<grid, 256, 0, stream>>>(a->dy, a->pre0, a->pre1, a->m, (int)a->n, a->ld_dy, a->ld_pre0, a->ld_pre1, nullptr, nullptr, ldo, vec, amax);
    B200_CUDA_CHECK(cudaGetLastError());
  }
  const dim3 grid(col_blocks, (unsigned)std::min<int64_t>(row_blocks, 32768));
  const auto kern = geglu ? (f16 ? glu_grad_kernel<B200MOE_ACT_GEGLU, true, false> : glu_grad_kernel<B200MOE_ACT_GEGLU, false, false>)
                          : (f16 ? glu_grad_kernel<B200MOE_ACT_SWIGLU, true, false> : glu_grad_kernel<B200MOE_ACT_SWIGLU, false, false>);
  kern<<<grid, 256, 0, stream>>>(a->dy, a->pre0, a->pre1, a->m, (int)a->n, a->ld_dy, a->ld_pre0, a->ld_pre1, dg, du, ldo, vec, amax);
  B200_CUDA_CHECK(cudaGetLastError());
  const void* dz[2] = {dg, du};
  return dense_grad_products(a, 2, dz, ldo, amax, di, stream);
}

extern "C" int b200moe_linear_backward(const b200moe_dense_args* a, void* stream_v) {
  const char* op = "linear_backward";
  cudaStream_t stream = (cudaStream_t)stream_v;
  DeviceInfo* di = nullptr;
  int rc = dense_check_common(op, a, false, &di);
  if (rc) return rc;
  if (a->y_dtype != a->dtype && a->y_dtype != B200MOE_DTYPE_F32) return fail(B200MOE_E_UNSUPPORTED, "%s: dtype %d of dy", op, a->y_dtype);
  if (a->m == 0) return zero_outputs(a, false, stream);
  const bool has_act = a->act != B200MOE_ACT_NONE;
  if (!a->dy || (has_act && !a->pre0)) return fail(B200MOE_E_NULL, "%s: dy, and with an activation the pre-activation, are required", op);
  if (a->ld_dy < a->n || (has_act && a->ld_pre0 < a->n)) return fail(B200MOE_E_SHAPE, "%s: a pitch is below n", op);
  const bool f16 = a->dtype == B200MOE_DTYPE_F16;
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < dense_workspace(a->m, a->n, false, f16))
    return fail(B200MOE_E_WORKSPACE, "%s: needs %lld bytes of 16-byte aligned workspace", op, (long long)dense_workspace(a->m, a->n, false, f16));
  const bool dy_f32 = a->y_dtype == B200MOE_DTYPE_F32;
  int64_t ldo = (a->n + 7) / 8 * 8;
  // without an activation the gradient products read dy itself, where TMA can
  const bool as_is = !has_act && !dy_f32 && aligned16(a->dy) && a->ld_dy % 8 == 0;
  const void* dz = as_is ? a->dy : a->workspace;
  // (an fp16 dy that is only moved into padded rows keeps its values)
  uint32_t* amax = f16 && (has_act || dy_f32) && (a->dx || a->dw0) ? amax_word(a, false, f16) : nullptr;
  if (!as_is || a->dbias) {
    int64_t rows_per_block;
    const int row_blocks = grad_row_blocks(a->m, a->n, &rows_per_block);
    float* sums = !a->dbias ? nullptr : (row_blocks == 1 ? a->dbias : (float*)((uint8_t*)a->workspace + round256(a->m * ldo * 2)));
    const int64_t dy_unit = dy_f32 ? 4 : 8;
    const int vec = aligned16(a->dy) && a->ld_dy % dy_unit == 0 && (!has_act || (aligned16(a->pre0) && a->ld_pre0 % 8 == 0));
    const dim3 grid((unsigned)((a->n + GRAD_COLS - 1) / GRAD_COLS), (unsigned)row_blocks);
    auto launch = [&](bool find) {
      const auto kern = a->act == B200MOE_ACT_RELU   ? act_grad_of<B200MOE_ACT_RELU>(f16, dy_f32, find)
                        : a->act == B200MOE_ACT_SILU ? act_grad_of<B200MOE_ACT_SILU>(f16, dy_f32, find)
                        : a->act == B200MOE_ACT_GELU ? act_grad_of<B200MOE_ACT_GELU>(f16, dy_f32, find)
                                                     : act_grad_of<B200MOE_ACT_NONE>(f16, dy_f32, find);
      kern<<<grid, 256, 0, stream>>>(a->dy, has_act ? a->pre0 : nullptr, a->m, (int)a->n, a->ld_dy, a->ld_pre0, as_is || find ? nullptr : a->workspace, ldo,
                                     find ? nullptr : sums, vec, rows_per_block, amax);
      return cudaGetLastError();
    };
    if (amax) {
      B200_CUDA_CHECK(cudaMemsetAsync(amax, 0, sizeof(uint32_t), stream));
      B200_CUDA_CHECK(launch(true));
    }
    B200_CUDA_CHECK(launch(false));
    if (sums && row_blocks > 1) {
      column_sum_kernel<<<(unsigned)((a->n + 255) / 256), 256, 0, stream>>>(sums, row_blocks, (int)a->n, a->dbias);
      B200_CUDA_CHECK(cudaGetLastError());
    }
  }
  const void* dzs[2] = {dz, nullptr};
  return dense_grad_products(a, 1, dzs, as_is ? a->ld_dy : ldo, amax, di, stream);
}
