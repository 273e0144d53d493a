// The gate in front of the experts: top-k choice with its weights, and the gradient of the logits.
//
//   choice   the topk largest of l + 0 (or, with a selection bias b, of score(l) + b), ties to the lowest index;
//            a logit of -inf is never chosen, and a slot that finds no expert gets id -1 and weight 0
//   weights  w_j = scale * score_j, or normalised over the chosen ones scale * score_j / sum_i score_i, with
//            score = softmax over the row, or sigmoid.  The bias decides the choice only.
//
// The normalised sigmoid is formed from u_i = e^(min(l_i, 0) - m) / (1 + e^-|l_i|) with m the largest min(l_j, 0) of the
// choice: sigmoid(l_i) = e^m u_i, so the quotient of two numbers that may both underflow is never formed.
#include <type_traits>

#include "b200moe.h"
#include "common.cuh"

namespace b200moe {

constexpr int ROUTER_MAX_EXPERTS = 1024;
constexpr int ROUTER_MAX_TOPK = 32;

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
  if (dtype == B200MOE_DTYPE_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == B200MOE_DTYPE_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int64_t i, float v, int dtype) {
  if (dtype == B200MOE_DTYPE_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == B200MOE_DTYPE_F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Keys that order like the values (NaN above everything, 0 and -0 equal: the addition turns -0 into 0 and any NaN into the
// positive one); a key that is not above kNever, that of -inf, is never chosen
constexpr uint32_t kNever = 0x007FFFFFu;
constexpr uint64_t kNever64 = 0x000FFFFFFFFFFFFFull;
__device__ __forceinline__ uint32_t order_key(float v) {
  const int32_t b = __float_as_int(v + 0.0f);
  return (uint32_t)(b ^ ((b >> 31) | (int32_t)0x80000000));
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ uint64_t order_key64(double v) {
  if (v != v) return ~0ull;
  const int64_t b = __double_as_longlong(v + 0.0);
  return (uint64_t)(b ^ ((b >> 63) | (int64_t)(1ull << 63)));
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// over groups of kLanes lanes; NaN stays
template <int kLanes = 32>
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = kLanes / 2; d > 0; d >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
template <int kLanes = 32, typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int d = kLanes / 2; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ float sigmoid_exact_f(float v) { return 1.0f / (1.0f + expf(-v)); }

// Weight of the choice that this lane holds (lanes without one: chosen = false), the choices of a row in a group of kLanes
// lanes; called by the whole warp.  row_max / row_sum: of the whole row, for the softmax that is not normalised over the choice.
template <int kLanes>
__device__ __forceinline__ float choice_weight(float logit, bool chosen, int sigmoid, int normalize, float scale, float row_max, float row_sum) {
  if (normalize) {
    const float a = chosen ? (sigmoid && !(logit != logit) ? fminf(logit, 0.0f) : logit) : -INFINITY;
    const float m = warp_max<kLanes>(a);
    float e = chosen ? expf(a - m) : 0.0f;
    if (sigmoid && chosen) e /= 1.0f + expf(-fabsf(logit));
    const float s = warp_sum<kLanes>(e);
    return chosen ? scale * (e / s) : 0.0f;
  }
  if (!chosen) return 0.0f;
  return scale * (sigmoid ? sigmoid_exact_f(logit) : expf(logit - row_max) / row_sum);
}

// One warp per row; a lane holds kVec neighbouring experts of every 32 kVec.
//
// With more than 32 experts the choice goes by candidates: the topk-th largest of the lanes' own maxima is a lower bound of the
// topk-th largest value, and what reaches it (about topk + 2 of 256) is packed one to a lane and ranked by
// counting.  Of a biased sigmoid the lanes hold a float32 score that is off by less than 2e-6 (1 + |score|), so the bound
// is lowered by twice that; where two neighbours of the ranking are nearer than that to one another, the scores of all candidates
// are formed in 64 bits.  Rows with more than 32 candidates, and biased softmax scores (whose sum over the row is needed in
// 64 bits), take the maxima one after the other.
template <int kPerLane>
struct RowLayout {
  static constexpr int kVec = kPerLane >= 4 ? 4 : 1;
  static __device__ __forceinline__ int expert(int lane, int i) { return (i / kVec) * 32 * kVec + lane * kVec + i % kVec; }
  static __device__ __forceinline__ int lane(int expert) { return expert / kVec % 32; }
  static __device__ __forceinline__ int slot(int expert) { return expert / (32 * kVec) * kVec + expert % kVec; }
};

// (six blocks to an SM instead of four: 23.7 -> 22.0 us for 32768 x 256 with a bias; the warps wait for one another's loads and votes)
template <int kPerLane, bool kBias>
__global__ void __launch_bounds__(256, kPerLane <= 8 ? 6 : (kPerLane == 16 ? 4 : 2))
    router_topk_kernel(const void* __restrict__ logits, int dtype, int64_t rows, int experts, int64_t ld, const float* __restrict__ bias, int topk,
                       int sigmoid, int normalize, float scale, int vec, float* __restrict__ weights, int32_t* __restrict__ ids) {
  using Row = RowLayout<kPerLane>;
  __shared__ int2 s_choice[8][32];
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  int2* choice = s_choice[threadIdx.x >> 5];  // key, expert
  float v[kPerLane];
  if (Row::kVec == 4 && vec) {  // (experts a multiple of 4, rows aligned)
#pragma unroll
    for (int i = 0; i < kPerLane; i += 4) {
      const int e = Row::expert(lane, i);
      v[i] = v[(i + 1) % kPerLane] = v[(i + 2) % kPerLane] = v[(i + 3) % kPerLane] = -INFINITY;
      if (e < experts) {
        if (dtype == B200MOE_DTYPE_F32) {
          const float4 w = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(logits) + row * ld + e));
          v[i] = w.x, v[(i + 1) % kPerLane] = w.y, v[(i + 2) % kPerLane] = w.z, v[(i + 3) % kPerLane] = w.w;
        } else {
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(logits) + row * ld + e));
          const float2 lo = unpack16x2(w.x, dtype == B200MOE_DTYPE_F16), hi = unpack16x2(w.y, dtype == B200MOE_DTYPE_F16);
          v[i] = lo.x, v[(i + 1) % kPerLane] = lo.y, v[(i + 2) % kPerLane] = hi.x, v[(i + 3) % kPerLane] = hi.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) v[i] = Row::expert(lane, i) < experts ? load_any(logits, row * ld + Row::expert(lane, i), dtype) : -INFINITY;
  }
  float row_max = -INFINITY, row_sum = 1.0f;
  if (!sigmoid && !normalize) {
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) row_max = max_nan(row_max, v[i]);
    row_max = warp_max(row_max);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) s += v[i] == -INFINITY ? 0.0f : expf(v[i] - row_max);
    row_sum = warp_sum(s);
  }
  int my_id = -1;
  float my_logit = -INFINITY;
  bool done = false;
  if (kPerLane > 1 && (!kBias || sigmoid)) {
    uint32_t key[kPerLane], best = kNever;
    float offset[kBias ? kPerLane : 1];
    if constexpr (kBias) {
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) offset[i] = 0.0f;
      if (Row::kVec == 4 && vec) {
#pragma unroll
        for (int i = 0; i < kPerLane; i += 4) {
          if (Row::expert(lane, i) < experts) {
            const float4 w = __ldg(reinterpret_cast<const float4*>(bias + Row::expert(lane, i)));
            offset[i] = w.x, offset[(i + 1) % kPerLane] = w.y, offset[(i + 2) % kPerLane] = w.z, offset[(i + 3) % kPerLane] = w.w;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
          if (Row::expert(lane, i) < experts) offset[i] = __ldg(bias + Row::expert(lane, i));
      }
    }
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      float value = v[i];
      if constexpr (kBias) value = v[i] == -INFINITY ? v[i] : rcp_approx(1.0f + ex2_approx(v[i] * -1.4426950408889634f)) + offset[i];
      key[i] = order_key(value);
      best = max(best, key[i]);
    }
    uint32_t bound = kNever;
    for (int j = 0; j < topk; ++j) {
      bound = __reduce_max_sync(0xffffffffu, best);
      if (best == bound) best = kNever;
    }
    bool fits = true;
    if (kBias && bound > kNever) {
      const float b = key_value(bound);
      fits = fabsf(b) < INFINITY;  // neither NaN nor infinite
      bound = order_key(b - 4e-6f * (1.0f + fabsf(b)));
    }
    bound = max(bound, kNever + 1u);
    int count = 0;
    const unsigned before = (1u << lane) - 1;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const bool in = key[i] >= bound;
      const unsigned who = __ballot_sync(0xffffffffu, in);
      const int at = count + __popc(who & before);
      if (in && at < 32) choice[at] = make_int2((int)key[i], Row::expert(lane, i));
      count += __popc(who);
    }
    __syncwarp();
    if (fits && count <= 32) {
      const int2 mine = choice[lane];  // (lanes beyond the count hold what is not used)
      int place = 0;
      for (int q = 0; q < count; ++q) {
        const int2 other = choice[q];
        place += (uint32_t)other.x > (uint32_t)mine.x || (other.x == mine.x && other.y < mine.y);
      }
      __syncwarp();
      if (lane < count) choice[place] = mine;  // the places are a permutation of the candidates
      __syncwarp();
      if constexpr (kBias) {
        // (a NaN or an infinity is near nothing and needs no digits)
        const float score = key_value((uint32_t)choice[lane].x), next = key_value((uint32_t)choice[min(lane + 1, 31)].x);
        if (__any_sync(0xffffffffu, lane + 1 < count && score - next <= 4e-6f * (1.0f + fabsf(score)))) {
          uint64_t wide = 0;
          if (lane < count) wide = order_key64(1.0 / (1.0 + exp(-(double)load_any(logits, row * ld + mine.y, dtype))) + (double)bias[mine.y]);
          place = 0;
          for (int q = 0; q < count; ++q) {
            const uint64_t other = __shfl_sync(0xffffffffu, wide, q);
            const int id = __shfl_sync(0xffffffffu, mine.y, q);
            place += other > wide || (other == wide && id < mine.y);
          }
          __syncwarp();
          if (lane < count) choice[place] = mine;
          __syncwarp();
        }
      }
      if (lane < min(count, topk)) {
        my_id = choice[lane].y;
        my_logit = kBias ? load_any(logits, row * ld + my_id, dtype) : key_value((uint32_t)choice[lane].x);
      }
      done = true;
    }
  }
  if (!done) {
    // 32-bit keys of the logits, or 64-bit keys of the biased scores: those decide between neighbours that differ in the
    // last bits of a float32, so they are formed in 64 bits
    using Key = typename std::conditional<kBias, uint64_t, uint32_t>::type;
    Key key[kPerLane];
    if constexpr (kBias) {
      double wide[kPerLane], top = -INFINITY, sum = 0.0;
      if (!sigmoid) {
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) top = fmax(top, (double)v[i]);
        for (int d = 16; d > 0; d >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, d));
      }
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        wide[i] = v[i] == -INFINITY ? 0.0 : (sigmoid ? 1.0 / (1.0 + exp(-(double)v[i])) : exp((double)v[i] - top));
        sum += wide[i];
      }
      if (!sigmoid) sum = warp_sum(sum);
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const int e = Row::expert(lane, i);
        key[i] = v[i] == -INFINITY ? kNever64 : order_key64((sigmoid ? wide[i] : wide[i] / sum) + (double)(e < experts ? bias[e] : 0.0f));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) key[i] = order_key(v[i]);
    }
    const Key never = kBias ? (Key)kNever64 : (Key)kNever;
    for (int j = 0; j < topk; ++j) {
      Key best = never;
      int at = 0;
      float logit = 0.0f;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i)
        if (key[i] > best) best = key[i], at = i, logit = v[i];
      Key top;
      if constexpr (kBias) {
        const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
        const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
        top = (uint64_t)hi << 32 | lo;
      } else {
        top = __reduce_max_sync(0xffffffffu, best);
      }
      if (top <= never) break;  // nothing left that may be chosen
      const int id = __reduce_min_sync(0xffffffffu, best == top ? Row::expert(lane, at) : 0x7fffffff);
      const float l = __shfl_sync(0xffffffffu, logit, Row::lane(id));
      if (lane == j) my_id = id, my_logit = l;
      if (lane == Row::lane(id)) {
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
          if (i == Row::slot(id)) key[i] = never;
      }
    }
  }
  const float w = choice_weight<32>(my_logit, my_id >= 0, sigmoid, normalize, scale, row_max, row_sum);
  if (lane < topk) {
    weights[row * topk + lane] = w;
    ids[row * topk + lane] = my_id;
  }
}

// dlogits [rows, experts] from the gradient of the weights and the choice.  With c the chosen set and dw' = scale dw:
//   softmax, normalised   dl_i = w_i (dw_i - sum_c w_j dw_j / scale)              (i in c, else 0)
//   sigmoid, normalised   the same times 1 - sigmoid(l_i)
//   sigmoid               dl_i = dw'_i s_i (1 - s_i)
//   softmax               dl_e = p_e (dw'_e - sum_c p_j dw'_j)                   (every e; dw'_e = 0 outside c)
// An expert that occurs twice gets the sum of both gradients.  A row's choice sits in kLanes lanes, 32 / kLanes rows to a warp
// (the whole-row softmax takes a warp for each); the rows of a warp are cleared as one piece.
template <int kLanes>
__global__ void __launch_bounds__(256)
    router_grad_kernel(const float* __restrict__ dweights, const void* __restrict__ logits, int dtype, const int32_t* __restrict__ ids, int64_t rows,
                       int experts, int64_t ld, int topk, int sigmoid, int normalize, float scale, void* __restrict__ dlogits) {
  constexpr int kRows = 32 / kLanes;
  const int lane = threadIdx.x & 31;
  const int64_t row0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * kRows;
  if (row0 >= rows) return;
  const int64_t row = row0 + lane / kLanes;
  const int j = lane % kLanes;
  const bool mine = row < rows && j < topk;
  int id = mine ? ids[row * topk + j] : -1;
  if (id >= experts) id = -1;
  const bool chosen = id >= 0;
  const float logit = chosen ? load_any(logits, row * ld + id, dtype) : -INFINITY;
  const float dw = chosen ? dweights[row * topk + j] : 0.0f;
  const bool whole_row = kLanes == 32 && !sigmoid && !normalize;
  float row_max = -INFINITY, row_sum = 1.0f;
  if (whole_row) {
    for (int e = lane; e < experts; e += 32) row_max = max_nan(row_max, load_any(logits, row * ld + e, dtype));
    row_max = warp_max(row_max);
    float s = 0.0f;
    for (int e = lane; e < experts; e += 32) {
      const float v = load_any(logits, row * ld + e, dtype);
      s += v == -INFINITY ? 0.0f : expf(v - row_max);
    }
    row_sum = warp_sum(s);
  }
  const float w = choice_weight<kLanes>(logit, chosen, sigmoid, normalize, scale, row_max, row_sum);
  const float dot = warp_sum<kLanes>(w * dw);
  float g = normalize ? w * (dw - (scale != 0.0f ? dot / scale : 0.0f)) : w * dw;
  if (sigmoid) g *= sigmoid_exact_f(-logit);
  if (!chosen) g = 0.0f;
  float total = g;
  const unsigned same = __match_any_sync(0xffffffffu, chosen ? (lane / kLanes) << 16 | id : -1 - lane);
  if (__any_sync(0xffffffffu, __popc(same) > 1)) {
    total = 0.0f;
    for (int q = 0; q < kLanes; ++q) {
      const int other = __shfl_sync(0xffffffffu, id, q, kLanes);
      const float v = __shfl_sync(0xffffffffu, g, q, kLanes);
      if (other == id) total += v;
    }
  }
  if (whole_row) {
    for (int e = lane; e < experts; e += 32) {
      const float l = load_any(logits, row * ld + e, dtype);
      store_any(dlogits, row * experts + e, l != -INFINITY ? -(expf(l - row_max) / row_sum) * dot : 0.0f, dtype);
    }
  } else {
    const int64_t size = dtype == B200MOE_DTYPE_F32 ? 4 : 2;
    const int count = (int)min((int64_t)kRows, rows - row0) * experts;
    uint8_t* dst = reinterpret_cast<uint8_t*>(dlogits) + row0 * experts * size;
    if (experts % 8 == 0) {  // rows of a multiple of 16 bytes
      for (int q = lane; q < count * (int)size / 16; q += 32) reinterpret_cast<uint4*>(dst)[q] = make_uint4(0, 0, 0, 0);
    } else {
      for (int q = lane; q < count; q += 32) store_any(dst, q, 0.0f, dtype);
    }
  }
  __syncwarp();  // the rows are written before their chosen entries are
  if (chosen) {
    if (whole_row && logit != -INFINITY) total -= (expf(logit - row_max) / row_sum) * dot;
    store_any(dlogits, row * experts + id, total, dtype);
  }
}

static int router_check(const char* op, const void* logits, int dtype, int64_t rows, int32_t experts, int64_t ld, int32_t topk, int32_t score) {
  if (rows < 0 || experts < 1 || experts > ROUTER_MAX_EXPERTS || ld < experts)
    return fail(B200MOE_E_SHAPE, "%s: rows %lld, experts %d (at most %d), pitch %lld", op, (long long)rows, experts, ROUTER_MAX_EXPERTS, (long long)ld);
  if (topk < 1 || topk > experts || topk > ROUTER_MAX_TOPK) return fail(B200MOE_E_SHAPE, "%s: topk %d (1 to %d, at most the experts)", op, topk, ROUTER_MAX_TOPK);
  if (dtype != B200MOE_DTYPE_F32 && dtype != B200MOE_DTYPE_BF16 && dtype != B200MOE_DTYPE_F16) return fail(B200MOE_E_UNSUPPORTED, "%s: dtype %d", op, dtype);
  if (score != B200MOE_SCORE_SOFTMAX && score != B200MOE_SCORE_SIGMOID) return fail(B200MOE_E_UNSUPPORTED, "%s: score function %d", op, score);
  if (rows > 0x3fffffff8ll) return fail(B200MOE_E_SHAPE, "%s: too many rows", op);
  if (rows > 0 && !logits) return fail(B200MOE_E_NULL, "%s: logits are required", op);
  return B200MOE_OK;
}

template <int kPerLane>
static void router_launch(const void* logits, int dtype, int64_t rows, int experts, int64_t ld, const float* bias, int topk, int sigmoid, int normalize,
                          float scale, float* weights, int32_t* ids, cudaStream_t stream) {
  const unsigned grid = (unsigned)((rows + 7) / 8);
  const int vec = experts % 4 == 0 && ld % 4 == 0 && (uintptr_t)logits % 16 == 0 && (uintptr_t)bias % 16 == 0;
  if (bias) router_topk_kernel<kPerLane, true><<<grid, 256, 0, stream>>>(logits, dtype, rows, experts, ld, bias, topk, sigmoid, normalize, scale, vec, weights, ids);
  else router_topk_kernel<kPerLane, false><<<grid, 256, 0, stream>>>(logits, dtype, rows, experts, ld, bias, topk, sigmoid, normalize, scale, vec, weights, ids);
}

}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_router_topk(const void* logits, int32_t dtype, int64_t rows, int32_t experts, int64_t ld, const float* bias, int32_t topk,
                                   int32_t score, int32_t normalize, float scale, float* weights, int32_t* ids, void* stream_v) {
  int rc = router_check("router_topk", logits, dtype, rows, experts, ld, topk, score);
  if (rc || rows == 0) return rc;
  if (!weights || !ids) return fail(B200MOE_E_NULL, "router_topk: weights and ids are required");
  cudaStream_t stream = (cudaStream_t)stream_v;
  const int sig = score == B200MOE_SCORE_SIGMOID;
#define B200_ROUTER(V) router_launch<V>(logits, dtype, rows, experts, ld, bias, topk, sig, normalize != 0, scale, weights, ids, stream)
  if (experts <= 32) B200_ROUTER(1);
  else if (experts <= 64) B200_ROUTER(2);
  else if (experts <= 128) B200_ROUTER(4);
  else if (experts <= 256) B200_ROUTER(8);
  else if (experts <= 512) B200_ROUTER(16);
  else B200_ROUTER(32);
#undef B200_ROUTER
  B200_CUDA_CHECK(cudaGetLastError());
  return B200MOE_OK;
}

extern "C" int b200moe_router_topk_backward(const float* dweights, const void* logits, int32_t dtype, const int32_t* ids, int64_t rows, int32_t experts,
                                            int64_t ld, int32_t topk, int32_t score, int32_t normalize, float scale, void* dlogits, void* stream_v) {
  int rc = router_check("router_topk_backward", logits, dtype, rows, experts, ld, topk, score);
  if (rc || rows == 0) return rc;
  if (!dweights || !ids || !dlogits) return fail(B200MOE_E_NULL, "router_topk_backward: dweights, ids and dlogits are required");
  if ((uintptr_t)dlogits & 15) return fail(B200MOE_E_ALIGN, "router_topk_backward: dlogits must start on a 16-byte boundary");
  const bool whole_row = score == B200MOE_SCORE_SOFTMAX && !normalize;
  const int lanes = whole_row || topk > 16 ? 32 : (topk > 8 ? 16 : 8);
  const unsigned grid = (unsigned)((rows + 8 * (32 / lanes) - 1) / (8 * (32 / lanes)));
#define B200_ROUTER_GRAD(L)                                                                                                                       \
  router_grad_kernel<L><<<grid, 256, 0, (cudaStream_t)stream_v>>>(dweights, logits, dtype, ids, rows, experts, ld, topk, score == B200MOE_SCORE_SIGMOID, \
                                                                  normalize != 0, scale, dlogits)
  if (lanes == 8) B200_ROUTER_GRAD(8);
  else if (lanes == 16) B200_ROUTER_GRAD(16);
  else B200_ROUTER_GRAD(32);
#undef B200_ROUTER_GRAD
  B200_CUDA_CHECK(cudaGetLastError());
  return B200MOE_OK;
}
