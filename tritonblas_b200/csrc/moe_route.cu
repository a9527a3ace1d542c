// Expert router: the k largest logits of every row, their ids and weights, and the gradient of the logits.
//
//   S(t)    = the k largest l[t, :], larger first, ties to the lowest index; -inf and NaN are never chosen
//   softmax: p_i = exp(l_i - max) / sum_i exp(l_i - max)        sigmoid: p_i = 1 / (1 + exp(-l_i))
//   w_j     = p_{S_j}, or p_{S_j} / sum_S p when renormalised (softmax: the sum over all experts cancels and is not formed)
//   d l     softmax, renormalised:  w_j (g_j - sum_S g w) on S, 0 elsewhere
//           softmax:                p_i (g~_i - sum_S g p), g~ = g on S, 0 elsewhere
//           sigmoid:                g_j w_j (1 - p_j) on S;  renormalised: g_j replaced by g_j - sum_S g w
//             (w_j = p_j, or p_j / sum_S p, is what the forward pass returned; 1 - p_j = 1 / (1 + exp(l_j)) is formed from the
//             logit, since a rounded p_j next to 1 has none of its bits)
//
// A row is held in the registers of 4 to 32 lanes, eight logits each (16 or 32 above 256 experts), so a warp works on up to
// eight rows at once; one pass over the logits in either direction, statistics in fp32. The choice is made on the logits
// themselves (softmax and sigmoid are increasing), so it does not depend on how an exponential rounds: every logit becomes an
// integer that orders like it, with the complement of its index below (16-bit logits leave 13 bits of a 32-bit word for that,
// fp32 ones take 64 bits), so a maximum is the next choice and ties go to the lowest index by themselves. Every lane sorts its
// eight keys once; a round is a maximum over the lanes' first keys and a shift in the lane that held it.
// What bounds it is the number of instructions per row, then the latency of a launch: 32771 rows of 256 bf16 logits, top-8, softmax
// over all experts, 36 us forward and gradient (592 and 420 warp instructions a row, 86 and 79 % of the issue slots; the bytes alone:
// 5.6 us); 16384 x 64: 5.0 us; a launch of three rows: 2.6 us. The exponentials are expf: the fast form took 33 us instead of 36, but
// its error grows with the distance from the row's maximum.
// No reference counterpart (the reference has no MoE path).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common_host.h"
#include "ptx.cuh"
#include "token_ops.cuh"

namespace tb {

namespace {

constexpr int kRouteWarps = 8;
constexpr int kRouteMaxExperts = 1024;  // what the dispatch plan kernels take
constexpr int kRouteMaxTopk = 32;
constexpr unsigned kFull = 0xffffffffu;
constexpr float kNegInf = -__builtin_huge_valf();

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float v, float& o) { o = v; }
__device__ __forceinline__ void from_float(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC > 16 ? 16 : sizeof(T) * VEC) Pack {
  T v[VEC];
};

// Element i of a lane is expert ((i / VEC) * LANES + sub) * VEC + i % VEC, sub being the lane's place among the row's LANES.
template <int LANES, int VEC>
__device__ __forceinline__ int expert_index(int i, int sub) {
  return ((i / VEC) * LANES + sub) * VEC + (i % VEC);
}

// NaN never compares greater: it becomes -inf here, as do the places behind the last expert.
template <typename T, int LANES, int VPT, int VEC>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int experts, int sub, bool in_range, float (&l)[VPT]) {
#pragma unroll
  for (int i = 0; i < VPT; i += VEC) {
    const int e = expert_index<LANES, VEC>(i, sub);
    if (in_range && e < experts) {  // VEC divides `experts` when VEC > 1, so a run lies inside the row or outside it as a whole
      const Pack<T, VEC> p = *reinterpret_cast<const Pack<T, VEC>*>(row + e);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float f = to_float(p.v[j]);
        l[i + j] = f > kNegInf ? f : kNegInf;
      }
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) l[i + j] = kNegInf;
    }
  }
}

// Keys: order of the value first, then the complement of the index; 0 is "nothing" (-inf, NaN, already taken).
constexpr unsigned kIndexMask = 0x1fffu;
__device__ __forceinline__ unsigned order_bits(float f) {  // increasing in f; -0 counts as +0
  const int s = __float_as_int(f + 0.0f);
  return static_cast<unsigned>(s ^ ((s >> 31) | 0x80000000));
}
__device__ __forceinline__ float order_value(unsigned o) {
  return __uint_as_float((o & 0x80000000u) ? (o ^ 0x80000000u) : ~o);
}
template <typename T>
struct Key {  // 16-bit logits: their fp32 images have at least 13 zero bits at the end
  using type = unsigned;
  static __device__ __forceinline__ type make(float f, int e) {
    return f > kNegInf ? ((order_bits(f) & ~kIndexMask) | (kIndexMask - static_cast<unsigned>(e))) : 0u;
  }
  static __device__ __forceinline__ int index(type k) { return static_cast<int>(kIndexMask - (k & kIndexMask)); }
  static __device__ __forceinline__ float value(type k) {
    const unsigned o = k & ~kIndexMask;
    return order_value((o & 0x80000000u) ? o : (o | kIndexMask));
  }
};
template <>
struct Key<float> {
  using type = unsigned long long;
  static __device__ __forceinline__ type make(float f, int e) {
    return f > kNegInf ? ((static_cast<type>(order_bits(f)) << 32) | (kIndexMask - static_cast<unsigned>(e))) : 0ull;
  }
  static __device__ __forceinline__ int index(type k) { return static_cast<int>(kIndexMask - (static_cast<unsigned>(k) & kIndexMask)); }
  static __device__ __forceinline__ float value(type k) { return order_value(static_cast<unsigned>(k >> 32)); }
};

template <int LANES>
__device__ __forceinline__ unsigned lanes_max(unsigned v) {
  if constexpr (LANES == 32) {
    return __reduce_max_sync(kFull, v);
  } else {
#pragma unroll
    for (int s = LANES / 2; s > 0; s >>= 1) v = max(v, __shfl_xor_sync(kFull, v, s));
    return v;
  }
}
template <int LANES>
__device__ __forceinline__ unsigned long long lanes_max(unsigned long long v) {
  if constexpr (LANES == 32) {
    const unsigned hi = __reduce_max_sync(kFull, static_cast<unsigned>(v >> 32));
    const unsigned lo = __reduce_max_sync(kFull, static_cast<unsigned>(v >> 32) == hi ? static_cast<unsigned>(v) : 0u);
    return (static_cast<unsigned long long>(hi) << 32) | lo;
  } else {
#pragma unroll
    for (int s = LANES / 2; s > 0; s >>= 1) v = max(v, __shfl_xor_sync(kFull, v, s));
    return v;
  }
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int s = LANES / 2; s > 0; s >>= 1) v += __shfl_xor_sync(kFull, v, s);
  return v;
}

// Eight keys in descending order: odd-even merge sort, 19 exchanges.
template <typename K>
__device__ __forceinline__ void sort8(K (&a)[8]) {
  auto exchange = [&](int i, int j) {
    const K hi = max(a[i], a[j]), lo = min(a[i], a[j]);
    a[i] = hi;
    a[j] = lo;
  };
  exchange(0, 1); exchange(2, 3); exchange(4, 5); exchange(6, 7);
  exchange(0, 2); exchange(1, 3); exchange(4, 6); exchange(5, 7);
  exchange(1, 2); exchange(5, 6);
  exchange(0, 4); exchange(1, 5); exchange(2, 6); exchange(3, 7);
  exchange(2, 4); exchange(3, 5);
  exchange(1, 2); exchange(3, 4); exchange(5, 6);
}

template <typename T, int LANES, int VPT, int VEC>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const T* __restrict__ logits, long long stride, long long tokens,
                                                                 int experts, int topk, int sigmoid, int renorm,
                                                                 float* __restrict__ weights, int* __restrict__ ids) {
  using K = typename Key<T>::type;
  constexpr int kRows = 32 / LANES;  // rows per warp
  __shared__ K s_choice[kRouteWarps][kRows][kRouteMaxTopk];
  __shared__ float s_score[kRouteWarps][kRows][kRouteMaxTopk];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % LANES, group = lane / LANES;
  const long long t = (static_cast<long long>(blockIdx.x) * kRouteWarps + warp) * kRows + group;
  const bool live = t < tokens;  // lanes without a row go along with empty ones
  griddep_launch_dependents();
  griddep_wait();
  float l[VPT];
  load_row<T, LANES, VPT, VEC>(logits + (live ? t * stride : 0), experts, sub, live, l);
  K a[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) a[i] = Key<T>::make(l[i], expert_index<LANES, VEC>(i, sub));
  K* choice = s_choice[warp][group];
  float* score = s_score[warp][group];
  if constexpr (VPT == 8) {
    sort8(a);
    for (int j = 0; j < topk; ++j) {
      const K best = lanes_max<LANES>(a[0]);
      if (sub == 0) choice[j] = best;
      if (a[0] == best) {
#pragma unroll
        for (int i = 0; i + 1 < VPT; ++i) a[i] = a[i + 1];
        a[VPT - 1] = 0;
      }
    }
  } else {  // more keys per lane than rounds, mostly: look for the lane's next key when its first one is taken
    K first = a[0];
#pragma unroll
    for (int i = 1; i < VPT; ++i) first = max(first, a[i]);
    for (int j = 0; j < topk; ++j) {
      const K best = lanes_max<LANES>(first);
      if (sub == 0) choice[j] = best;
      if (first == best) {
        first = 0;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          if (a[i] == best) a[i] = 0;
          first = max(first, a[i]);
        }
      }
    }
  }
  __syncwarp();
  const float top = choice[0] != 0 ? Key<T>::value(choice[0]) : 0.0f;
  // Renormalised sigmoid scores are formed over exp(m), m = min(top, 0), which cancels in the quotient: below -88 the scores
  // themselves leave fp32's range, their quotients do not. With m = 0 this is the plain 1 / (1 + exp(-l)).
  float m = 0.0f, unit = 1.0f;
  if (sigmoid && renorm) {
    m = fminf(top, 0.0f);
    unit = expf(m);
  }
  float sum = 0.0f;
  for (int j = sub; j < topk; j += LANES) {
    const K k = choice[j];
    float s = 0.0f;
    if (k != 0) s = sigmoid ? 1.0f / (unit + expf(m - Key<T>::value(k))) : expf(Key<T>::value(k) - top);
    score[j] = s;
    sum += s;
  }
  if (renorm) {
    sum = lanes_sum<LANES>(sum);
    if (sum == 0.0f) sum = 1.0f;  // nothing to choose
  } else if (sigmoid) {
    sum = 1.0f;
  } else {
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) sum += expf(l[i] - top);
    sum = lanes_sum<LANES>(sum);
  }
  if (live) {
    for (int j = sub; j < topk; j += LANES) {
      const K k = choice[j];
      weights[t * topk + j] = k != 0 ? score[j] / sum : 0.0f;
      ids[t * topk + j] = k != 0 ? Key<T>::index(k) : -1;
    }
  }
}

// Backward: `weights` and `ids` are what the forward pass returned, `grad` the gradient of the weights. The dense mode (softmax
// without renormalisation) reads the logits again: the first choice holds the row's maximum and, in its weight, the reciprocal
// of the sum, so p_i = exp(l_i - l_first) w_first needs no reduction. The chosen places meet the dense part in shared memory.
template <typename T, int LANES, int VPT, int VEC>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_bwd_kernel(const T* __restrict__ logits, long long stride, long long tokens, int experts, int topk, int sigmoid, int renorm,
                 const float* __restrict__ weights, const int* __restrict__ ids, const float* __restrict__ grad,
                 T* __restrict__ dlogits) {
  constexpr int kRows = 32 / LANES;
  __shared__ alignas(16) float s_row[kRouteWarps][kRows][LANES * VPT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % LANES, group = lane / LANES;
  const long long t = (static_cast<long long>(blockIdx.x) * kRouteWarps + warp) * kRows + group;
  const bool live = t < tokens;
  const bool dense = !sigmoid && !renorm;
  griddep_launch_dependents();
  griddep_wait();
  const T* row = logits + (live ? t * stride : 0);
  const long long c0 = live ? t * topk : 0;
  float p[VPT];
  if (dense) load_row<T, LANES, VPT, VEC>(row, experts, sub, live, p);
  float* buf = s_row[warp][group];
#pragma unroll
  for (int i = 0; i < VPT; i += 4) *reinterpret_cast<float4*>(buf + (i / 4 * LANES + sub) * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
  // one of the choices: id (-1: none), gradient and weight; most rows have at most one per lane, which is read once
  struct Choice {
    int e;
    float g, w;
  };
  auto chosen = [&](int j) {
    Choice c = {-1, 0.0f, 0.0f};
    if (live && j < topk) c.e = ids[c0 + j];
    if (c.e >= experts) c.e = -1;
    if (c.e >= 0) {
      c.g = grad[c0 + j];
      c.w = weights[c0 + j];
    }
    return c;
  };
  auto complement_of = [&](int e) { return 1.0f / (1.0f + expf(to_float(row[e]))); };
  const Choice mine = chosen(sub);
  float dot = 0.0f;  // sum of g w
  for (int j = sub; j < topk; j += LANES) {
    const Choice c = j == sub ? mine : chosen(j);
    dot += c.g * c.w;
  }
  dot = lanes_sum<LANES>(dot);
  __syncwarp();
  for (int j = sub; j < topk; j += LANES) {
    const Choice c = j == sub ? mine : chosen(j);
    if (c.e < 0) continue;
    float d = c.w * (renorm ? c.g - dot : c.g);
    if (sigmoid) d *= complement_of(c.e);
    buf[c.e] = d;
  }
  float first = 0.0f, inv = 0.0f;
  if (dense) {
    const int e = __shfl_sync(kFull, mine.e, group * LANES);
    inv = __shfl_sync(kFull, mine.w, group * LANES) * dot;  // nothing chosen: 0
    first = e >= 0 ? to_float(row[e]) : 0.0f;
  }
  __syncwarp();
  if (!live) return;
  T* drow = dlogits + t * static_cast<long long>(experts);
#pragma unroll
  for (int i = 0; i < VPT; i += VEC) {
    const int c = expert_index<LANES, VEC>(i, sub);
    if (c < experts) {
      Pack<T, VEC> o;
      float v[VEC];
      if constexpr (VEC == 8) {
        const float4 lo = *reinterpret_cast<const float4*>(buf + c), hi = *reinterpret_cast<const float4*>(buf + c + 4);
        v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
        v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
      } else {
        v[0] = buf[c];
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float d = v[j];
        if (dense) d -= expf(p[i + j] - first) * inv;
        from_float(d, o.v[j]);
      }
      *reinterpret_cast<Pack<T, VEC>*>(drow + c) = o;
    }
  }
}

struct RouteCall {
  const void* logits;
  long long stride, tokens;
  int experts, topk, sigmoid, renorm;
  float* weights;
  int* ids;
  const float* grad;  // null: forward
  void* dlogits;
  cudaStream_t stream;
};

template <typename T, int LANES, int VPT, int VEC>
int route_launch(const RouteCall& c) {
  constexpr int kPerBlock = kRouteWarps * (32 / LANES);
  const long long blocks = (c.tokens + kPerBlock - 1) / kPerBlock;
  if (c.grad == nullptr)
    return launch_token_kernel(route_kernel<T, LANES, VPT, VEC>, dim3(static_cast<unsigned>(blocks)), kRouteWarps * 32, 0, 0, c.stream,
                               "route_kernel launch", static_cast<const T*>(c.logits), c.stride, c.tokens, c.experts, c.topk, c.sigmoid,
                               c.renorm, c.weights, c.ids);
  return launch_token_kernel(route_bwd_kernel<T, LANES, VPT, VEC>, dim3(static_cast<unsigned>(blocks)), kRouteWarps * 32, 0, 0, c.stream,
                             "route_bwd_kernel launch", static_cast<const T*>(c.logits), c.stride, c.tokens, c.experts, c.topk, c.sigmoid,
                             c.renorm, static_cast<const float*>(c.weights), static_cast<const int*>(c.ids), c.grad,
                             static_cast<T*>(c.dlogits));
}

// Loads are eight elements wide where every row starts on a 16-byte boundary and holds whole runs of eight, single elements
// otherwise.
template <typename T, int LANES, int VPT>
int route_vec(const RouteCall& c) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(c.logits) | reinterpret_cast<uintptr_t>(c.dlogits) |
                         (c.tokens > 1 ? static_cast<uintptr_t>(c.stride) * sizeof(T) : 0);
  if (bits % 16 == 0 && c.experts % 8 == 0) return route_launch<T, LANES, VPT, 8>(c);
  return route_launch<T, LANES, VPT, 1>(c);
}

template <typename T>
int route_type(const RouteCall& c) {
  if (c.experts <= 32) return route_vec<T, 4, 8>(c);
  if (c.experts <= 64) return route_vec<T, 8, 8>(c);
  if (c.experts <= 128) return route_vec<T, 16, 8>(c);
  if (c.experts <= 256) return route_vec<T, 32, 8>(c);
  if (c.experts <= 512) return route_vec<T, 32, 16>(c);
  return route_vec<T, 32, 32>(c);
}

int route_call(const RouteCall& c, int dtype) {
  if (c.tokens < 0 || c.experts < 1 || c.experts > kRouteMaxExperts || c.topk < 1 || c.topk > c.experts ||
      c.topk > kRouteMaxTopk || c.tokens > 0x7fffffffLL * kRouteWarps || (c.tokens > 1 && c.stride < c.experts))
    return TB_ERR_INVALID;
  if (dtype != TB_DTYPE_F16 && dtype != TB_DTYPE_BF16 && dtype != TB_DTYPE_F32) return TB_ERR_UNSUPPORTED;
  if (c.tokens == 0) return TB_OK;
  if (c.logits == nullptr || c.weights == nullptr || c.ids == nullptr) return TB_ERR_INVALID;
  const uintptr_t es = dtype == TB_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(c.logits) % es || reinterpret_cast<uintptr_t>(c.dlogits) % es ||
      reinterpret_cast<uintptr_t>(c.weights) % 4 || reinterpret_cast<uintptr_t>(c.ids) % 4 ||
      reinterpret_cast<uintptr_t>(c.grad) % 4)
    return TB_ERR_ALIGNMENT;
  if (dtype == TB_DTYPE_F16) return route_type<__half>(c);
  if (dtype == TB_DTYPE_BF16) return route_type<__nv_bfloat16>(c);
  return route_type<float>(c);
}

}  // namespace
}  // namespace tb

extern "C" int tb_moe_route(const void* logits, int32_t dtype, int64_t row_stride, int64_t tokens, int32_t num_experts,
                            int32_t topk, int32_t sigmoid, int32_t renormalize, float* weights, int32_t* ids, void* stream) {
  tb::RouteCall c = {logits, row_stride, tokens, num_experts, topk, sigmoid != 0, renormalize != 0,
                     weights, ids, nullptr, nullptr, static_cast<cudaStream_t>(stream)};
  return tb::route_call(c, dtype);
}

extern "C" int tb_moe_route_backward(const void* logits, int32_t dtype, int64_t row_stride, int64_t tokens, int32_t num_experts,
                                     int32_t topk, int32_t sigmoid, int32_t renormalize, const float* weights,
                                     const int32_t* ids, const float* grad_weights, void* grad_logits, void* stream) {
  if (tokens > 0 && (grad_weights == nullptr || grad_logits == nullptr)) return TB_ERR_INVALID;
  if (tokens == 0) return TB_OK;
  tb::RouteCall c = {logits, row_stride, tokens, num_experts, topk, sigmoid != 0, renormalize != 0,
                     const_cast<float*>(weights), const_cast<int32_t*>(ids), grad_weights, grad_logits,
                     static_cast<cudaStream_t>(stream)};
  return tb::route_call(c, dtype);
}
