// Expert router: the k largest logits of every row, their ids and weights, and the gradient of the logits.
//
//   S(t)    = the k largest l[t, :], larger first, ties to the lowest index; -inf and NaN are never chosen
//   softmax: p_i = exp(l_i - max) / sum_i exp(l_i - max)        sigmoid: p_i = 1 / (1 + exp(-l_i))
//   w_j     = p_{S_j}, or p_{S_j} / sum_S p when renormalised (softmax: the sum over all experts cancels and is not formed)
//   d l     softmax, renormalised:  w_j (g_j - sum_S g w) on S, 0 elsewhere
//           softmax:                p_i (g~_i - sum_S g p), g~ = g on S, 0 elsewhere
//           sigmoid:                g_j p_j (1 - p_j) on S;  renormalised: g_j replaced by (g_j - sum_S g w) / sum_S p
//
// One warp per row, the whole row in registers: one pass over the logits in either direction, statistics in fp32. The
// choice is made on the logits themselves (softmax and sigmoid are increasing), so it does not depend on how an exponential
// rounds. A round of the selection is one 32-bit warp maximum over order-preserving keys and one warp minimum over the
// indices that hold it; only the lane that lost its best entry looks through its registers again.
// No reference counterpart (the reference has no MoE path).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common_host.h"
#include "ptx.cuh"

namespace tb {

bool pdl_enabled();  // api.cu

namespace {

constexpr int kRouteWarps = 8;
constexpr int kRouteMaxExperts = 1024;  // what the dispatch plan kernels take
constexpr int kRouteMaxTopk = 32;       // one lane holds one choice
constexpr unsigned kFull = 0xffffffffu;
constexpr float kNegInf = -__builtin_huge_valf();

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float v, float& o) { o = v; }
__device__ __forceinline__ void from_float(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// Element i of a lane's registers is expert ((i / VEC) * 32 + lane) * VEC + i % VEC: every load and store instruction of a
// warp covers one contiguous run.
template <int VEC>
__device__ __forceinline__ int expert_index(int i, int lane) {
  return ((i / VEC) * 32 + lane) * VEC + (i % VEC);
}

template <typename T, int VPT, int VEC>
__device__ __forceinline__ void load_row(const T* __restrict__ row, int experts, int lane, float (&l)[VPT]) {
#pragma unroll
  for (int i = 0; i < VPT; i += VEC) {
    const int e = expert_index<VEC>(i, lane);
    if (e < experts) {  // VEC divides `experts` when VEC > 1, so a run lies inside the row or outside it as a whole
      const Pack<T, VEC> p = *reinterpret_cast<const Pack<T, VEC>*>(row + e);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float f = to_float(p.v[j]);
        l[i + j] = f > kNegInf ? f : kNegInf;  // NaN never compares greater: it counts as -inf
      }
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) l[i + j] = kNegInf;
    }
  }
}

// Monotonic map of floats (no NaN) to unsigned: -inf -> 0x007fffff, so 0 marks an entry that is not there any more.
// -0 and +0 are equal as numbers and must tie, so both take +0's key.
__device__ __forceinline__ unsigned order_key(float f) {
  const unsigned u = __float_as_uint(f == 0.0f ? 0.0f : f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
constexpr unsigned kKeyNegInf = 0x007fffffu;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(kFull, v, s);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, s));
  return v;
}

template <typename T, int VPT, int VEC>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const T* __restrict__ logits, long long stride, long long tokens,
                                                                 int experts, int topk, int sigmoid, int renorm,
                                                                 float* __restrict__ weights, int* __restrict__ ids) {
  const int lane = threadIdx.x & 31;
  const long long t = static_cast<long long>(blockIdx.x) * kRouteWarps + (threadIdx.x >> 5);
  griddep_launch_dependents();
  griddep_wait();
  if (t >= tokens) return;
  float l[VPT];
  load_row<T, VPT, VEC>(logits + t * stride, experts, lane, l);

  unsigned gone = 0;  // bit i: element i has been chosen
  unsigned best = 0;
  int best_e = 0;
  auto rescan = [&]() {
    best = 0;
    best_e = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {  // ascending experts per lane: a tie keeps the first
      const unsigned k = ((gone >> i) & 1u) ? 0u : order_key(l[i]);
      if (k > best) {
        best = k;
        best_e = expert_index<VEC>(i, lane);
      }
    }
  };
  rescan();
  float mine = kNegInf, top = 0.0f;
  int mine_e = -1;
  for (int j = 0; j < topk; ++j) {
    const unsigned k = __reduce_max_sync(kFull, best);
    if (k <= kKeyNegInf) break;  // only -inf left: the other choices stay empty
    const int e = static_cast<int>(__reduce_min_sync(kFull, best == k ? static_cast<unsigned>(best_e) : 0xffffffffu));
    const float v = __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
    if (j == 0) top = v;
    if (lane == j) {
      mine = v;
      mine_e = e;
    }
    if (best == k && best_e == e) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (expert_index<VEC>(i, lane) == e) gone |= 1u << i;
      rescan();
    }
  }

  float w;
  if (sigmoid) {
    w = 1.0f / (1.0f + expf(-mine));  // -inf gives 0
  } else {
    w = expf(mine - top);
  }
  if (mine_e < 0) w = 0.0f;
  if (renorm) {
    const float s = warp_sum(w);
    w = s > 0.0f || s != s ? w / s : 0.0f;
  } else if (!sigmoid) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) s += expf(l[i] - top);
    s = warp_sum(s);
    w = mine_e < 0 ? 0.0f : w / s;
  }
  if (lane < topk) {
    weights[t * topk + lane] = w;
    ids[t * topk + lane] = mine_e;
  }
}

// Backward: `weights` and `ids` are what the forward pass returned, `grad` the gradient of the weights. The dense modes
// (softmax without renormalisation) read the logits again and form max and sum anew; the others only need the choice.
template <typename T, int VPT, int VEC>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_bwd_kernel(const T* __restrict__ logits, long long stride, long long tokens, int experts, int topk, int sigmoid, int renorm,
                 const float* __restrict__ weights, const int* __restrict__ ids, const float* __restrict__ grad,
                 T* __restrict__ dlogits) {
  const int lane = threadIdx.x & 31;
  const long long t = static_cast<long long>(blockIdx.x) * kRouteWarps + (threadIdx.x >> 5);
  griddep_launch_dependents();
  griddep_wait();
  if (t >= tokens) return;
  const T* row = logits + t * stride;
  float g = 0.0f, w = 0.0f;
  int e = -1;
  if (lane < topk) {
    e = ids[t * topk + lane];
    if (e >= experts) e = -1;
    if (e >= 0) {
      g = grad[t * topk + lane];
      w = weights[t * topk + lane];
    }
  }
  float d;  // gradient of this lane's chosen logit (softmax without renormalisation: before the dense part)
  float p[VPT];
  float gp = 0.0f;
  if (sigmoid) {
    float s = w;
    if (renorm) {
      s = e >= 0 ? 1.0f / (1.0f + expf(-to_float(row[e]))) : 0.0f;
      const float total = warp_sum(s), gw = warp_sum(g * w);
      g = total > 0.0f ? (g - gw) / total : 0.0f;
    }
    d = e >= 0 ? g * s * (1.0f - s) : 0.0f;
  } else if (renorm) {
    d = w * (g - warp_sum(g * w));
  } else {
    load_row<T, VPT, VEC>(row, experts, lane, p);
    float top = kNegInf, s = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) top = fmaxf(top, p[i]);
    top = warp_max(top);
    if (top == kNegInf) top = 0.0f;  // a row with nothing to choose: every p is 0
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      p[i] = expf(p[i] - top);
      s += p[i];
    }
    s = warp_sum(s);
    const float inv = s > 0.0f ? 1.0f / s : 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) p[i] *= inv;
    d = g * w;
    gp = warp_sum(d);
  }
  const bool dense = !sigmoid && !renorm;
  float out[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) out[i] = dense ? -p[i] * gp : 0.0f;
  for (int j = 0; j < topk; ++j) {
    const int ej = __shfl_sync(kFull, e, j);
    const float dj = __shfl_sync(kFull, d, j);
    if (ej >= 0 && (ej / VEC) % 32 == lane) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (expert_index<VEC>(i, lane) == ej) out[i] += dj;
    }
  }
  T* drow = dlogits + t * static_cast<long long>(experts);
#pragma unroll
  for (int i = 0; i < VPT; i += VEC) {
    const int c = expert_index<VEC>(i, lane);
    if (c < experts) {
      Pack<T, VEC> o;
#pragma unroll
      for (int j = 0; j < VEC; ++j) from_float(out[i + j], o.v[j]);
      *reinterpret_cast<Pack<T, VEC>*>(drow + c) = o;
    }
  }
}

// One row per warp, programmatic dependent launch as the GEMM kernels use it.
template <typename K, typename... Args>
int launch_rows(K kernel, long long rows, cudaStream_t st, const char* what, Args... args) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(static_cast<unsigned>((rows + kRouteWarps - 1) / kRouteWarps), 1, 1);
  lc.blockDim = dim3(kRouteWarps * 32, 1, 1);
  lc.stream = st;
  cudaLaunchAttribute attr[1];
  lc.attrs = attr;
  lc.numAttrs = 0;
  if (pdl_enabled()) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.numAttrs = 1;
  }
  cudaError_t e = cudaLaunchKernelEx(&lc, kernel, args...);
  if (e != cudaSuccess) return cuda_fail(e, what);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return TB_OK;
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

template <typename T, int VPT, int VEC>
int route_launch(const RouteCall& c) {
  if (c.grad == nullptr)
    return launch_rows(route_kernel<T, VPT, VEC>, c.tokens, c.stream, "route_kernel launch", static_cast<const T*>(c.logits),
                       c.stride, c.tokens, c.experts, c.topk, c.sigmoid, c.renorm, c.weights, c.ids);
  return launch_rows(route_bwd_kernel<T, VPT, VEC>, c.tokens, c.stream, "route_bwd_kernel launch",
                     static_cast<const T*>(c.logits), c.stride, c.tokens, c.experts, c.topk, c.sigmoid, c.renorm,
                     static_cast<const float*>(c.weights), static_cast<const int*>(c.ids), c.grad, static_cast<T*>(c.dlogits));
}

// Registers per lane: the smallest power of two that covers the row. Loads are as wide as rows allow: up to 16 bytes where
// every row starts on that boundary and holds whole runs, single elements otherwise.
template <typename T, int VPT>
int route_vec(const RouteCall& c) {
  constexpr int kWide = VPT < static_cast<int>(16 / sizeof(T)) ? VPT : static_cast<int>(16 / sizeof(T));
  if constexpr (kWide > 1) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(c.logits) | reinterpret_cast<uintptr_t>(c.dlogits) |
                           (c.tokens > 1 ? static_cast<uintptr_t>(c.stride) * sizeof(T) : 0);
    if (bits % (kWide * sizeof(T)) == 0 && c.experts % kWide == 0) return route_launch<T, VPT, kWide>(c);
  }
  return route_launch<T, VPT, 1>(c);
}

template <typename T>
int route_type(const RouteCall& c) {
  if (c.experts <= 32) return route_vec<T, 1>(c);
  if (c.experts <= 64) return route_vec<T, 2>(c);
  if (c.experts <= 128) return route_vec<T, 4>(c);
  if (c.experts <= 256) return route_vec<T, 8>(c);
  if (c.experts <= 512) return route_vec<T, 16>(c);
  return route_vec<T, 32>(c);
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
