// A whole mixture-of-experts feed-forward for a few tokens:
//     out[t] = sum_j w[t, j] * W2_e ( silu(G_e x_t) * (U_e x_t) ),   e = ids[t, j],   W1_e = [G_e | U_e]
//
// With at most 128 tokens every weight of an expert meets a handful of rows, so the layer is bound by reading the chosen
// experts' weights once: (distinct experts) * 3 * ffn * hidden * 2 bytes. Two launches:
//   moe_mlp_plan_kernel  one CTA (one warp up to 32 pairs): the distinct (expert, token) rows in expert order, the counters
//                        of the next launch zeroed;
//   moe_mlp_kernel       one persistent CTA per SM that works through three kinds of units, taken in order from a counter:
//     1  (expert, tile of ffn)     D[feature, token] = W1 tile . X^T, silu(gate) * up in the epilogue, h in 16-bit pairs;
//     2  (row group, tile of hidden) D[hidden, row]  = W2 tile . H^T, times the routing weight, fp32 to the workspace;
//     3  (run of the output)       the sum over a token's rows in slot order, one cast.
// The weights stand on the 64- or 128-row side of the tensor-core tile and the tokens on its narrow side, so a stage of the
// shared-memory ring is almost only weights. A unit of the second kind waits for its expert's units of the first kind (a
// counter per expert), one of the third kind for all units of the second. The weight loader does not: it runs ahead into the
// second kind's weights while the first kind still drains, so HBM never pauses between the projections.
//
// Nothing here needs the CTAs to be resident together. Units are taken in increasing order by CTAs that run, and a unit only
// waits for units with smaller numbers, which are then being worked on by CTAs that run.
//
// Rounding: sums, activation, routing weights and the sum over experts are fp32. The tensor core takes h in 16 bits, so h is
// kept as two 16-bit halves, h = hi + lo with lo = round(h - hi), and multiplied by both: the MMAs double, the bytes do not,
// and the result stays as close to the formula as its own rounding allows (a single 16-bit h would double the squared error).
// fp16 has neither the range nor the small numbers for that, so there the halves stand in units of their own, 2^8 and 2^-3,
// which the second epilogue multiplies back in (each half has its own columns of the product): h is held to 2^-22 relative or
// 2^-28 absolute, whichever is more, up to 65504 * 2^8; above that it is infinite. The floor is chosen against the output's own
// smallest step, 2^-24: rows of W2 with a norm of up to about 10 add less than half of it. (Without the units the floor was
// 2^-25, 3e-3 of an h of 1e-5, and the limit 65504.) bf16 has fp32's range: its units are 1.
// No reference counterpart (the reference has no MoE path).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common_host.h"
#include "ptx.cuh"
#include "token_ops.cuh"

namespace tb {

namespace {

constexpr int kMlpMaxTokens = 128;
constexpr int kMlpMaxTopk = 32;
constexpr int kMlpMaxExperts = 1024;
constexpr int kMlpMaxPairs = kMlpMaxTokens * kMlpMaxTopk;
constexpr int kMlpThreads = 7 * 32;  // four epilogue warps, weight loader, MMA issuer, activation loader
constexpr int kWarpWeights = 4, kWarpMma = 5, kWarpAct = 6;
constexpr int kQueueDepth = 4;
constexpr int kQueueConsumers = 6;  // MMA issuer, activation loader, four epilogue warps
constexpr int kMaxStages = 10;  // 160 KB of weights ahead: more only lengthens every other round trip to memory
constexpr int kRowBytes = 128;      // K extent of a stage: one 128-byte swizzle row
constexpr int kStageK = 64;         // the same in 16-bit elements
// Slabs of 64 K elements per stage: every stage carries at least 16 KB of weights. The roles spend about 380 clocks per stage
// on waits and branches that nothing hides; with 8 KB stages that was more than the 350 clocks HBM needs for one (measured at
// one token, 64-row tiles: 33 GB/s per SM, 44 with 16 KB).
__host__ __device__ constexpr int mlp_slabs(int m) { return m == 64 ? 2 : 1; }

// Workspace: int32 words, then h (16-bit, two planes), then the weighted rows (fp32).
struct MlpLayout {
  // word offsets
  static constexpr int kNumExperts = 0;   // distinct experts
  static constexpr int kNumGroups = 2;    // row groups: at most group_cap rows of one expert
  static constexpr int kNextUnit = 4;     // counters
  static constexpr int kRowsDone = 5;     // units of the second kind that are complete, times the four epilogue warps
  static constexpr int kLists = 8;
  int pairs, experts, groups;             // capacities
  __host__ __device__ int expert_done() const { return kLists; }                       // [experts] units of the first kind done, times four
  __host__ __device__ int expert_id() const { return expert_done() + experts; }        // [experts] id of the i-th distinct one
  __host__ __device__ int expert_off() const { return expert_id() + experts; }         // [experts + 1] first row
  __host__ __device__ int group_slot() const { return expert_off() + experts + 1; }    // [groups] distinct expert of the group
  __host__ __device__ int group_expert() const { return group_slot() + groups; }       // [groups] its id
  __host__ __device__ int group_off() const { return group_expert() + groups; }        // [groups] first row
  __host__ __device__ int group_end() const { return group_off() + groups; }           // [groups] one past the last row
  __host__ __device__ int row_token() const { return group_end() + groups; }           // [pairs]
  __host__ __device__ int row_weight() const { return row_token() + pairs; }           // [pairs] fp32
  __host__ __device__ int pair_row() const { return row_weight() + pairs; }            // [pairs] row of a (token, slot), -1 = none
  __host__ __device__ long long words() const { return pair_row() + pairs; }
};

struct MlpParams {
  MlpLayout lay;
  int* ws;
  int tokens, topk, hidden, ffn;
  int n1;           // columns of the first kind: tokens rounded up to the MMA's granularity
  int group_cap;    // rows of a group
  int stages, stage_bytes;
  int act1_bytes, act2_bytes;  // shared memory of one slab of activations of either kind
  int acc_stride, tmem_cols;
  int f_tiles, h_tiles;  // units per expert / row group
  int quads_per_thread;  // third kind: float4 runs of one token's output per thread
  int runs;              // third kind: units per token
  void* h;               // [row][hi, lo][ffn]
  float* y;
  void* out;
  long long out_stride;
  int out_vec;           // rows of `out` start on 8-byte boundaries
  int bf16;
  uint32_t idesc;        // without the rows and columns
  int* status;
  unsigned long long timeout_ns;
};

// ------------------------------------------------------------------------------------------------------------ plan
// ids of both widths; an id outside [0, num_experts) routes nowhere. The same expert twice in one token's list is one row
// with the weights added (in slot order). The order of an expert's rows depends on the order of atomics; every row is one
// column of the products, computed alike wherever it stands, and the sum over a token's rows goes by slot, so no result
// depends on it.
// One thread per expert: 256 where that is enough, since the kernel is a chain of barriers and round trips on the layer's critical
// path.
template <int kPlanThreads>
__global__ void __launch_bounds__(kPlanThreads)
moe_mlp_plan_kernel(const void* __restrict__ ids, int is64, const float* __restrict__ weights, int tokens, int topk, int num_experts,
                    int group_cap, MlpLayout lay, int* __restrict__ ws) {
  __shared__ int s_id[kMlpMaxPairs];
  __shared__ float s_weight[kMlpMaxPairs];
  __shared__ int s_count[kPlanThreads];
  __shared__ int s_cursor[kPlanThreads];
  __shared__ int s_scan[3][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pairs = tokens * topk;
  griddep_launch_dependents();  // the layer kernel touches no memory before this one is through
  griddep_wait();
  s_count[tid] = 0;
  for (int f = tid; f < pairs; f += kPlanThreads) {
    const long long e = is64 ? static_cast<const long long*>(ids)[f] : static_cast<long long>(static_cast<const int*>(ids)[f]);
    s_weight[f] = weights[f];
    s_id[f] = (e >= 0 && e < num_experts) ? static_cast<int>(e) : -1;
  }
  __syncthreads();
  for (int f = tid; f < pairs; f += kPlanThreads) {
    const int e = s_id[f], first = f / topk * topk;
    bool own = e >= 0;
    for (int g = first; g < f; ++g) own = own && s_id[g] != e;
    if (own) atomicAdd(&s_count[e], 1);
  }
  __syncthreads();
  // exclusive sums over the experts of (is used, rows, groups)
  const int rows = s_count[tid];
  int v[3] = {rows > 0 ? 1 : 0, rows, (rows + group_cap - 1) / group_cap};
  int inc[3];
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    int x = v[q];
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, x, s);
      if (lane >= s) x += o;
    }
    inc[q] = x;
    if (lane == 31) s_scan[q][warp] = x;
  }
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      int x = lane < kPlanThreads / 32 ? s_scan[q][lane] : 0;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, x, s);
        if (lane >= s) x += o;
      }
      s_scan[q][lane] = x;
    }
  }
  __syncthreads();
  int ex[3];
#pragma unroll
  for (int q = 0; q < 3; ++q) ex[q] = inc[q] - v[q] + (warp > 0 ? s_scan[q][warp - 1] : 0);
  s_cursor[tid] = ex[1];
  if (rows > 0) {
    ws[lay.expert_id() + ex[0]] = tid;
    ws[lay.expert_off() + ex[0]] = ex[1];
    for (int g = 0; g < v[2]; ++g) {
      ws[lay.group_slot() + ex[2] + g] = ex[0];
      ws[lay.group_expert() + ex[2] + g] = tid;
      ws[lay.group_off() + ex[2] + g] = ex[1] + g * group_cap;
      ws[lay.group_end() + ex[2] + g] = ex[1] + min((g + 1) * group_cap, rows);
    }
  }
  for (int i = tid; i < lay.experts; i += kPlanThreads) ws[lay.expert_done() + i] = 0;
  if (tid == 0) {
    ws[MlpLayout::kNumExperts] = s_scan[0][31];
    ws[MlpLayout::kNumGroups] = s_scan[2][31];
    ws[lay.expert_off() + s_scan[0][31]] = s_scan[1][31];
    ws[MlpLayout::kNextUnit] = 0;
    ws[MlpLayout::kRowsDone] = 0;
  }
  __syncthreads();
  for (int f = tid; f < pairs; f += kPlanThreads) {
    const int e = s_id[f], t = f / topk, first = t * topk;
    bool own = e >= 0;
    for (int g = first; g < f; ++g) own = own && s_id[g] != e;
    int row = -1;
    if (own) {
      float w = s_weight[f];
      for (int g = f + 1; g < first + topk; ++g)
        if (s_id[g] == e) w += s_weight[g];
      row = atomicAdd(&s_cursor[e], 1);
      ws[lay.row_token() + row] = t;
      reinterpret_cast<float*>(ws)[lay.row_weight() + row] = w;
    }
    ws[lay.pair_row() + f] = row;
  }
}

// The same for at most 32 (token, slot) pairs and groups that hold every token, one pair per lane of a single warp: no barrier, one
// round trip. 3.4 us alone against 5.6; on the layer 57.5 -> 55.7 us at one token.
__global__ void __launch_bounds__(32)
moe_mlp_plan_warp_kernel(const void* __restrict__ ids, int is64, const float* __restrict__ weights, int tokens, int topk, int num_experts,
                         int group_cap, MlpLayout lay, int* __restrict__ ws) {
  constexpr unsigned kFull = 0xffffffffu;
  const int lane = threadIdx.x, pairs = tokens * topk;
  griddep_launch_dependents();  // the layer kernel touches no memory before this one is through
  griddep_wait();
  long long e64 = -1;
  float w = 0.0f;
  if (lane < pairs) {
    e64 = is64 ? static_cast<const long long*>(ids)[lane] : static_cast<long long>(static_cast<const int*>(ids)[lane]);
    w = weights[lane];
  }
  const int e = (e64 >= 0 && e64 < num_experts) ? static_cast<int>(e64) : -1;
  const int t = lane / topk;
  // lanes with the same expert, and those of them in the same token; the first of the latter owns the row
  const unsigned same = __match_any_sync(kFull, e);
  const int first_lane = t * topk;
  const int last_lane = first_lane + topk;
  const unsigned token_lanes = (first_lane < 32 ? kFull << first_lane : 0u) & (last_lane < 32 ? ~(kFull << last_lane) : kFull);
  const unsigned repeats = same & token_lanes;
  const bool own = e >= 0 && lane == __ffs(repeats) - 1;
  float sum = w;
  for (int j = 0; j < 32; ++j) {  // repeats of the expert in the token, in slot order behind the owner
    const float o = __shfl_sync(kFull, w, j);
    if (own && j > lane && ((repeats >> j) & 1u)) sum += o;
  }
  const unsigned owners = __ballot_sync(kFull, own);
  const unsigned rows_of = same & owners;                                   // owners of this lane's expert
  const bool lead = own && lane == __ffs(rows_of) - 1;                      // one lane per distinct expert
  int slot = 0, off = 0;                                                    // distinct experts and rows before this one
  const unsigned leads = __ballot_sync(kFull, lead);
  const int rows = __popc(rows_of);
  for (int j = 0; j < 32; ++j) {
    const int oe = __shfl_sync(kFull, e, j), orows = __shfl_sync(kFull, rows, j);
    if (((leads >> j) & 1u) && oe < e) {
      ++slot;
      off += orows;
    }
  }
  const int num = __popc(leads), total = __popc(owners);
  if (lead) {
    ws[lay.expert_id() + slot] = e;
    ws[lay.expert_off() + slot] = off;
    ws[lay.group_slot() + slot] = slot;
    ws[lay.group_expert() + slot] = e;
    ws[lay.group_off() + slot] = off;
    ws[lay.group_end() + slot] = off + rows;
  }
  const int row = off + __popc(rows_of & ((1u << lane) - 1u));
  if (own) {
    ws[lay.row_token() + row] = t;
    reinterpret_cast<float*>(ws)[lay.row_weight() + row] = sum;
  }
  if (lane < pairs) ws[lay.pair_row() + lane] = own ? row : -1;
  if (lane < lay.experts) ws[lay.expert_done() + lane] = 0;
  if (lane == 0) {
    ws[MlpLayout::kNumExperts] = num;
    ws[MlpLayout::kNumGroups] = num;
    ws[lay.expert_off() + num] = total;
    ws[MlpLayout::kNextUnit] = 0;
    ws[MlpLayout::kRowsDone] = 0;
  }
}

// ------------------------------------------------------------------------------------------------------------ layer
// Weights are read once per call (or once per row group, soon after each other): their lines leave L2 first, so that h, the
// weighted rows and x are still there when they are read. Measured at 128 tokens, 64 experts of 4096 x 1536: 404 us
// without the hint, 392 with it.
__device__ __forceinline__ void tma_load_5d_hint(void* smem_dst, const CUtensorMap* tmap, uint64_t* bar, int x, int y, int z, int w,
                                                 int v, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5, %6, %7}], "
      "[%2], %8;" ::"r"(smem_u32(smem_dst)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_hint(void* smem_dst, const CUtensorMap* tmap, uint64_t* bar, int x, int y, int z,
                                                 uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5}], [%2], %6;" ::
          "r"(smem_u32(smem_dst)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "l"(policy)
      : "memory");
}
// Orders generic-proxy accesses to global memory before later accesses of the async proxy (TMA), and the other way round.
__device__ __forceinline__ void fence_proxy_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ int load_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void add_release(int* p, int v) {
  asm volatile("red.release.gpu.global.add.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}

// Bounded wait until *counter reaches `want`; every lane of the warp calls it and gets the same answer.
__device__ __forceinline__ bool counter_wait_warp(const int* counter, int want, const WaitCtx& w) {
  bool ok = true;
  if ((threadIdx.x & 31) == 0 && load_acquire(counter) < want) {
    const uint64_t t0 = global_timer_ns();
    uint32_t spins = 0;
    while (load_acquire(counter) < want) {
      if ((++spins & 0x3F) == 0) {
        if (*w.abort_flag) ok = false;
        if (ok && global_timer_ns() - t0 > w.timeout_ns) {
          *w.abort_flag = 1;
          atomicCAS(w.status, 0, TB_DEV_TIMEOUT_EXPERT_TILES);
          ok = false;
        }
        if (!ok) break;
      }
      __nanosleep(spins < 8 ? 32 : 128);
    }
  }
  ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
  if (ok) load_acquire(counter);  // each lane's own acquire
  return ok;
}

// One unit as the weight loader hands it to the other roles.
struct Unit {
  int kind;    // 1, 2, 3; 0 = no more units
  int expert;  // id
  int tile;    // tile of ffn / hidden, or the run of the output
  int off;     // first row of the expert (kind 1) or group (kind 2)
  int rows;
  int slot;    // index among the distinct experts
};
constexpr int kUnitWords = 6;

template <typename T>
__device__ __forceinline__ unsigned short to_bits(float v);
template <>
__device__ __forceinline__ unsigned short to_bits<__nv_bfloat16>(float v) {
  return __bfloat16_as_ushort(__float2bfloat16_rn(v));
}
template <>
__device__ __forceinline__ unsigned short to_bits<__half>(float v) {
  return __half_as_ushort(__float2half_rn(v));
}
template <typename T>
__device__ __forceinline__ float from_bits(unsigned short v);
template <>
__device__ __forceinline__ float from_bits<__nv_bfloat16>(unsigned short v) {
  return __bfloat162float(__ushort_as_bfloat16(v));
}
template <>
__device__ __forceinline__ float from_bits<__half>(unsigned short v) {
  return __half2float(__ushort_as_half(v));
}

// Units of the two halves of h: hi * kHi + lo * kLo.
template <typename T>
struct HalfUnits {
  static constexpr float kHi = 1.0f, kLo = 1.0f;
};
template <>
struct HalfUnits<__half> {
  static constexpr float kHi = 256.0f, kLo = 0.125f;  // kHi / kLo = 2^11: the rest of the largest hi still fits lo
};

__device__ __forceinline__ float4 add4(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
// Four consecutive outputs; `vec`: the address is a multiple of 8.
template <typename T>
__device__ __forceinline__ void store_quad(unsigned short* o, float4 v, int vec) {
  const ushort4 b = make_ushort4(to_bits<T>(v.x), to_bits<T>(v.y), to_bits<T>(v.z), to_bits<T>(v.w));
  if (vec) {
    *reinterpret_cast<ushort4*>(o) = b;
  } else {
    o[0] = b.x;
    o[1] = b.y;
    o[2] = b.z;
    o[3] = b.w;
  }
}

// M1, M2: weight rows of a tile of the first and the second kind (256: two MMA tiles of 128). A 64-row accumulator occupies
// lanes 0-15 of every warp's 32 TMEM lanes, a 128-row one all.
template <typename T, int M1, int M2>
__global__ void __launch_bounds__(kMlpThreads, 1)
moe_mlp_kernel(const __grid_constant__ CUtensorMap tmap_w1, const __grid_constant__ CUtensorMap tmap_w2,
               const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_h2,
               const __grid_constant__ CUtensorMap tmap_h8, const __grid_constant__ CUtensorMap tmap_h32, const MlpParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], tmem_full[2], tmem_empty[2];
  __shared__ uint64_t queue_full[kQueueDepth], queue_empty[kQueueDepth];
  __shared__ int queue[kQueueDepth][kUnitWords];
  __shared__ int col_row[4][kMlpMaxTokens];  // per epilogue warp: row of a column's token, -1 = not routed here
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &abort_word;
  const WaitCtx wctx{abort_flag, p.status, p.timeout_ns};
  const int stages = p.stages;
  constexpr int kRows1 = M1 < 128 ? M1 : 128, kRows2 = M2 < 128 ? M2 : 128;  // rows of one MMA
  constexpr int kSubs = M1 / kRows1;                                         // MMA tiles side by side that share the activations
  constexpr int kSlabs1 = mlp_slabs(M1), kSlabs2 = mlp_slabs(M2);             // 64-element slabs of K per stage
  constexpr uint32_t kWeightBytes = kSlabs1 * M1 * kRowBytes;                 // of a stage, of either kind
  static_assert(M2 / kRows2 == kSubs && kSlabs2 * M2 * kRowBytes == kWeightBytes, "both kinds share the ring");
  constexpr int kGroups = kRows1 / 64;  // eight-feature groups (16 rows: 8 gate, 8 up) per epilogue warp and MMA tile
  if (threadIdx.x == 0) {
    abort_word = 0;
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full_bar[s], 2);  // weight loader and activation loader
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], 4);
    }
    for (int i = 0; i < kQueueDepth; ++i) {
      mbar_init(&queue_full[i], 1);
      mbar_init(&queue_empty[i], kQueueConsumers);
    }
    mbar_fence_init();
    prefetch_tmap(&tmap_w1);
    prefetch_tmap(&tmap_w2);
    prefetch_tmap(&tmap_x);
  }
  if (warp == kWarpMma) {
    tmem_alloc<1>(&tmem_slot, static_cast<uint32_t>(p.tmem_cols));
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  griddep_launch_dependents();
  griddep_wait();

  const int* ws = p.ws;
  const int num_experts = __ldcg(ws + MlpLayout::kNumExperts), num_groups = __ldcg(ws + MlpLayout::kNumGroups);
  const int units1 = num_experts * p.f_tiles, units2 = num_groups * p.h_tiles;
  const int units3 = p.tokens * p.runs;
  constexpr int kAlign2 = M2 < 128 ? 8 : 16;  // columns of an MMA come in multiples of this
  const int kb1 = (p.hidden + kSlabs1 * kStageK - 1) / (kSlabs1 * kStageK), kb2 = (p.ffn + kSlabs2 * kStageK - 1) / (kSlabs2 * kStageK);

  // The next unit out of the queue; every lane of a consuming warp calls it.
  auto take = [&](int seq, bool& ok) -> Unit {
    const int i = seq & (kQueueDepth - 1);
    ok = mbar_wait_warp(&queue_full[i], (seq / kQueueDepth) & 1u, wctx, TB_DEV_TIMEOUT_TILE_QUEUE);
    Unit u = {0, 0, 0, 0, 0, 0};
    if (ok) {
      const volatile int* q = queue[i];
      u.kind = q[0];
      u.expert = q[1];
      u.tile = q[2];
      u.off = q[3];
      u.rows = q[4];
      u.slot = q[5];
    }
    __syncwarp();
    if (lane == 0 && ok) mbar_arrive(&queue_empty[i]);
    return u;
  };

  if (warp == kWarpWeights) {
    // -------------------------------------------------------------- scheduler and weight loader
    int s = 0, seq = 0;
    uint32_t ph = 0;
    bool ok = true;
    // The number of the next unit and its row of the plan are asked for while the current unit's loads go out: under load a
    // round trip takes several microseconds, and nothing else would hide it.
    const uint64_t policy = evict_first_policy();
    int next = 0;
    Unit pending = {0, 0, 0, 0, 0, 0};
    // the first 32 experts of the plan, one per lane: most of the time a unit of the first kind needs no load at all
    const int my_expert = lane < p.lay.experts ? __ldcg(ws + p.lay.expert_id() + lane) : 0;
    const int my_off = lane < p.lay.experts ? __ldcg(ws + p.lay.expert_off() + lane) : 0;
    const int my_end = lane < p.lay.experts ? __ldcg(ws + p.lay.expert_off() + lane + 1) : 0;
    auto ask = [&]() {
      if (lane == 0) next = atomicAdd(p.ws + MlpLayout::kNextUnit, 1);
    };
    auto look_up = [&]() {
      const int idx = __shfl_sync(0xffffffffu, next, 0);
      pending = Unit{0, 0, 0, 0, 0, 0};
      if (idx < units1) {
        pending.kind = 1;
        pending.slot = idx / p.f_tiles;
        pending.tile = idx - pending.slot * p.f_tiles;
        if (pending.slot < 32) {
          pending.expert = __shfl_sync(0xffffffffu, my_expert, pending.slot);
          pending.off = __shfl_sync(0xffffffffu, my_off, pending.slot);
          pending.rows = __shfl_sync(0xffffffffu, my_end, pending.slot);  // one past the last row
        } else {
          pending.expert = __ldcg(ws + p.lay.expert_id() + pending.slot);
          pending.off = __ldcg(ws + p.lay.expert_off() + pending.slot);
          pending.rows = __ldcg(ws + p.lay.expert_off() + pending.slot + 1);
        }
      } else if (idx < units1 + units2) {
        pending.kind = 2;
        const int g = (idx - units1) / p.h_tiles;
        pending.tile = idx - units1 - g * p.h_tiles;
        pending.slot = __ldcg(ws + p.lay.group_slot() + g);
        pending.expert = __ldcg(ws + p.lay.group_expert() + g);
        pending.off = __ldcg(ws + p.lay.group_off() + g);
        pending.rows = __ldcg(ws + p.lay.group_end() + g);
      } else if (idx < units1 + units2 + units3) {
        pending.kind = 3;
        pending.tile = idx - units1 - units2;
      }
    };
    ask();
    look_up();
    while (true) {
      Unit u = pending;
      u.rows -= u.off;
      const int i = seq & (kQueueDepth - 1);
      ok = mbar_wait_warp(&queue_empty[i], ((seq / kQueueDepth) & 1u) ^ 1u, wctx, TB_DEV_TIMEOUT_TILE_QUEUE);
      if (!ok) break;
      if (lane == 0) {
        volatile int* q = queue[i];
        q[0] = u.kind;
        q[1] = u.expert;
        q[2] = u.tile;
        q[3] = u.off;
        q[4] = u.rows;
        q[5] = u.slot;
        mbar_arrive(&queue_full[i]);
      }
      __syncwarp();
      ++seq;
      if (u.kind == 0) break;
      if (u.kind == 3) {
        ask();
        look_up();
        continue;
      }
      const int nkb = u.kind == 1 ? kb1 : kb2;
      const int ask_at = nkb > 16 ? nkb - 16 : 0, look_at = nkb > 6 ? nkb - 6 : nkb - 1;
      auto load = [&](int kb) {
        uint8_t* dst = ring + static_cast<size_t>(s) * p.stage_bytes;
        mbar_arrive_expect_tx(&full_bar[s], kWeightBytes);
        if (u.kind == 1) {
#pragma unroll
          for (int b = 0; b < kSlabs1; ++b)
            tma_load_5d_hint(dst + b * M1 * kRowBytes, &tmap_w1, &full_bar[s], (kb * kSlabs1 + b) * kStageK, 0, 0, u.tile * (M1 / 16),
                             u.expert, policy);
        } else {
#pragma unroll
          for (int b = 0; b < kSlabs2; ++b)
            tma_load_3d_hint(dst + b * M2 * kRowBytes, &tmap_w2, &full_bar[s], (kb * kSlabs2 + b) * kStageK, u.tile * M2, u.expert, policy);
        }
      };
      for (int kb = 0; kb < nkb; ++kb) {
        if (kb == ask_at) ask();
        if (kb == look_at) look_up();
        ok = wait_warp(&empty_bar[s], ph ^ 1, wctx, TB_DEV_TIMEOUT_SMEM_EMPTY);
        if (!ok) break;
        if (elect_one()) load(kb);
        __syncwarp();
        if (++s == stages) {
          s = 0;
          ph ^= 1;
        }
      }
      if (!ok) break;
    }
  } else if (warp == kWarpAct) {
    // -------------------------------------------------------------- activation loader
    // Only rows that exist are copied. What stands in the other rows of the operand (an earlier stage's values) makes columns
    // of the product that nobody reads, and a column depends on its own row alone.
    int s = 0, seq = 0;
    uint32_t ph = 0;
    bool ok = true;
    while (true) {
      const Unit u = take(seq++, ok);
      if (!ok || u.kind == 0) break;
      if (u.kind == 3) continue;
      // rows of h (hi and lo of every row of the group) come in the smallest copies that do not multiply their number
      const int h_rows = 2 * u.rows, h_box = h_rows <= 2 ? 2 : (h_rows <= 8 ? 8 : 32);
      const CUtensorMap* h_map = h_box == 2 ? &tmap_h2 : (h_box == 8 ? &tmap_h8 : &tmap_h32);
      if (u.kind == 2) {
        ok = counter_wait_warp(p.ws + p.lay.expert_done() + u.slot, 4 * p.f_tiles, wctx);
        if (!ok) break;
        fence_proxy_async_all();  // h was written by ordinary stores of other SMs; it is read by TMA below
      }
      const int nkb = u.kind == 1 ? kb1 : kb2;
      const CUtensorMap* map = u.kind == 1 ? &tmap_x : h_map;
      const int rows = u.kind == 1 ? p.tokens : (h_rows + h_box - 1) / h_box * h_box;
      const int box = u.kind == 1 ? p.tokens : h_box, row0 = u.kind == 1 ? 0 : 2 * u.off;
      const int slabs = u.kind == 1 ? kSlabs1 : kSlabs2, act_bytes = u.kind == 1 ? p.act1_bytes : p.act2_bytes;
      for (int kb = 0; kb < nkb; ++kb) {
        ok = wait_warp(&empty_bar[s], ph ^ 1, wctx, TB_DEV_TIMEOUT_SMEM_EMPTY);
        if (!ok) break;
        if (elect_one()) {
          uint8_t* dst = ring + static_cast<size_t>(s) * p.stage_bytes + kWeightBytes;
          mbar_arrive_expect_tx(&full_bar[s], static_cast<uint32_t>(slabs * rows * kRowBytes));
          for (int b = 0; b < slabs; ++b)
            for (int r = 0; r < rows; r += box)
              tma_load_2d(dst + b * act_bytes + r * kRowBytes, map, &full_bar[s], (kb * slabs + b) * kStageK, row0 + r);
        }
        __syncwarp();
        if (++s == stages) {
          s = 0;
          ph ^= 1;
        }
      }
      if (!ok) break;
    }
  } else if (warp == kWarpMma) {
    // -------------------------------------------------------------- MMA issuer
    int s = 0, seq = 0, acc = 0;
    uint32_t ph = 0, acc_parity = 0;
    bool ok = true;
    const uint64_t desc0 = make_smem_desc(smem_u32(ring), 16, 1024);
    while (true) {
      const Unit u = take(seq++, ok);
      if (!ok || u.kind == 0) break;
      if (u.kind == 3) continue;
      const int n = u.kind == 1 ? p.n1 : ((2 * u.rows + kAlign2 - 1) & ~(kAlign2 - 1));
      const int nkb = u.kind == 1 ? kb1 : kb2;
      const uint32_t idesc = p.idesc | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>((u.kind == 1 ? kRows1 : kRows2) >> 4) << 24);
      const uint32_t d = tmem_base + static_cast<uint32_t>(acc * kSubs * p.acc_stride);
      ok = wait_warp(&tmem_empty[acc], ((acc_parity >> acc) & 1u) ^ 1u, wctx, TB_DEV_TIMEOUT_TMEM_EMPTY);
      if (!ok) break;
      tc_fence_after();
      for (int kb = 0; kb < nkb; ++kb) {
        ok = wait_warp(&full_bar[s], ph, wctx, TB_DEV_TIMEOUT_SMEM_FULL);
        if (!ok) break;
        if (elect_one()) {
          const uint64_t stage = desc0 + static_cast<uint64_t>((s * p.stage_bytes) >> 4);
          auto issue = [&](int b, uint32_t slab_bytes, int act_bytes, int mma_rows) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int j = 0; j < kSubs; ++j)
                umma<0, 1>(d + j * p.acc_stride, stage + ((b * slab_bytes + j * mma_rows * kRowBytes) >> 4) + 2 * k,
                           stage + ((kWeightBytes + b * act_bytes) >> 4) + 2 * k, idesc, (b > 0 || k > 0) ? 1u : (kb > 0 ? 1u : 0u));
          };
          if (u.kind == 1) {
#pragma unroll
            for (int b = 0; b < kSlabs1; ++b) issue(b, M1 * kRowBytes, p.act1_bytes, kRows1);
          } else {
#pragma unroll
            for (int b = 0; b < kSlabs2; ++b) issue(b, M2 * kRowBytes, p.act2_bytes, kRows2);
          }
          umma_commit(&empty_bar[s]);
          if (kb + 1 == nkb) umma_commit(&tmem_full[acc]);
        }
        __syncwarp();
        if (++s == stages) {
          s = 0;
          ph ^= 1;
        }
      }
      if (!ok) break;
      acc_parity ^= 1u << acc;
      acc ^= 1;
    }
  } else {
    // -------------------------------------------------------------- epilogue (warps 0-3, one per TMEM lane quarter)
    int seq = 0, acc = 0;
    uint32_t parity = 0;
    bool ok = true;
    const float* row_weight = reinterpret_cast<const float*>(ws) + p.lay.row_weight();
    while (true) {
      const Unit u = take(seq++, ok);
      if (!ok || u.kind == 0) break;
      if (u.kind == 3) {
        // the sum over a token's rows, in slot order
        const int t = u.tile / p.runs, quads = p.hidden / 4;
        const int q0 = (u.tile - t * p.runs) * p.quads_per_thread * 128 + threadIdx.x;
        const int q1 = min(quads, q0 + p.quads_per_thread * 128);
        const int* rows = ws + p.lay.pair_row() + t * p.topk;
        unsigned short* o = reinterpret_cast<unsigned short*>(p.out) + t * p.out_stride;
        int r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = j < p.topk ? __ldcg(rows + j) : -1;  // on their way while the rows are still written
        ok = counter_wait_warp(p.ws + MlpLayout::kRowsDone, 4 * units2, wctx);
        if (!ok) break;
        if (p.topk <= 8) {
          const float4* src[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) src[j] = reinterpret_cast<const float4*>(p.y + static_cast<long long>(max(r[j], 0)) * p.hidden);
          // two runs of the token at a time: sixteen loads in flight, none of them conditional (a place without a row reads
          // row 0 and drops it)
          for (int q = q0; q < q1; q += 256) {
            float4 a[8], b[8];
            const int second = q + 128 < q1 ? q + 128 : q;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              a[j] = __ldcg(src[j] + q);
              b[j] = __ldcg(src[j] + second);
            }
            float4 sum_a = make_float4(0.f, 0.f, 0.f, 0.f), sum_b = sum_a;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (r[j] >= 0) {
                sum_a = add4(sum_a, a[j]);
                sum_b = add4(sum_b, b[j]);
              }
            }
            store_quad<T>(o + q * 4, sum_a, p.out_vec);
            if (second != q) store_quad<T>(o + second * 4, sum_b, p.out_vec);
          }
        } else {
          for (int q = q0; q < q1; q += 128) {
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int j = 0; j < p.topk; ++j) {
              const int r = __ldcg(rows + j);
              if (r >= 0) sum = add4(sum, __ldcg(reinterpret_cast<const float4*>(p.y + static_cast<long long>(r) * p.hidden) + q));
            }
            store_quad<T>(o + q * 4, sum, p.out_vec);
          }
        }
        continue;
      }
      if (u.kind == 1) {
        // which columns are this expert's: looked up while the product is still being accumulated
        for (int c = lane; c < p.tokens; c += 32) col_row[warp][c] = -1;
        __syncwarp();
        for (int r = lane; r < u.rows; r += 32) col_row[warp][__ldcg(ws + p.lay.row_token() + u.off + r)] = u.off + r;
        __syncwarp();
      }
      ok = __all_sync(0xffffffffu, mbar_wait(&tmem_full[acc], (parity >> acc) & 1u, wctx, TB_DEV_TIMEOUT_TMEM_FULL));
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(warp * 32) << 16) + static_cast<uint32_t>(acc * kSubs * p.acc_stride);
      const int n = u.kind == 1 ? p.n1 : 2 * u.rows;
      for (int sub = 0; sub < kSubs; ++sub)
      for (int c0 = 0; c0 < n; c0 += 32) {
        uint32_t r[32];
        tmem_ld_32x32(t_row + sub * p.acc_stride + c0, r);
        tmem_ld_wait(r);
        if (sub + 1 == kSubs && c0 + 32 >= n) {  // the last columns sit in registers
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tmem_empty[acc]);
        }
        if (u.kind == 1) {
          // lanes 0-7 of a run of 16 hold gate features, lanes 8-15 the matching up features
          const int f = u.tile * (M1 / 2) + sub * (kRows1 / 2) + (warp * kGroups + (lane >> 4)) * 8 + (lane & 7);
          const bool mine = (lane & 8) == 0 && (kRows1 == 128 || lane < 16) && f < p.ffn;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const int row = c0 + j < p.tokens ? col_row[warp][c0 + j] : -1;
            if (row >= 0) {  // the same for the whole warp
              const float g = __uint_as_float(r[j]);
              const float up = __shfl_xor_sync(0xffffffffu, g, 8);
              const float h = g / (1.0f + expf(-g)) * up;
              const unsigned short hi = to_bits<T>(h * (1.0f / HalfUnits<T>::kHi));
              // an infinite h has no low half (inf - inf)
              const float rest = h - from_bits<T>(hi) * HalfUnits<T>::kHi;
              const unsigned short lo =
                  fabsf(rest) < __builtin_huge_valf() ? to_bits<T>(rest * (1.0f / HalfUnits<T>::kLo)) : static_cast<unsigned short>(0);
              if (mine) {
                unsigned short* dst = reinterpret_cast<unsigned short*>(p.h) + static_cast<long long>(row) * 2 * p.ffn + f;
                dst[0] = hi;
                dst[p.ffn] = lo;
              }
            }
          }
        } else {
          const int hcol = u.tile * M2 + sub * kRows2 + warp * (kRows2 / 4) + lane;
          const bool mine = (kRows2 == 128 || lane < 16) && hcol < p.hidden;
#pragma unroll
          for (int j = 0; j < 32; j += 2) {  // the products with both halves of h stand side by side
            const int row = (c0 + j) >> 1;
            if (row < u.rows && mine)
              __stcg(p.y + static_cast<long long>(u.off + row) * p.hidden + hcol,
                     __ldcg(row_weight + u.off + row) *
                         (__uint_as_float(r[j]) * HalfUnits<T>::kHi + __uint_as_float(r[j + 1]) * HalfUnits<T>::kLo));
          }
        }
      }
      parity ^= 1u << acc;
      acc ^= 1;
      // publish this warp's part of the unit: every epilogue warp counts for itself, so none waits for another. The release
      // of lane 0 covers the warp's stores (they come before the __syncwarp).
      __syncwarp();
      if (lane == 0) add_release(u.kind == 1 ? p.ws + p.lay.expert_done() + u.slot : p.ws + MlpLayout::kRowsDone, 1);
    }
  }

  // ------------------------------------------------------------------ teardown
  __syncwarp();
  if (*abort_flag) {
    // A wait gave up: let copies and MMAs already in flight land before shared memory and TMEM are released.
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kWarpMma) {
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, static_cast<uint32_t>(p.tmem_cols));
  }
}

// ------------------------------------------------------------------------------------------------------------ host
struct MlpShape {
  MlpLayout lay;
  int m1, m2;         // weight rows of a tile of either projection
  int n1, group_cap;
  int h_rows;         // rows of h a stage of the second projection has room for
  long long h_offset, y_offset, bytes;  // byte offsets in the workspace
};

// Weight rows of a tile of either projection (the second kind waits for all of an expert's units of the first, so those are
// dealt in the smaller tiles). Measured back to back with 64 + 64 / 64 + 128 / 128 + 128 rows, tokens x chosen of hidden x ffn:
//   1 x 8 of 4096 x 1536: 56.4 / 58.3 / 64.7 us      1 x 2 of 4096 x 4096: 48.2 / 54.8 / 53.6
//   5 x 4 of 2048 x 704:  48.0 / 36.5 / 39.9         4 x 6 of 2048 x 1408: 65.2 / 63.4 / 64.2
//  16 x 8 of 4096 x 1536:  313 /  306 /  310        32 x 8: 353 / 345 / 346        64 x 8: 388 / 376 / 359
// 64 rows of the second kind pay only for single tokens, as long as a unit stays long enough (1 x 8 of 2048 x 768: 28.8 / 28.9).
// Above 64 tokens their share of a stage is as large as 128 weight rows', so a tile has 256: 408 against 414 us at 128 tokens.
void mlp_tile_rows(int tokens, int topk, int ffn, int* m1, int* m2) {
  *m1 = tokens > 64 ? 256 : (tokens <= 32 ? 64 : 128);
  *m2 = tokens > 64 ? 256 : (tokens * topk <= 8 && ffn >= 1024 ? 64 : 128);
}

// Columns of the two projections and the workspace they need. The rows of an expert go in groups of at most half the token
// columns (but 16), so that both halves of h take no more shared memory in a stage than the tokens do: an expert that more
// than half of the tokens choose is read once per group, the second time out of L2.
MlpShape mlp_shape(int tokens, int topk, int num_experts, int hidden, int ffn) {
  MlpShape s;
  mlp_tile_rows(tokens, topk, ffn, &s.m1, &s.m2);
  const int align = s.m1 == 64 ? 8 : 16;
  s.n1 = (tokens + align - 1) / align * align;
  s.group_cap = tokens < 16 ? tokens : ((tokens + 15) / 16 * 8 < 16 ? 16 : (tokens + 15) / 16 * 8);
  // rows of h arrive in copies of 2, 8 or 32
  s.h_rows = s.group_cap <= 4 ? 8 : (2 * s.group_cap + 31) / 32 * 32;
  if (s.h_rows < 16 && s.m2 > 64) s.h_rows = 16;
  s.lay.pairs = tokens * topk;
  s.lay.experts = num_experts < s.lay.pairs ? num_experts : s.lay.pairs;
  s.lay.groups = s.lay.experts + s.lay.pairs / s.group_cap;
  auto up = [](long long v) { return (v + 255) & ~255ll; };
  s.h_offset = up(s.lay.words() * 4);
  s.y_offset = s.h_offset + up(2ll * s.lay.pairs * ffn * 2);
  s.bytes = s.y_offset + up(4ll * s.lay.pairs * hidden);
  return s;
}

bool mlp_sizes_ok(int tokens, int topk, int num_experts, int hidden, int ffn) {
  return tokens >= 0 && tokens <= kMlpMaxTokens && topk >= 1 && topk <= kMlpMaxTopk && num_experts >= 1 &&
         num_experts <= kMlpMaxExperts && hidden >= 8 && ffn >= 8 && hidden % 8 == 0 && ffn % 8 == 0 &&
         hidden <= (1 << 20) && ffn <= (1 << 20);
}

template <typename T, int M1, int M2>
int mlp_launch(const CUtensorMap& w1, const CUtensorMap& w2, const CUtensorMap& x, const CUtensorMap (&h)[3], const MlpParams& p,
               int grid, int smem_bytes, int device, cudaStream_t stream) {
  auto kernel = moe_mlp_kernel<T, M1, M2>;
  static SmemOptIn configured;
  const int rc = opt_in_smem(kernel, smem_bytes, device, configured, "cudaFuncSetAttribute(moe_mlp)");
  if (rc != TB_OK) return rc;
  return launch_token_kernel(kernel, dim3(static_cast<unsigned>(grid)), kMlpThreads, smem_bytes, 0, stream, "moe_mlp_kernel launch", w1, w2, x, h[0],
                             h[1], h[2], p);
}

template <typename T>
auto mlp_variant(int m1, int m2) {
  return m1 == 256 ? mlp_launch<T, 256, 256> : (m1 == 128 ? mlp_launch<T, 128, 128> : (m2 == 128 ? mlp_launch<T, 64, 128> : mlp_launch<T, 64, 64>));
}

int mlp_impl(const tb_moe_mlp_args& a, cudaStream_t stream) {
  if (!mlp_sizes_ok(a.tokens, a.topk, a.num_experts, a.hidden, a.ffn)) return TB_ERR_INVALID;
  if (a.dtype != TB_DTYPE_BF16 && a.dtype != TB_DTYPE_F16) return TB_ERR_UNSUPPORTED;
  if (a.tokens == 0) return TB_OK;
  if (a.x == nullptr || a.w1 == nullptr || a.w2 == nullptr || a.topk_ids == nullptr || a.topk_weights == nullptr ||
      a.out == nullptr)
    return TB_ERR_INVALID;
  if ((a.tokens > 1 && (a.x_row_stride < a.hidden || a.out_row_stride < a.hidden)) || a.w1_row_stride < a.hidden ||
      a.w2_row_stride < a.ffn || a.w1_expert_stride < 0 || a.w2_expert_stride < 0)
    return TB_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(a.out) % 2 || reinterpret_cast<uintptr_t>(a.topk_weights) % 4 ||
      reinterpret_cast<uintptr_t>(a.topk_ids) % (a.ids_are_int64 ? 8 : 4))
    return TB_ERR_ALIGNMENT;
  const MlpShape s = mlp_shape(a.tokens, a.topk, a.num_experts, a.hidden, a.ffn);
  if (a.workspace == nullptr || a.workspace_bytes < s.bytes) return TB_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a.workspace) % 256) return TB_ERR_ALIGNMENT;
  int device = 0, num_sms = 0, smem_optin = 0;
  int* status = nullptr;
  int rc = current_device_limits(&device, &num_sms, &smem_optin, &status);
  if (rc != TB_OK) return rc;

  char* ws = static_cast<char*>(a.workspace);
  MlpParams p = {};
  p.lay = s.lay;
  p.ws = reinterpret_cast<int*>(ws);
  p.tokens = a.tokens;
  p.topk = a.topk;
  p.hidden = a.hidden;
  p.ffn = a.ffn;
  p.n1 = s.n1;
  p.group_cap = s.group_cap;
  p.h = ws + s.h_offset;
  p.y = reinterpret_cast<float*>(ws + s.y_offset);
  p.out = a.out;
  p.out_stride = a.out_row_stride;
  p.out_vec = (reinterpret_cast<uintptr_t>(a.out) % 8 == 0 && (a.tokens == 1 || a.out_row_stride % 4 == 0)) ? 1 : 0;
  p.bf16 = a.dtype == TB_DTYPE_BF16 ? 1 : 0;
  p.status = status;
  p.timeout_ns = a.wait_timeout_ms > 0 ? static_cast<unsigned long long>(a.wait_timeout_ms) * 1000000ull : 2000000000ull;

  const int slabs1 = mlp_slabs(s.m1), slabs2 = mlp_slabs(s.m2);
  p.act1_bytes = s.n1 * kRowBytes;
  p.act2_bytes = s.h_rows * kRowBytes;
  const int act = slabs1 * p.act1_bytes > slabs2 * p.act2_bytes ? slabs1 * p.act1_bytes : slabs2 * p.act2_bytes;
  p.stage_bytes = slabs1 * s.m1 * kRowBytes + act;
  p.stages = (smem_optin - 8192) / p.stage_bytes;  // beside the ring: barriers, queue, column tables, the ring's alignment
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  if (p.stages < 2) return TB_ERR_UNSUPPORTED;
  const int smem_bytes = p.stages * p.stage_bytes + 1024;
  const int cols = s.n1 > s.h_rows ? s.n1 : s.h_rows;
  p.acc_stride = cols < 32 ? 32 : (cols + 31) / 32 * 32;
  p.tmem_cols = 64;
  while (p.tmem_cols < 2 * (s.m1 > 128 ? 2 : 1) * p.acc_stride) p.tmem_cols <<= 1;
  p.f_tiles = (a.ffn + s.m1 / 2 - 1) / (s.m1 / 2);
  p.h_tiles = (a.hidden + s.m2 - 1) / s.m2;
  // the sum over a token's rows: about as many units as SMs, or one per token when there are more tokens
  const int token_runs = (a.hidden / 4 + 127) / 128;
  p.runs = num_sms / a.tokens < 1 ? 1 : (num_sms / a.tokens > token_runs ? token_runs : num_sms / a.tokens);
  p.quads_per_thread = (token_runs + p.runs - 1) / p.runs;
  p.runs = (token_runs + p.quads_per_thread - 1) / p.quads_per_thread;
  // fp32 accumulators; operand format (0 = f16, 1 = bf16); rows and columns are added per unit
  const uint32_t fmt = p.bf16 ? 1u : 0u;
  p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10);

  CUtensorMap tw1, tw2, tx, th[3];
  const uint64_t es = 2;
  {
    // W1 as [expert][ffn / 8][gate, up][8][hidden]: a box of M/16 x 2 x 8 rows lands as runs of 8 gate rows and the 8 matching
    // up rows, so gate and up of a feature end in the same warp's TMEM lanes, 8 lanes apart
    const uint64_t row = static_cast<uint64_t>(a.w1_row_stride) * es;
    const uint64_t dims[5] = {static_cast<uint64_t>(a.hidden), 8, 2, static_cast<uint64_t>(a.ffn / 8), static_cast<uint64_t>(a.num_experts)};
    const uint64_t strides[4] = {row, row * a.ffn, row * 8, a.num_experts > 1 ? static_cast<uint64_t>(a.w1_expert_stride) * es : row * 2 * a.ffn};
    const uint32_t box[5] = {kStageK, 8, 2, static_cast<uint32_t>(s.m1 / 16), 1};
    if ((rc = encode_nd(&tw1, a.dtype, a.w1, 5, dims, strides, box)) != TB_OK) return rc;
  }
  {
    const uint64_t dims[3] = {static_cast<uint64_t>(a.ffn), static_cast<uint64_t>(a.hidden), static_cast<uint64_t>(a.num_experts)};
    const uint64_t row = static_cast<uint64_t>(a.w2_row_stride) * es;
    const uint64_t strides[2] = {row, a.num_experts > 1 ? static_cast<uint64_t>(a.w2_expert_stride) * es : row * a.hidden};
    const uint32_t box[3] = {kStageK, static_cast<uint32_t>(s.m2), 1};
    if ((rc = encode_nd(&tw2, a.dtype, a.w2, 3, dims, strides, box)) != TB_OK) return rc;
  }
  const uint64_t x_stride = static_cast<uint64_t>(a.tokens > 1 ? a.x_row_stride : a.hidden) * es;
  if ((rc = encode_2d(&tx, a.dtype, a.x, a.hidden, a.tokens, x_stride, kStageK, a.tokens, 1)) != TB_OK) return rc;
  const uint32_t h_box[3] = {2, 8, 32};
  for (int i = 0; i < 3; ++i)
    if ((rc = encode_2d(&th[i], a.dtype, p.h, a.ffn, 2ull * s.lay.pairs, a.ffn * es, kStageK, h_box[i], 1)) != TB_OK) return rc;

  const bool one_warp = s.lay.pairs <= 32 && a.tokens <= s.group_cap, narrow = a.num_experts <= 256;
  auto plan = one_warp ? moe_mlp_plan_warp_kernel : (narrow ? moe_mlp_plan_kernel<256> : moe_mlp_plan_kernel<kMlpMaxExperts>);
  rc = launch_token_kernel(plan, dim3(1), one_warp ? 32 : (narrow ? 256 : kMlpMaxExperts), 0, 0, stream, "moe_mlp_plan_kernel launch", a.topk_ids,
                           static_cast<int>(a.ids_are_int64 != 0), a.topk_weights, static_cast<int>(a.tokens), static_cast<int>(a.topk),
                           static_cast<int>(a.num_experts), s.group_cap, s.lay, p.ws);
  if (rc != TB_OK) return rc;
  auto launch = p.bf16 ? mlp_variant<__nv_bfloat16>(s.m1, s.m2) : mlp_variant<__half>(s.m1, s.m2);
  return launch(tw1, tw2, tx, th, p, num_sms, smem_bytes, device, stream);
}

}  // namespace
}  // namespace tb

extern "C" int64_t tb_moe_mlp_workspace_bytes(int32_t tokens, int32_t topk, int32_t num_experts, int32_t hidden, int32_t ffn) {
  if (!tb::mlp_sizes_ok(tokens, topk, num_experts, hidden, ffn) || tokens == 0) return 0;
  return tb::mlp_shape(tokens, topk, num_experts, hidden, ffn).bytes;
}

extern "C" int tb_moe_mlp(const tb_moe_mlp_args* args, void* stream) {
  if (args == nullptr) return TB_ERR_INVALID;
  return tb::mlp_impl(*args, static_cast<cudaStream_t>(stream));
}
