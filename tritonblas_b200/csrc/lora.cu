// A shared projection with one low-rank adapter per row (the requests of a batch, each with its own):
//     out[t] = x[t] W + bias + s_a (x[t] A_a^T) B_a^T,   a = adapter_ids[t]  (outside [0, num_adapters): no adapter)
//
// Two launches. lora_project_kernel forms v[t] = s_a x[t] A_a^T (rank numbers per row) and lays it out for the second one: for
// every tile of rows that the GEMM works on, the list of the adapters that occur in it and, per listed adapter, a block of the
// tile's rows that holds v in that adapter's rows and zeros in all others. The GEMM (gemm_kernel, LOWRANK) then walks those
// blocks against the adapters' B as further K stages of the same tile, so the update costs its bytes and no pass over the
// output, and the sum is rounded once. The GEMM starts while the projection still runs.
//
// The projection is bound by reading x and the used adapters' A once: every warp takes K slices, loads both operands straight
// into the fragments of mma.sync (16 bytes per lane and row; the order of K inside a slice is the same for both, so it need
// not be the instruction's), and the partial sums meet in shared memory and, when one block does not keep the SMs busy, across
// a cluster. v is rounded to the operands' 16-bit type once, after the scale: it is the A operand of a tensor-core product.
// Its error is eps / 2 of each of `rank` terms of the update, next to the one rounding of the output.
// No reference counterpart (the reference has no adapters).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common_host.h"
#include "ptx.cuh"

namespace tb {

bool pdl_enabled();  // api.cu

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxRank = 128;
constexpr int kMaxTileRows = 256;
constexpr long long kFlagBytes = 4096;  // stream-K flags at the start of the GEMM's workspace

struct ProjectParams {
  const void* x;
  long long x_stride;
  const void* a;
  long long a_adapter_stride, a_row_stride;
  const void* ids;
  int is64;
  const float* scales;  // null: 1
  int tokens, k, rank, num_adapters;
  int tile_rows;        // rows of a GEMM tile
  int max_slots;        // list entries per tile
  int v_cols;           // columns of a block (rank rounded up to 64)
  int splits;           // CTAs of a cluster that share K
  int k_chunk;          // K per CTA, a multiple of 32
  void* v;
  int* list;            // [tiles][1 + max_slots]
  unsigned* flags;      // stream-K flags to clear
  int flag_words;
};

template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                  uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ T cast16(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 cast16<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half cast16<__half>(float v) { return __float2half_rn(v); }

// Sum of one float per CTA of the cluster at the same shared-memory offset, in rank order.
__device__ __forceinline__ float cluster_sum(const float* mine, int splits) {
  const uint32_t addr = smem_u32(mine);
  float s = 0.0f;
  for (int r = 0; r < splits; ++r) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_cluster(addr, r)) : "memory");
    s += v;
  }
  return s;
}

// One cluster (of `splits` CTAs along K) per run of 16 * MT rows; blockIdx.y deals the adapters of the run. NT: n-tiles of 8
// ranks held in registers.
template <typename T, int NT, int MT>
__global__ void __launch_bounds__(kThreads) lora_project_kernel(const ProjectParams p) {
  constexpr int kRows = 16 * MT, kCols = 8 * NT;
  __shared__ alignas(16) int s_ids[kMaxTileRows];
  __shared__ int s_list[kMaxTileRows];
  __shared__ int s_warp_firsts[kWarps];
  __shared__ int s_present;
  __shared__ float s_red[kWarps][kRows][8];
  __shared__ float s_part[kRows][kCols];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = p.splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int run = blockIdx.x / p.splits;
  const int row0 = run * kRows;                 // first row of the run
  const int tile = row0 / p.tile_rows, tile_row0 = tile * p.tile_rows;
  griddep_wait();
  griddep_launch_dependents();

  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = tid; i < p.flag_words; i += kThreads) p.flags[i] = 0u;

  // Adapters of the tile in the order of their first rows; every block of the tile computes the same list.
  int id = -1;
  if (tid < p.tile_rows && tile_row0 + tid < p.tokens) {
    const long long v = p.is64 ? static_cast<const long long*>(p.ids)[tile_row0 + tid]
                               : static_cast<long long>(static_cast<const int*>(p.ids)[tile_row0 + tid]);
    if (v >= 0 && v < p.num_adapters) id = static_cast<int>(v);
  }
  s_ids[tid] = id;
  __syncthreads();
  bool first = id >= 0;
#pragma unroll 4
  for (int j = 0; j < (warp + 1) * 32; j += 4) {
    const int4 o = *reinterpret_cast<const int4*>(s_ids + j);
    first = first && !(o.x == id && j < tid) && !(o.y == id && j + 1 < tid) && !(o.z == id && j + 2 < tid) && !(o.w == id && j + 3 < tid);
  }
  const unsigned votes = __ballot_sync(0xffffffffu, first);
  if (lane == 0) s_warp_firsts[warp] = __popc(votes);
  __syncthreads();
  int before = __popc(votes & ((1u << lane) - 1u)), count = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += s_warp_firsts[w];
    count += s_warp_firsts[w];
  }
  if (first) s_list[before] = id;
  __syncthreads();
  if (row0 == tile_row0 && blockIdx.y == 0 && rank == 0) {
    int* list = p.list + static_cast<long long>(tile) * (1 + p.max_slots);
    if (tid == 0) list[0] = count;
    if (tid < count) list[1 + tid] = s_list[tid];
  }

  const T* x = static_cast<const T*>(p.x);
  const int g = lane >> 2, q = lane & 3;
  const int k_begin = rank * p.k_chunk, k_end = min(p.k, k_begin + p.k_chunk);
  for (int slot = blockIdx.y; slot < count; slot += gridDim.y) {
    const int adapter = s_list[slot];
    T* block = static_cast<T*>(p.v) + (static_cast<long long>(tile) * p.max_slots + slot) * p.tile_rows * p.v_cols +
               static_cast<long long>(row0 - tile_row0) * p.v_cols;
    if (tid == 0) s_present = 0;
    __syncthreads();
    if (tid < kRows && s_ids[row0 - tile_row0 + tid] == adapter) s_present = 1;
    __syncthreads();
    if (s_present == 0) {  // the same answer in every CTA of the cluster
      if (rank == 0)
        for (int i = tid; i < kRows * p.v_cols / 8; i += kThreads) reinterpret_cast<uint4*>(block)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      continue;
    }
    float acc[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.0f;
    const T* a = static_cast<const T*>(p.a) + adapter * p.a_adapter_stride;
    constexpr int kUnroll = (NT * MT <= 4) ? 4 : (NT * MT <= 16 ? 2 : 1);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    // K in steps of 32 per warp: four lanes cover 64 contiguous bytes of a row
    for (int k0 = k_begin + warp * 32; k0 < k_end; k0 += kWarps * 32 * kUnroll) {
      uint4 xa[kUnroll][MT][2], bb[kUnroll][NT];
#pragma unroll
      for (int s = 0; s < kUnroll; ++s) {
        const int k = k0 + s * kWarps * 32 + q * 8;
        const bool in_k = k < k_end;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int r = n * 8 + g;
          bb[s][n] = in_k && r < p.rank ? __ldg(reinterpret_cast<const uint4*>(a + r * p.a_row_stride + k)) : zero;
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int t = row0 + m * 16 + h * 8 + g;
            xa[s][m][h] = in_k && t < p.tokens ? __ldg(reinterpret_cast<const uint4*>(x + t * p.x_stride + k)) : zero;
          }
      }
#pragma unroll
      for (int s = 0; s < kUnroll; ++s)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            mma_16816<T>(acc[m][n], xa[s][m][0].x, xa[s][m][1].x, xa[s][m][0].y, xa[s][m][1].y, bb[s][n].x, bb[s][n].y);
            mma_16816<T>(acc[m][n], xa[s][m][0].z, xa[s][m][1].z, xa[s][m][0].w, xa[s][m][1].w, bb[s][n].z, bb[s][n].w);
          }
    }
    // the warps' sums, one n-tile at a time
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        s_red[warp][m * 16 + g][2 * q] = acc[m][n][0];
        s_red[warp][m * 16 + g][2 * q + 1] = acc[m][n][1];
        s_red[warp][m * 16 + g + 8][2 * q] = acc[m][n][2];
        s_red[warp][m * 16 + g + 8][2 * q + 1] = acc[m][n][3];
      }
      __syncthreads();
      for (int i = tid; i < kRows * 8; i += kThreads) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += s_red[w][i >> 3][i & 7];
        s_part[i >> 3][n * 8 + (i & 7)] = v;
      }
      __syncthreads();
    }
    if (p.splits > 1) {
      cluster_arrive();
      cluster_wait();
    }
    const float scale = p.scales != nullptr ? p.scales[adapter] : 1.0f;
    // the CTAs of a cluster write a share of the block each
    for (int i = tid + rank * kThreads; i < kRows * p.v_cols; i += kThreads * p.splits) {
      const int r = i / p.v_cols, c = i - r * p.v_cols;
      float v = 0.0f;
      if (c < p.rank && s_ids[row0 - tile_row0 + r] == adapter)
        v = scale * (p.splits > 1 ? cluster_sum(&s_part[r][c], p.splits) : s_part[r][c]);
      block[i] = cast16<T>(v);
    }
    if (p.splits > 1) {  // nobody overwrites or leaves its sums while another CTA still reads them
      cluster_arrive();
      cluster_wait();
    } else {
      __syncthreads();
    }
  }
}

template <typename T, int NT, int MT>
int project_launch(const ProjectParams& p, int runs, int stripes, cudaStream_t stream) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(static_cast<unsigned>(runs * p.splits), static_cast<unsigned>(stripes), 1);
  lc.blockDim = dim3(kThreads, 1, 1);
  lc.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.splits);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  lc.attrs = attr;
  lc.numAttrs = 1;
  if (pdl_enabled()) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    lc.numAttrs = 2;
  }
  cudaError_t e = cudaLaunchKernelEx(&lc, lora_project_kernel<T, NT, MT>, p);
  if (e != cudaSuccess) return cuda_fail(e, "lora_project_kernel launch");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return TB_OK;
}

// Rows a block of the projection takes: 16 for a decode batch, 64 (32 with ranks above 64, whose sums fill the registers) for
// longer ones, where it is the re-reading of A out of L2 that counts.
int project_rows(int tokens, int rank) { return tokens <= 64 ? 16 : (rank > 64 ? 32 : 64); }

template <typename T>
int project(const ProjectParams& p, int runs, int stripes, cudaStream_t stream) {
  if (p.tokens <= 64) {
    if (p.rank <= 16) return project_launch<T, 2, 1>(p, runs, stripes, stream);
    if (p.rank <= 32) return project_launch<T, 4, 1>(p, runs, stripes, stream);
    if (p.rank <= 64) return project_launch<T, 8, 1>(p, runs, stripes, stream);
    return project_launch<T, 16, 1>(p, runs, stripes, stream);
  }
  if (p.rank <= 16) return project_launch<T, 2, 4>(p, runs, stripes, stream);
  if (p.rank <= 32) return project_launch<T, 4, 4>(p, runs, stripes, stream);
  if (p.rank <= 64) return project_launch<T, 8, 4>(p, runs, stripes, stream);
  return project_launch<T, 16, 2>(p, runs, stripes, stream);
}

// How a call is cut and where its pieces stand in the workspace.
struct LoraPlan {
  tb_config cfg;
  int streamk;
  int tile_rows, tiles, max_slots, v_cols;
  long long v_offset, v_rows, list_offset, gemm_offset, gemm_bytes, bytes;
};

int lora_plan(const tb_lora_args& a, tb_gemm_args* g, LoraPlan* l) {
  *g = {};
  g->m = a.m; g->n = a.n; g->k = a.k;
  g->a_dtype = g->b_dtype = g->c_dtype = a.dtype;
  g->a = a.x; g->a_stride_m = a.m > 1 ? a.x_row_stride : a.k; g->a_stride_k = 1;
  g->b = a.w; g->b_stride_k = a.w_stride_k; g->b_stride_n = a.w_stride_n;
  g->c = a.out; g->c_stride_m = a.out_stride_m; g->c_stride_n = a.out_stride_n;
  g->bias = a.bias; g->bias_stride = a.bias_stride; g->bias_dtype = a.bias_dtype;
  g->wait_timeout_ms = a.wait_timeout_ms;
  const int rc = low_rank_config(*g, &l->cfg, &l->streamk);
  if (rc != TB_OK) return rc;
  const int pair = l->cfg.cta_pair == 2 ? 2 : 1;
  l->tile_rows = l->cfg.swap_ab ? l->cfg.block_n : 128 * pair;
  l->tiles = (a.m + l->tile_rows - 1) / l->tile_rows;
  l->max_slots = l->tile_rows < a.num_adapters ? l->tile_rows : a.num_adapters;
  l->v_cols = (a.rank + 63) / 64 * 64;
  l->v_rows = static_cast<long long>(l->tiles) * l->max_slots * l->tile_rows;
  auto up = [](long long v) { return (v + 255) & ~255ll; };
  l->gemm_offset = 0;
  l->gemm_bytes = l->streamk ? up(tb_gemm_workspace_bytes(&l->cfg, 0)) : 0;
  l->list_offset = l->gemm_bytes;
  l->v_offset = l->list_offset + up(4ll * l->tiles * (1 + l->max_slots));
  l->bytes = l->v_offset + up(l->v_rows * l->v_cols * 2);
  return TB_OK;
}

bool lora_sizes_ok(const tb_lora_args& a) {
  return a.m >= 0 && a.n >= 0 && a.k >= 8 && a.k % 8 == 0 && a.rank >= 8 && a.rank % 8 == 0 && a.rank <= kMaxRank &&
         a.num_adapters >= 1 && (a.dtype == TB_DTYPE_BF16 || a.dtype == TB_DTYPE_F16);
}

int lora_impl(const tb_lora_args& a, cudaStream_t stream) {
  if (a.dtype != TB_DTYPE_BF16 && a.dtype != TB_DTYPE_F16) return TB_ERR_UNSUPPORTED;
  if (!lora_sizes_ok(a)) return TB_ERR_INVALID;
  if (a.m == 0 || a.n == 0) return TB_OK;
  if (a.x == nullptr || a.w == nullptr || a.lora_a == nullptr || a.lora_b == nullptr || a.adapter_ids == nullptr || a.out == nullptr)
    return TB_ERR_INVALID;
  if ((a.m > 1 && a.x_row_stride < a.k) || a.lora_a_row_stride < a.k || a.lora_b_row_stride < a.rank || a.lora_a_adapter_stride < 0 ||
      a.lora_b_adapter_stride < 0 || (a.w_stride_k != 1 && a.w_stride_n != 1))
    return TB_ERR_INVALID;
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.lora_a) |
                              reinterpret_cast<uintptr_t>(a.lora_b) | reinterpret_cast<uintptr_t>(a.workspace);
  const int64_t strides = (a.m > 1 ? a.x_row_stride : 0) | a.lora_a_row_stride | a.lora_b_row_stride |
                          (a.num_adapters > 1 ? a.lora_a_adapter_stride | a.lora_b_adapter_stride : 0) |
                          (a.w_stride_k == 1 ? (a.n > 1 ? a.w_stride_n : 0) : a.w_stride_k);
  if (addresses % 16 || strides % 8 || reinterpret_cast<uintptr_t>(a.adapter_ids) % (a.ids_are_int64 ? 8 : 4) ||
      reinterpret_cast<uintptr_t>(a.scales) % 4)
    return TB_ERR_ALIGNMENT;
  tb_gemm_args g;
  LoraPlan l;
  int rc = lora_plan(a, &g, &l);
  if (rc != TB_OK) return rc;
  if (a.workspace == nullptr || a.workspace_bytes < l.bytes) return TB_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a.workspace) % 256) return TB_ERR_ALIGNMENT;
  int device = 0, num_sms = 0, smem_optin = 0;
  int* status = nullptr;
  if ((rc = current_device_limits(&device, &num_sms, &smem_optin, &status)) != TB_OK) return rc;
  char* ws = static_cast<char*>(a.workspace);

  ProjectParams p = {};
  p.x = a.x; p.x_stride = g.a_stride_m;
  p.a = a.lora_a; p.a_adapter_stride = a.lora_a_adapter_stride; p.a_row_stride = a.lora_a_row_stride;
  p.ids = a.adapter_ids; p.is64 = a.ids_are_int64 != 0;
  p.scales = a.scales;
  p.tokens = a.m; p.k = a.k; p.rank = a.rank; p.num_adapters = a.num_adapters;
  p.tile_rows = l.tile_rows; p.max_slots = l.max_slots; p.v_cols = l.v_cols;
  p.v = ws + l.v_offset;
  p.list = reinterpret_cast<int*>(ws + l.list_offset);
  p.flags = reinterpret_cast<unsigned*>(ws + l.gemm_offset);
  p.flag_words = l.streamk ? static_cast<int>(kFlagBytes / 4) : 0;
  // Runs cover whole tiles: the rows behind the last token are zeros in every block. Adapters are dealt over up to two blocks
  // per SM, and what is left of those goes along K (at least 512 elements each).
  const int rows = project_rows(a.m, a.rank);
  const int runs = l.tiles * (l.tile_rows / rows);
  const int live_runs = (a.m + rows - 1) / rows;
  int stripes = 2 * num_sms / live_runs;
  const int most = rows < l.max_slots ? rows : l.max_slots;
  stripes = stripes < 1 ? 1 : (stripes > most ? most : stripes);
  p.splits = 1;
  while (p.splits < 8 && live_runs * stripes * p.splits * 2 <= 2 * num_sms && a.k / (p.splits * 2) >= 512) p.splits *= 2;
  p.k_chunk = ((a.k + p.splits - 1) / p.splits + 31) / 32 * 32;
  rc = a.dtype == TB_DTYPE_BF16 ? project<__nv_bfloat16>(p, runs, stripes, stream) : project<__half>(p, runs, stripes, stream);
  if (rc != TB_OK) return rc;

  g.streamk = l.streamk;
  g.workspace = ws + l.gemm_offset;
  g.workspace_bytes = l.gemm_bytes;
  g.epoch = 1;  // the projection clears the flags of every call
  LowRank lr = {};
  lr.v = p.v;
  lr.v_rows = l.v_rows;
  lr.kblocks = l.v_cols / 64;
  lr.rank = a.rank;
  lr.tile_rows = l.tile_rows;
  lr.b = a.lora_b;
  lr.b_adapter_stride = a.lora_b_adapter_stride;
  lr.b_row_stride = a.lora_b_row_stride;
  lr.num_adapters = a.num_adapters;
  lr.n = a.n;
  lr.list = p.list;
  lr.list_stride = 1 + l.max_slots;
  return gemm_low_rank(g, l.cfg, lr, stream);
}

}  // namespace
}  // namespace tb

extern "C" int64_t tb_lora_workspace_bytes(const tb_lora_args* args) {
  if (args == nullptr || !tb::lora_sizes_ok(*args) || args->m == 0 || args->n == 0) return 0;
  tb_gemm_args g;
  tb::LoraPlan l;
  return tb::lora_plan(*args, &g, &l) == TB_OK ? l.bytes : 0;
}

extern "C" int tb_lora_gemm(const tb_lora_args* args, void* stream) {
  if (args == nullptr) return TB_ERR_INVALID;
  return tb::lora_impl(*args, static_cast<cudaStream_t>(stream));
}
