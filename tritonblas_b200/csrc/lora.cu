// A shared projection with one low-rank adapter per row (the requests of a batch, each with its own):
//     out[t] = x[t] W + bias + s_a (x[t] A_a^T) B_a^T,   a = adapter_ids[t]  (outside [0, num_adapters): no adapter)
//
// Two launches. The first one forms v[t] = s_a x[t] A_a^T (rank numbers per row) and lays it out for the second: for every tile of
// rows that the product works on, the list of the adapters that occur in it and, per listed adapter, a block of the tile's rows
// that holds v in that adapter's rows and zeros in all others. The product (lora_decode.cu up to 64 rows, gemm_kernel with
// LOWRANK above) then walks those blocks against the adapters' B as further K stages of the same tile, so the update costs its
// bytes and no pass over the output, and the sum is rounded once. It starts while the first launch still runs. No CTA of
// either waits for one outside its own cluster, so calls on several streams cannot block each other.
//
// The projection is bound by reading x and the used adapters' A once; it has a form for decode batches (mostly one adapter per
// row) and one for longer ones.
//
// Rounding: all sums are fp32. v is an operand of a tensor-core product, so it is kept as two 16-bit halves, v = hi + lo with
// lo = round(v - hi), which stand side by side in a row of its block, 16 to 64 ranks at a time, and are both multiplied by the same
// rows of B. That holds v to 2^-16 (bf16), or to 2^-22 or 2^-25 absolute, whichever is more (fp16, whose v is infinite above 65504:
// the update adds up in the product's own accumulator, so it can have no unit of its own).
// An infinity or NaN in one adapter's B would reach the tile's other rows, whose blocks hold zeros: see low_rank.cuh.
// No reference counterpart (the reference has no adapters).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>

#include "common_host.h"
#include "low_rank.cuh"
#include "selector.h"  // the SM count when there is no device
#include "ptx.cuh"
#include "token_ops.cuh"

namespace tb {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxRank = 128;
constexpr int kMaxStages = 6;
constexpr int kMaxTileRows = 256;
constexpr int kTableBits = 9, kTable = 1 << kTableBits;
constexpr long long kCounterBytes = 4096;  // four counters per dealt tile, of which there are fewer than SMs

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
  int v_width;          // ranks of a stage of the product: a block's row is their high halves, then the low ones, for v_cols ranks
  int v_cols;           // rank rounded up to a multiple of v_width
  int splits;           // CTAs of a cluster that share K
  int k_chunk;          // K per CTA, a multiple of 32
  void* v;
  int* list;            // [tiles][1 + max_slots]
  LowRankRows rows;     // left in the workspace for the second launch
  LowRankRows* rows_out;
  unsigned* counters;   // of the decode kernel, to clear
  int counter_words;
  // tensor-core form
  int rank_pad;         // rank rounded up to 16
  int stages, stage_bytes, tmem_cols;
  uint32_t idesc;
  int* status;
  unsigned long long timeout_ns;
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
// The two halves of v; an infinite v has no low half (inf - inf).
template <typename T>
__device__ __forceinline__ T low_half(float v, T hi) {
  const float rest = v - static_cast<float>(hi);
  return cast16<T>(fabsf(rest) < __builtin_huge_valf() ? rest : 0.0f);
}

// Sum of one float per CTA of the cluster (at most 8) at the same shared-memory offset, in rank order.
__device__ __forceinline__ float cluster_sum(const float* mine, int splits) {
  const uint32_t addr = smem_u32(mine);
  float v[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    v[r] = 0.0f;
    if (r < splits) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[r]) : "r"(mapa_cluster(addr, r)) : "memory");
  }
  float s = v[0];
#pragma unroll
  for (int r = 1; r < 8; ++r) s += v[r];
  return s;
}

// The same for eight floats `pitch` apart; the loads of four CTAs are all in flight before the first sum.
__device__ __forceinline__ void cluster_sum8(const float* mine, int pitch, int splits, float (&sum)[8]) {
  const uint32_t addr = smem_u32(mine);
#pragma unroll
  for (int j = 0; j < 8; ++j) sum[j] = 0.0f;
  for (int r0 = 0; r0 < splits; r0 += 4) {
    float v[4][8];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t remote = mapa_cluster(addr, min(r0 + r, splits - 1));
#pragma unroll
      for (int j = 0; j < 8; ++j) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[r][j]) : "r"(remote + j * pitch * 4) : "memory");
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r0 + r < splits) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += v[r][j];
      }
  }
}

// What a block knows about its run of kRows rows: the adapters that occur in it and where they stand in its tile's list.
template <int kRows>
struct RunLists {
  int ids[kMaxTileRows];                                                       // of the tile's rows; -1 = no adapter
  int key[kTable], first[kTable], run_first[kTable], slot[kTable];             // adapters of the tile, hashed
  int run_ids[kRows], run_slots[kRows];                                        // adapters of the run, by their first rows
  bool present[kMaxTileRows];                                                  // per place in the list: occurs in the run
  int firsts[2][kWarps];
};

// Fills `l` for the run of kRows rows at row0 (all threads of a block of kThreads, ends with a barrier), writes the tile's list
// (`writer`: the one block of the tile that does) and returns the lengths of the tile's and of the run's list. Adapters stand in
// the order of their first rows, so every block of a tile finds the same list; equal ids meet in a small hash table that keeps
// the lowest row.
template <int kRows>
__device__ __forceinline__ int2 find_adapters(const ProjectParams& p, RunLists<kRows>& l, int row0, bool writer) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tile = row0 / p.tile_rows, tile_row0 = tile * p.tile_rows;
  const int run_row = tid - (row0 - tile_row0);  // row of the run this thread speaks for, if it is one
  const bool in_run = run_row >= 0 && run_row < kRows;
  int id = -1;
  if (tid < p.tile_rows && tile_row0 + tid < p.tokens) {
    const long long v = p.is64 ? static_cast<const long long*>(p.ids)[tile_row0 + tid]
                               : static_cast<long long>(static_cast<const int*>(p.ids)[tile_row0 + tid]);
    if (v >= 0 && v < p.num_adapters) id = static_cast<int>(v);
  }
  l.ids[tid] = id;
  for (int i = tid; i < kTable; i += kThreads) {
    l.key[i] = -1;
    l.first[i] = l.run_first[i] = kMaxTileRows;
  }
  __syncthreads();
  int entry = static_cast<int>((static_cast<unsigned>(id) * 2654435761u) >> (32 - kTableBits));
  if (id >= 0) {
    while (true) {  // the table has twice as many places as the tile has rows: a free one always comes
      const int before = atomicCAS(&l.key[entry], -1, id);
      if (before == -1 || before == id) break;
      entry = (entry + 1) & (kTable - 1);
    }
    atomicMin(&l.first[entry], tid);
    if (in_run) atomicMin(&l.run_first[entry], run_row);
  }
  __syncthreads();
  const bool first = id >= 0 && l.first[entry] == tid;
  const bool run_first = id >= 0 && in_run && l.run_first[entry] == run_row;
  const unsigned votes = __ballot_sync(0xffffffffu, first), run_votes = __ballot_sync(0xffffffffu, run_first);
  if (lane == 0) {
    l.firsts[0][warp] = __popc(votes);
    l.firsts[1][warp] = __popc(run_votes);
  }
  __syncthreads();
  const unsigned below = (1u << lane) - 1u;
  int slot_of_first = __popc(votes & below), turn_of_first = __popc(run_votes & below), count = 0, present = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) {
      slot_of_first += l.firsts[0][w];
      turn_of_first += l.firsts[1][w];
    }
    count += l.firsts[0][w];
    present += l.firsts[1][w];
  }
  int* list = p.list + static_cast<long long>(tile) * (1 + p.max_slots);
  if (first) {
    l.slot[entry] = slot_of_first;
    l.present[slot_of_first] = l.run_first[entry] < kMaxTileRows;
    if (writer) list[1 + slot_of_first] = id;
  }
  if (writer && tid == 0) list[0] = count;
  __syncthreads();
  if (run_first) {
    l.run_ids[turn_of_first] = id;
    l.run_slots[turn_of_first] = l.slot[entry];
  }
  __syncthreads();
  return make_int2(count, present);
}

// The run's rows in the blocks of the tile's other adapters are zeros; dealt over the blocks of the grid's y axis.
template <int kRows, typename T>
__device__ __forceinline__ void clear_absent(const ProjectParams& p, const RunLists<kRows>& l, T* tile_blocks, int count, int rank) {
  const long long block_stride = static_cast<long long>(p.tile_rows) * 2 * p.v_cols;
  for (int slot = blockIdx.y; slot < count; slot += gridDim.y) {
    if (l.present[slot]) continue;
    uint4* block = reinterpret_cast<uint4*>(tile_blocks + slot * block_stride);
    for (int i = threadIdx.x + rank * kThreads; i < kRows * 2 * p.v_cols / 8; i += kThreads * p.splits) block[i] = make_uint4(0, 0, 0, 0);
  }
}

__device__ __forceinline__ void cluster_or_block_sync(int splits) {
  if (splits > 1) {
    __syncwarp();  // the cluster barrier's instructions are .aligned, and what comes before them here branches per lane
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------------ decode batches
// One cluster (of `splits` CTAs along K) per run of 16 rows; blockIdx.y deals the adapters of the run, 8 NT ranks at a time. Every
// warp takes K slices and loads both operands straight into the fragments of mma.sync (16 bytes per lane and row; the order of K
// inside a slice is the same for both, so it need not be the instruction's).
// 120 registers: see lora_decode_kernel, whose block is to join this one's on its SM.
template <typename T, int NT>
__global__ void __maxnreg__(120) lora_project_kernel(const ProjectParams p) {
  constexpr int kRows = 16, kCols = 8 * NT;
  __shared__ RunLists<kRows> lists;
  __shared__ float s_red[kWarps][kRows][8];
  __shared__ float s_part[kRows][kCols];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = p.splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int run = blockIdx.x / p.splits;
  const int row0 = run * kRows;                 // first row of the run
  const int tile = row0 / p.tile_rows, tile_row0 = tile * p.tile_rows;
  griddep_wait();
  griddep_launch_dependents();

  if (blockIdx.x == 0 && blockIdx.y == 0) {
    for (int i = tid; i < p.counter_words; i += kThreads) p.counters[i] = 0u;
    if (tid == 0) *p.rows_out = p.rows;
  }
  const int2 found = find_adapters<kRows>(p, lists, row0, row0 == tile_row0 && blockIdx.y == 0 && rank == 0);
  const int* run_ids = lists.ids + (row0 - tile_row0);
  const int v_row = 2 * p.v_cols;
  T* tile_blocks = static_cast<T*>(p.v) + static_cast<long long>(tile) * p.max_slots * p.tile_rows * v_row +
                   static_cast<long long>(row0 - tile_row0) * v_row;
  clear_absent<kRows>(p, lists, tile_blocks, found.x, rank);

  const T* x = static_cast<const T*>(p.x);
  const int g = lane >> 2, q = lane & 3;
  const int k_begin = rank * p.k_chunk, k_end = min(p.k, k_begin + p.k_chunk);
  const int slices = (p.rank + kCols - 1) / kCols;
  for (int item = blockIdx.y; item < found.y * slices; item += gridDim.y) {
    const int turn = item / slices, c0 = (item - turn * slices) * kCols;  // first rank of the slice
    const int ranks = p.rank - c0;
    const int adapter = lists.run_ids[turn];
    T* block = tile_blocks + lists.run_slots[turn] * static_cast<long long>(p.tile_rows) * v_row +
               2 * (c0 & ~(p.v_width - 1)) + (c0 & (p.v_width - 1));  // kCols divides v_width
    const float scale = p.scales != nullptr ? __ldg(p.scales + adapter) : 1.0f;
    // only rows with this adapter are read; the others enter the product as zeros
    bool live[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) live[h] = run_ids[h * 8 + g] == adapter;
    const T* x_lane = x + (row0 + g) * p.x_stride + q * 8;
    const T* a_lane = static_cast<const T*>(p.a) + adapter * p.a_adapter_stride + (c0 + g) * p.a_row_stride + q * 8;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
    constexpr int kUnroll = 4;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    // K in steps of 32 per warp: four lanes cover 64 contiguous bytes of a row
    for (int k0 = k_begin + warp * 32; k0 < k_end; k0 += kWarps * 32 * kUnroll) {
      uint4 xa[kUnroll][2], bb[kUnroll][NT];
#pragma unroll
      for (int s = 0; s < kUnroll; ++s) {
        const int k = k0 + s * kWarps * 32;
        const bool in_k = k + q * 8 < k_end;
#pragma unroll
        for (int n = 0; n < NT; ++n)
          bb[s][n] = in_k && n * 8 < ranks ? __ldg(reinterpret_cast<const uint4*>(a_lane + n * 8 * p.a_row_stride + k)) : zero;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          xa[s][h] = in_k && live[h] ? __ldg(reinterpret_cast<const uint4*>(x_lane + h * 8 * p.x_stride + k)) : zero;
      }
#pragma unroll
      for (int s = 0; s < kUnroll; ++s) {
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_16816<T>(acc[n], xa[s][0].x, xa[s][1].x, xa[s][0].y, xa[s][1].y, bb[s][n].x, bb[s][n].y);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_16816<T>(acc[n], xa[s][0].z, xa[s][1].z, xa[s][0].w, xa[s][1].w, bb[s][n].z, bb[s][n].w);
      }
    }
    // the warps' sums, one n-tile at a time
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      s_red[warp][g][2 * q] = acc[n][0];
      s_red[warp][g][2 * q + 1] = acc[n][1];
      s_red[warp][g + 8][2 * q] = acc[n][2];
      s_red[warp][g + 8][2 * q + 1] = acc[n][3];
      __syncthreads();
      for (int i = tid; i < kRows * 8; i += kThreads) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += s_red[w][i >> 3][i & 7];
        s_part[i >> 3][n * 8 + (i & 7)] = v;
      }
      __syncthreads();
    }
    cluster_or_block_sync(p.splits);
    // the CTAs of a cluster write a share of the block each
    for (int i = tid + rank * kThreads; i < kRows * kCols; i += kThreads * p.splits) {
      const int r = i / kCols, c = i % kCols;
      float v = 0.0f;
      if (c < ranks && run_ids[r] == adapter)
        v = scale * (p.splits > 1 ? cluster_sum(&s_part[r][c], p.splits) : s_part[r][c]);
      const T hi = cast16<T>(v);
      block[r * v_row + c] = hi;
      block[r * v_row + p.v_width + c] = low_half<T>(v, hi);
    }
    cluster_or_block_sync(p.splits);  // nobody overwrites or leaves its sums while another CTA still reads them
  }
}

// ------------------------------------------------------------------------------------------------------ longer batches
// One cluster (of `splits` CTAs along K) per run of 128 rows; blockIdx.y deals the adapters of the run. A product of the run's
// rows with the adapter's `rank` rows on the tensor cores: TMA into a ring, one MMA warp, the accumulator read back, the CTAs'
// partial sums joined over the cluster in rank order. Warps: 0 loads, 1 issues, 4-7 read the accumulator; all write v.
// Every thread reaches every barrier whether its waits succeeded or not, so a wait that runs out ends the kernel.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
lora_project_tc_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_a, const ProjectParams p) {
  constexpr int kRows = 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* part = reinterpret_cast<float*>(ring);  // [rank_pad][128] partial sums, over the drained ring
  __shared__ RunLists<kRows> lists;
  __shared__ uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], acc_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_word;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = p.splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int row0 = static_cast<int>(blockIdx.x) / p.splits * kRows;
  const int tile = row0 / p.tile_rows, tile_row0 = tile * p.tile_rows;
  const WaitCtx wctx{&abort_word, p.status, p.timeout_ns};
  if (tid == 0) {
    abort_word = 0;
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(&acc_bar, 1);
    mbar_fence_init();
    prefetch_tmap(&tmap_x);
    prefetch_tmap(&tmap_a);
  }
  if (warp == 1) {
    tmem_alloc<1>(&tmem_slot, static_cast<uint32_t>(p.tmem_cols));
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) *p.rows_out = p.rows;
  const int2 found = find_adapters<kRows>(p, lists, row0, row0 == tile_row0 && blockIdx.y == 0 && cta == 0);
  const int* run_ids = lists.ids + (row0 - tile_row0);
  const int v_row = 2 * p.v_cols, width = p.v_width;
  T* tile_blocks = static_cast<T*>(p.v) + static_cast<long long>(tile) * p.max_slots * p.tile_rows * v_row +
                   static_cast<long long>(row0 - tile_row0) * v_row;
  clear_absent<kRows>(p, lists, tile_blocks, found.x, cta);

  const int kb_begin = cta * p.k_chunk / 64;
  const int kbs = max(0, min((p.k + 63) / 64, kb_begin + p.k_chunk / 64) - kb_begin);
  int s = 0;
  uint32_t ph = 0, acc_ph = 0;
  for (int turn = blockIdx.y; turn < found.y; turn += gridDim.y) {
    const int adapter = lists.run_ids[turn];
    T* block = tile_blocks + lists.run_slots[turn] * static_cast<long long>(p.tile_rows) * v_row;
    const float scale = p.scales != nullptr ? __ldg(p.scales + adapter) : 1.0f;
    if (abort_word) {
      // an earlier turn's wait ran out: nothing more is loaded or multiplied
    } else if (warp == 0) {
      fence_proxy_async_smem();  // the last turn's sums stood where the copies land
      for (int kb = 0; kb < kbs; ++kb) {
        if (!mbar_wait_warp(&empty_bar[s], ph ^ 1, wctx, TB_DEV_TIMEOUT_SMEM_EMPTY)) break;
        if (elect_one()) {
          uint8_t* dst = ring + static_cast<size_t>(s) * p.stage_bytes;
          mbar_arrive_expect_tx(&full_bar[s], static_cast<uint32_t>(p.stage_bytes));
          tma_load_2d(dst, &tmap_x, &full_bar[s], (kb_begin + kb) * 64, row0);
          tma_load_3d(dst + kRows * 128, &tmap_a, &full_bar[s], (kb_begin + kb) * 64, 0, adapter);
        }
        __syncwarp();
        if (++s == p.stages) {
          s = 0;
          ph ^= 1;
        }
      }
    } else if (warp == 1) {
      const uint64_t desc0 = make_smem_desc(smem_u32(ring), 16, 1024);
      bool ok = true;
      tc_fence_after();  // the last turn's sums have been read
      for (int kb = 0; kb < kbs; ++kb) {
        ok = mbar_wait_warp(&full_bar[s], ph, wctx, TB_DEV_TIMEOUT_SMEM_FULL);
        if (!ok) break;
        if (elect_one()) {
          const uint64_t a = desc0 + static_cast<uint64_t>((s * p.stage_bytes) >> 4), b = a + ((kRows * 128) >> 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma<0, 1>(tmem_base, a + 2 * k, b + 2 * k, p.idesc, (kb > 0 || k > 0) ? 1u : 0u);
          umma_commit(&empty_bar[s]);
          if (kb + 1 == kbs) umma_commit(&acc_bar);
        }
        __syncwarp();
        if (++s == p.stages) {
          s = 0;
          ph ^= 1;
        }
      }
    } else if (warp >= 4) {
      const int r = (warp & 3) * 32 + lane;
      bool ok = true;
      if (kbs > 0) ok = __all_sync(0xffffffffu, mbar_wait(&acc_bar, acc_ph, wctx, TB_DEV_TIMEOUT_TMEM_FULL));
      tc_fence_after();
      for (int c0 = 0; c0 < p.rank_pad; c0 += 32) {
        uint32_t v[32];
        if (ok && kbs > 0) {
          tmem_ld_32x32(tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + c0, v);
          tmem_ld_wait(v);
        }
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c0 + j < p.rank_pad) part[(c0 + j) * kRows + r] = kbs > 0 ? __uint_as_float(v[j]) : 0.0f;
      }
      tc_fence_before();
    }
    if (kbs > 0) acc_ph ^= 1;
    cluster_or_block_sync(p.splits);
    // the CTAs of a cluster write a share of the rows each, eight ranks per thread
    const int share = kRows / p.splits, groups = p.v_cols / 8;
    for (int i = tid; i < share * groups; i += kThreads) {
      const int r = cta * share + i % share, c = i / share * 8;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.0f;
      if (c < p.rank && run_ids[r] == adapter) {
        const float* mine = part + c * kRows + r;
        if (p.splits > 1) {
          cluster_sum8(mine, kRows, p.splits, v);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = mine[j * kRows];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= scale;
      }
      alignas(16) T hi[8], lo[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        hi[j] = cast16<T>(v[j]);
        lo[j] = low_half<T>(v[j], hi[j]);
      }
      T* o = block + static_cast<long long>(r) * v_row + 2 * (c & ~(width - 1)) + (c & (width - 1));
      *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(hi);
      *reinterpret_cast<uint4*>(o + width) = *reinterpret_cast<const uint4*>(lo);
    }
    cluster_or_block_sync(p.splits);  // nobody overwrites or leaves its sums while another CTA still reads them
  }
  if (abort_word) {
    // A wait gave up: let copies and MMAs already in flight land before shared memory and TMEM are released.
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, static_cast<uint32_t>(p.tmem_cols));
  }
}

// The carve-out is asked for at its largest: an SM keeps the division between L1 and shared memory while blocks run on it, and the
// second launch's blocks are to join these (1 row of 4096 x 4096: 15.0 -> 14.5 us at the time).
template <typename K>
int prefer_shared(K kernel, int device, bool (&done)[64]) {
  static std::mutex mu;
  std::lock_guard<std::mutex> lk(mu);
  if (!done[device & 63]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(carveout)");
    done[device & 63] = true;
  }
  return TB_OK;
}

template <typename... Params, typename... Args>
int project_launch(void (*kernel)(Params...), int runs, const ProjectParams& p, int stripes, int smem_bytes, cudaStream_t stream,
                   Args... args) {
  return launch_token_kernel(kernel, dim3(static_cast<unsigned>(runs * p.splits), static_cast<unsigned>(stripes), 1), kThreads, smem_bytes, p.splits,
                             stream, "lora_project_kernel launch", args..., p);
}

template <typename T, int NT>
int project_decode_nt(const ProjectParams& p, int runs, int stripes, int device, cudaStream_t stream) {
  static bool done[64] = {};
  const int rc = prefer_shared(lora_project_kernel<T, NT>, device, done);
  return rc != TB_OK ? rc : project_launch(lora_project_kernel<T, NT>, runs, p, stripes, 0, stream);
}

template <typename T>
int project_decode(const ProjectParams& p, int runs, int stripes, int device, cudaStream_t stream) {
  if (p.rank <= 16) return project_decode_nt<T, 2>(p, runs, stripes, device, stream);
  return project_decode_nt<T, 4>(p, runs, stripes, device, stream);
}

template <typename T>
int project_tc(const tb_lora_args& a, ProjectParams& p, int runs, int stripes, int device, cudaStream_t stream) {
  p.rank_pad = (p.rank + 15) / 16 * 16;
  p.stage_bytes = (128 + p.rank_pad) * 128;
  p.stages = 96 * 1024 / p.stage_bytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  p.tmem_cols = 32;
  while (p.tmem_cols < p.rank_pad) p.tmem_cols <<= 1;
  p.idesc = (1u << 4) | ((a.dtype == TB_DTYPE_BF16 ? 1u : 0u) * ((1u << 7) | (1u << 10))) |
            (static_cast<uint32_t>(p.rank_pad >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
  // the ring also holds a CTA's sums once it is drained
  const int ring = p.stages * p.stage_bytes;
  const int smem_bytes = (ring > p.rank_pad * 512 ? ring : p.rank_pad * 512) + 1024;
  CUtensorMap tx, ta;
  int rc = encode_2d(&tx, a.dtype, a.x, a.k, a.m, static_cast<uint64_t>(p.x_stride) * 2, 64, 128, 1);
  if (rc != TB_OK) return rc;
  const uint64_t dims[3] = {static_cast<uint64_t>(a.k), static_cast<uint64_t>(a.rank), static_cast<uint64_t>(a.num_adapters)};
  const uint64_t strides[2] = {static_cast<uint64_t>(a.lora_a_row_stride) * 2,
                               static_cast<uint64_t>(a.num_adapters > 1 ? a.lora_a_adapter_stride : a.lora_a_row_stride * a.rank) * 2};
  const uint32_t box[3] = {64, static_cast<uint32_t>(p.rank_pad), 1};
  if ((rc = encode_nd(&ta, a.dtype, a.lora_a, 3, dims, strides, box)) != TB_OK) return rc;
  auto kernel = lora_project_tc_kernel<T>;
  static SmemOptIn configured;
  if ((rc = opt_in_smem(kernel, smem_bytes, device, configured, "cudaFuncSetAttribute(lora_project_tc)")) != TB_OK) return rc;
  return project_launch(kernel, runs, p, stripes, smem_bytes, stream, tx, ta);
}

// How a call is cut and where its pieces stand in the workspace.
struct LoraPlan {
  bool decode;
  LoraDecodeShape shape;  // decode
  tb_config cfg;          // otherwise
  int tile_rows, tiles, max_slots, v_cols, v_width, pack, kblocks;
  long long v_offset, v_rows, list_offset, rows_offset, gemm_offset, gemm_bytes, bytes;
};

int lora_plan(const tb_lora_args& a, int num_sms, tb_gemm_args* g, LoraPlan* l) {
  *g = {};
  g->m = a.m; g->n = a.n; g->k = a.k;
  g->a_dtype = g->b_dtype = g->c_dtype = a.dtype;
  g->a = a.x; g->a_stride_m = a.m > 1 ? a.x_row_stride : a.k; g->a_stride_k = 1;
  g->b = a.w; g->b_stride_k = a.w_stride_k; g->b_stride_n = a.w_stride_n;
  g->c = a.out; g->c_stride_m = a.out_stride_m; g->c_stride_n = a.out_stride_n;
  g->bias = a.bias; g->bias_stride = a.bias_stride; g->bias_dtype = a.bias_dtype;
  g->wait_timeout_ms = a.wait_timeout_ms;
  l->decode = a.m <= 64;
  if (l->decode) {
    l->tile_rows = (a.m + 15) / 16 * 16;
  } else {
    const int rc = low_rank_config(*g, &l->cfg);
    if (rc != TB_OK) return rc;
    l->tile_rows = 128 * (l->cfg.cta_pair == 2 ? 2 : 1);
  }
  l->tiles = (a.m + l->tile_rows - 1) / l->tile_rows;
  l->max_slots = l->tile_rows < a.num_adapters ? l->tile_rows : a.num_adapters;
  // small ranks share a stage of the product, which has room for 64 ranks up to 64 rows and for 32 above: see GemmParams::lr_pack
  const int stage_ranks = l->decode ? 64 : 32;
  l->pack = a.rank <= 16 ? stage_ranks / 16 : (a.rank <= 32 ? stage_ranks / 32 : 1);
  l->v_width = stage_ranks / l->pack;
  l->kblocks = (a.rank + l->v_width - 1) / l->v_width;
  l->v_cols = l->kblocks * l->v_width;
  if (l->decode) {
    const int most = a.m < l->max_slots ? a.m : l->max_slots;
    l->shape = lora_decode_shape(a.m, a.n, a.k, (most + l->pack - 1) / l->pack * l->kblocks, num_sms);
  }
  l->v_rows = static_cast<long long>(l->tiles) * l->max_slots * l->tile_rows;
  if (l->v_rows > 0x7fffffffll) return TB_ERR_UNSUPPORTED;  // a row coordinate of a copy has 32 bits; shorter batches fit
  auto up = [](long long v) { return (v + 255) & ~255ll; };
  l->gemm_offset = 0;
  // decode: counters (cleared by the projection) at the front, then partial tiles
  l->gemm_bytes = l->decode ? kCounterBytes + up(l->shape.part_bytes) : 0;
  l->rows_offset = l->gemm_bytes;
  l->list_offset = l->rows_offset + up(sizeof(LowRankRows));
  l->v_offset = l->list_offset + up(4ll * l->tiles * (1 + l->max_slots));
  l->bytes = l->v_offset + up(l->v_rows * 2 * l->v_cols * 2);
  return TB_OK;
}

bool lora_sizes_ok(const tb_lora_args& a) {
  // row, tile and stage numbers have 32 bits; so has the sum of all dealt tiles' stages, fewer tiles than SMs of k / 64 each
  return a.m >= 0 && a.m <= (1 << 30) && a.n >= 0 && a.n <= (1 << 30) && a.k >= 8 && a.k <= (1 << 28) && a.k % 8 == 0 && a.rank >= 8 &&
         a.rank % 8 == 0 && a.rank <= kMaxRank && a.num_adapters >= 1 && (a.dtype == TB_DTYPE_BF16 || a.dtype == TB_DTYPE_F16);
}

int lora_impl(const tb_lora_args& a, cudaStream_t stream) {
  if (a.dtype != TB_DTYPE_BF16 && a.dtype != TB_DTYPE_F16) return TB_ERR_UNSUPPORTED;
  if (!lora_sizes_ok(a)) return TB_ERR_INVALID;
  if (a.m == 0 || a.n == 0) return TB_OK;
  if (a.x == nullptr || a.w == nullptr || a.lora_a == nullptr || a.lora_b == nullptr || a.adapter_ids == nullptr || a.out == nullptr)
    return TB_ERR_INVALID;
  if ((a.m > 1 && a.x_row_stride < a.k) || a.lora_a_row_stride < a.k || a.lora_b_row_stride < a.rank || a.lora_a_adapter_stride < 0 ||
      a.lora_b_adapter_stride < 0 || (a.w_stride_k == 1 ? a.n > 1 && a.w_stride_n < a.k : a.w_stride_n != 1 || a.w_stride_k < a.n))
    return TB_ERR_INVALID;
  const uintptr_t addresses = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.lora_a) |
                              reinterpret_cast<uintptr_t>(a.lora_b) | reinterpret_cast<uintptr_t>(a.workspace);
  const int64_t strides = (a.m > 1 ? a.x_row_stride : 0) | a.lora_a_row_stride | a.lora_b_row_stride |
                          (a.num_adapters > 1 ? a.lora_a_adapter_stride | a.lora_b_adapter_stride : 0) |
                          (a.w_stride_k == 1 ? (a.n > 1 ? a.w_stride_n : 0) : a.w_stride_k);
  if (addresses % 16 || strides % 8 || reinterpret_cast<uintptr_t>(a.adapter_ids) % (a.ids_are_int64 ? 8 : 4) ||
      reinterpret_cast<uintptr_t>(a.scales) % 4 || reinterpret_cast<uintptr_t>(a.out) % 2 ||
      reinterpret_cast<uintptr_t>(a.bias) % (a.bias_dtype == TB_DTYPE_F32 ? 4 : 2))
    return TB_ERR_ALIGNMENT;
  if (a.bias != nullptr && a.bias_dtype != TB_DTYPE_F32 && a.bias_dtype != TB_DTYPE_F16 && a.bias_dtype != TB_DTYPE_BF16)
    return TB_ERR_UNSUPPORTED;
  int device = 0, num_sms = 0, smem_optin = 0;
  int* status = nullptr;
  const int device_rc = current_device_limits(&device, &num_sms, &smem_optin, &status);
  if (device_rc != TB_OK) num_sms = MachineModel().num_sms;  // the other arguments are checked all the same
  tb_gemm_args g;
  LoraPlan l;
  int rc = lora_plan(a, num_sms, &g, &l);
  if (rc != TB_OK) return rc;
  if (a.workspace == nullptr || a.workspace_bytes < l.bytes) return TB_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a.workspace) % 256) return TB_ERR_ALIGNMENT;
  if (device_rc != TB_OK) return device_rc;
  char* ws = static_cast<char*>(a.workspace);

  ProjectParams p = {};
  p.x = a.x; p.x_stride = g.a_stride_m;
  p.a = a.lora_a; p.a_adapter_stride = a.lora_a_adapter_stride; p.a_row_stride = a.lora_a_row_stride;
  p.ids = a.adapter_ids; p.is64 = a.ids_are_int64 != 0;
  p.scales = a.scales;
  p.tokens = a.m; p.k = a.k; p.rank = a.rank; p.num_adapters = a.num_adapters;
  p.tile_rows = l.tile_rows; p.max_slots = l.max_slots; p.v_cols = l.v_cols; p.v_width = l.v_width;
  p.v = ws + l.v_offset;
  p.list = reinterpret_cast<int*>(ws + l.list_offset);
  p.rows = {a.x, g.a_stride_m, a.w, a.w_stride_k, a.w_stride_n, a.lora_b, a.lora_b_adapter_stride, a.lora_b_row_stride, a.adapter_ids,
            p.list, p.v, a.bias, a.bias_stride, a.out, a.out_stride_m, a.out_stride_n, p.is64, a.num_adapters, 1 + l.max_slots,
            2 * l.v_cols, l.v_width, l.tile_rows, a.k, a.rank, a.bias_dtype, a.dtype == TB_DTYPE_BF16 ? 1 : 0};
  p.rows_out = reinterpret_cast<LowRankRows*>(ws + l.rows_offset);
  p.counters = reinterpret_cast<unsigned*>(ws + l.gemm_offset);
  p.counter_words = l.decode ? 4 * l.shape.dealt_tiles : 0;
  p.status = status;
  p.timeout_ns = a.wait_timeout_ms > 0 ? static_cast<unsigned long long>(a.wait_timeout_ms) * 1000000ull : 2000000000ull;
  // Runs cover whole tiles: the rows behind the last token are zeros in every block. A decode batch has up to one adapter per
  // row: they are dealt over blocks first, and K is split as long as there is one block per SM, with an eighth to spare for where
  // clusters do not fit: beside a second one the product's block would have no registers (64 rows of 4096 x 8192, 64 adapters of
  // rank 16: 32.7 us, 34.5 with up to 148 blocks, 37 with 296; 32 rows: 25.2 / 26.3 / 30). Longer batches have few adapters per
  // run: K is split first, up to a block per SM, and what is left of two per SM takes the adapters.
  const bool decode = l.decode;
  const int rows = decode ? 16 : 128;
  const int runs = l.tiles * (l.tile_rows / rows);
  const int live_runs = (a.m + rows - 1) / rows;
  const int most = rows < l.max_slots ? rows : l.max_slots;
  int stripes = 1;
  p.splits = 1;
  if (decode) {
    const int blocks = num_sms * 7 / 8;
    stripes = (most < a.m ? most : a.m) * ((a.rank + 31) / 32);
    if (live_runs * stripes > blocks) stripes = blocks / live_runs;
    const int by_blocks = blocks / (live_runs * stripes), by_k = a.k / 256;
    p.splits = by_blocks < by_k ? by_blocks : by_k;
    p.splits = p.splits < 1 ? 1 : (p.splits > 8 ? 8 : p.splits);
  } else {
    while (p.splits < 8 && live_runs * p.splits * 2 <= num_sms && a.k / (p.splits * 2) >= 256) p.splits *= 2;
    stripes = 2 * num_sms / (live_runs * p.splits);
    stripes = stripes < 1 ? 1 : (stripes > most ? most : stripes);
  }
  const int k_unit = decode ? 32 : 64;
  p.k_chunk = ((a.k + p.splits - 1) / p.splits + k_unit - 1) / k_unit * k_unit;
  const bool bf16 = a.dtype == TB_DTYPE_BF16;
  if (decode)
    rc = bf16 ? project_decode<__nv_bfloat16>(p, runs, stripes, device, stream) : project_decode<__half>(p, runs, stripes, device, stream);
  else
    rc = bf16 ? project_tc<__nv_bfloat16>(a, p, runs, stripes, device, stream) : project_tc<__half>(a, p, runs, stripes, device, stream);
  if (rc != TB_OK) return rc;

  LowRank lr = {};
  lr.v = p.v;
  lr.v_rows = l.v_rows;
  lr.pack = l.pack;
  lr.kblocks = l.kblocks;
  lr.rank = a.rank;
  lr.tile_rows = l.tile_rows;
  lr.b = a.lora_b;
  lr.b_adapter_stride = a.lora_b_adapter_stride;
  lr.b_row_stride = a.lora_b_row_stride;
  lr.num_adapters = a.num_adapters;
  lr.n = a.n;
  lr.rows = p.rows_out;
  lr.list = p.list;
  lr.list_stride = 1 + l.max_slots;
  if (l.decode)
    return lora_decode(a, l.shape, lr, ws + l.gemm_offset + kCounterBytes, ws + l.gemm_offset, device, smem_optin, status, stream);
  return gemm_low_rank(g, l.cfg, lr, stream);
}

}  // namespace
}  // namespace tb

extern "C" int64_t tb_lora_workspace_bytes(const tb_lora_args* args) {
  if (args == nullptr || !tb::lora_sizes_ok(*args) || args->m == 0 || args->n == 0) return 0;
  // without a usable device: the B200's SM count
  int device = 0, num_sms = 0, smem_optin = 0;
  int* status = nullptr;
  if (tb::current_device_limits(&device, &num_sms, &smem_optin, &status) != TB_OK) num_sms = tb::MachineModel().num_sms;
  tb_gemm_args g;
  tb::LoraPlan l;
  return tb::lora_plan(*args, num_sms, &g, &l) == TB_OK ? l.bytes : 0;
}

extern "C" int tb_lora_gemm(const tb_lora_args* args, void* stream) {
  if (args == nullptr) return TB_ERR_INVALID;
  return tb::lora_impl(*args, static_cast<cudaStream_t>(stream));
}
