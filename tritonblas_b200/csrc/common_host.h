// Host-side declarations shared by the translation units of libtritonblas_b200.so.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/tritonblas_b200.h"

namespace tb {

extern std::atomic<long long> g_launches;

int cuda_fail(cudaError_t e, const char* what);
int cu_fail(int code, const char* what);

// Device word that kernels write a failure code into (allocated once per device by the library).
int* device_status_word(int device);

// 2-D row-major tensor map [outer][inner]; box = box_inner x box_outer elements.
int encode_2d(CUtensorMap* map, int dtype, const void* base, uint64_t inner, uint64_t outer, uint64_t outer_stride_bytes,
              uint32_t box_inner, uint32_t box_outer, int swizzle);  // swizzle: 0 none, 1 128B, 2 128B with 32-byte chunks

// Tensor map of any rank up to 5 over 16-bit or wider elements, dims and box innermost first, strides in bytes of dimensions
// 1 .. rank-1; box[0] elements must be 128, 64 or 32 bytes: the swizzle has that width.
int encode_nd(CUtensorMap* map, int dtype, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
              const uint32_t* box);

// Low-rank update of a dense launch (see GemmParams::lr_list): the tokens' masked projections v, one block of tile_rows rows per
// token tile and listed adapter, and lora_b (num_adapters, n, rank). A row is `kblocks` times as many high 16-bit halves as a stage
// has ranks of one adapter (32 / pack, in the decode form 64 / pack) and as many low ones.
struct LowRankRows;  // low_rank.cuh
struct LowRank {
  const void* v;
  int64_t v_rows;
  int kblocks, pack, rank, tile_rows;
  const void* b;
  int64_t b_adapter_stride, b_row_stride;
  int num_adapters, n;
  const int* list;
  int list_stride;
  const LowRankRows* rows;
};
// Configuration the library would pick for `a` (more than 64 rows): data-parallel, narrow tiles; and the launch of `a` with that
// configuration and the update.
int low_rank_config(const tb_gemm_args& a, tb_config* cfg);
int gemm_low_rank(const tb_gemm_args& a, const tb_config& cfg, const LowRank& lr, cudaStream_t stream);

// Decode form of the same product (lora_decode.cu), up to 64 rows: how it is cut, and its launch.
// `parts` holds part_bytes, `arrived` 4 * dealt_tiles zeroed words.
struct LoraDecodeShape {
  int cols, grid, full_tiles, dealt_tiles, deal_ctas, pieces;
  long long part_bytes;
};
LoraDecodeShape lora_decode_shape(int tokens, int n, int k, int update_stages, int grid);
int lora_decode(const tb_lora_args& a, const LoraDecodeShape& s, const LowRank& lr, void* parts, void* arrived, int device,
                int smem_optin, int* status, cudaStream_t stream);

// The current device: its number, SMs, shared memory a block may opt in to, and failure word.
int current_device_limits(int* device, int* num_sms, int* smem_optin, int** status);

}  // namespace tb
