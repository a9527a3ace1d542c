// Elements of a projection with low-rank updates, one by one.
//
// The update of a tile is one matrix product in which rows without an adapter hold zeros in that adapter's block, so an infinity or
// NaN in lora_b[a] makes NaN of rows that have nothing to do with a. Both product kernels look for sums that are not finite
// (one multiply-add per element, nothing else as long as all are) and have those elements formed again from the definition:
//     out[t, n] = sum_k x[t, k] W[k, n] + bias[n] + sum_r v[t, r] B_a[n, r],   a = adapter_ids[t],  no other adapter.
// An element that is not finite by this formula stays so. Only batches with such values pay for it: a warp takes one element at a
// time, and goes by the row's own update and by the row of x first, either of which may hold the NaN itself.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/tritonblas_b200.h"
#include "ptx.cuh"

namespace tb {

// What an element is made of; the first launch leaves it in the workspace, so that the product kernels carry one pointer.
struct LowRankRows {
  const void* x;
  long long x_stride;
  const void* w;
  long long w_k, w_n;
  const void* b;
  long long b_adapter, b_row;
  const void* ids;
  const int* list;
  const void* v;
  const void* bias;
  long long bias_stride;
  void* out;
  long long out_m, out_n;
  int is64, num_adapters, list_stride, v_row, v_width, tile_rows, k, rank, bias_dtype, bf16;
};

namespace low_rank {

__device__ __forceinline__ float from16(unsigned short u, int bf16) {
  return bf16 ? __uint_as_float(static_cast<unsigned>(u) << 16) : __half2float(__ushort_as_half(u));
}
__device__ __forceinline__ bool finite(float f) { return fabsf(f) < __builtin_huge_valf(); }

// Forms the elements of rows [t0, t1) and columns [n0, n1) that came out non-finite again, where another row's adapter can be the
// reason. A whole warp calls it, after its own stores to them.
static __device__ __noinline__ void redo(const LowRankRows* rows, int t0, int t1, int n0, int n1) {
  griddep_wait();  // of the first launch
  __syncwarp();
  LowRankRows a;  // from L2, as all that the first launch wrote
  static_assert(sizeof(LowRankRows) % 8 == 0, "copied in words of eight bytes");
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(LowRankRows) / 8); ++i)
    reinterpret_cast<unsigned long long*>(&a)[i] = __ldcg(reinterpret_cast<const unsigned long long*>(rows) + i);
  const int lane = threadIdx.x & 31, width = n1 - n0;
  const unsigned short *xs = static_cast<const unsigned short*>(a.x), *ws = static_cast<const unsigned short*>(a.w);
  const unsigned short *bs = static_cast<const unsigned short*>(a.b), *vs = static_cast<const unsigned short*>(a.v);
  unsigned short* out = static_cast<unsigned short*>(a.out);
  const int count = max(t1 - t0, 0) * max(width, 0);
  int seen_t = -1;        // the row that was looked at last,
  bool nan_row = false;   // and whether its x holds a NaN: then so does every element
  for (int base = 0; base < count; base += 32) {
    const int e = base + lane, my_t = t0 + e / width, my_n = n0 + e % width;
    bool odd = false;
    if (e < count) odd = !finite(from16(__ldcg(out + my_t * a.out_m + my_n * a.out_n), a.bf16));
    for (unsigned who = __ballot_sync(0xffffffffu, odd); who != 0; who &= who - 1) {
      const int l = __ffs(who) - 1;
      const int t = __shfl_sync(0xffffffffu, my_t, l), n = __shfl_sync(0xffffffffu, my_n, l);
      const long long id = a.is64 ? static_cast<const long long*>(a.ids)[t] : static_cast<long long>(static_cast<const int*>(a.ids)[t]);
      const int tile = t / a.tile_rows;
      const int* list = a.list + static_cast<long long>(tile) * a.list_stride;
      const int listed = __ldcg(list);
      int place = 0;  // of the row's adapter in the list, counted from 1
      bool others = false;
      for (int i = lane; i < listed; i += 32) {
        if (__ldcg(list + 1 + i) == id) place = i + 1;
        else others = true;
      }
      place = static_cast<int>(__reduce_max_sync(0xffffffffu, static_cast<unsigned>(place)));
      if (!__any_sync(0xffffffffu, others)) continue;
      const unsigned short* x = xs + t * a.x_stride;
      if (t != seen_t) {
        bool nan = false;
        for (int k = lane; k < a.k; k += 32) nan = nan || isnan(from16(x[k], a.bf16));
        nan_row = __any_sync(0xffffffffu, nan);
        seen_t = t;
      }
      if (nan_row) continue;
      const unsigned short* w = ws + n * a.w_n;
      float s = 0.0f;
      if (place > 0) {
        const unsigned short* v = vs + ((static_cast<long long>(tile) * (a.list_stride - 1) + place - 1) * a.tile_rows + t % a.tile_rows) * a.v_row;
        const unsigned short* b = bs + id * a.b_adapter + n * a.b_row;
        for (int r = lane; r < a.rank; r += 32) {
          const int at = 2 * (r & ~(a.v_width - 1)) + (r & (a.v_width - 1));
          s = fmaf(from16(__ldcg(v + at), a.bf16) + from16(__ldcg(v + at + a.v_width), a.bf16), from16(b[r], a.bf16), s);
        }
        if (__any_sync(0xffffffffu, isnan(s))) continue;
      }
      if (a.w_k == 1) {  // rows of x and columns of w start on 16-byte boundaries, k is a multiple of 8
        for (int k = lane * 8; k < a.k; k += 256) {
          const uint4 xq = *reinterpret_cast<const uint4*>(x + k), wq = *reinterpret_cast<const uint4*>(w + k);
          const unsigned xu[4] = {xq.x, xq.y, xq.z, xq.w}, wu[4] = {wq.x, wq.y, wq.z, wq.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s = fmaf(from16(xu[j] & 0xffffu, a.bf16), from16(wu[j] & 0xffffu, a.bf16), s);
            s = fmaf(from16(xu[j] >> 16, a.bf16), from16(wu[j] >> 16, a.bf16), s);
          }
        }
      } else {
        for (int k = lane; k < a.k; k += 32) s = fmaf(from16(x[k], a.bf16), from16(w[k * a.w_k], a.bf16), s);
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if (a.bias != nullptr) {
        const long long i = n * a.bias_stride;
        s += a.bias_dtype == TB_DTYPE_F32 ? static_cast<const float*>(a.bias)[i]
                                          : from16(static_cast<const unsigned short*>(a.bias)[i], a.bias_dtype == TB_DTYPE_BF16);
      }
      if (lane == 0)
        out[t * a.out_m + n * a.out_n] = a.bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(s)) : __half_as_ushort(__float2half_rn(s));
    }
  }
  __syncwarp();
}

}  // namespace low_rank
}  // namespace tb
