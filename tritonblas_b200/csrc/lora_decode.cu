// The shared projection of a decode batch (up to 64 rows) with its rows' low-rank updates: the second launch of lora.cu.
//     out[t, n] = sum_k x[t, k] W[k, n] + bias[n] + sum over the listed adapters a of sum_r v_a[t, r] B_a[n, r]
// v_a is what the first launch wrote: the rows' scaled rank-sized products in two 16-bit halves, zero in rows of other adapters.
//
// Bound by reading W and the used B once. W's rows (output features) stand on the 128-row side of the tensor-core tile and the
// tokens on its narrow side, a stage of the ring is 16 KB of weights and the tokens' share. Tiles that fill whole
// rounds of the SMs are worked on one per CTA; the K range of the others is dealt evenly over all CTAs, so every CTA reads
// the same number of bytes, and their parts meet in the workspace: each warp of the epilogue counts itself in for its quarter
// of the tile, and the one that comes last adds the parts up in a fixed order. Nobody waits for another CTA.
// The parts come first, the ones that take a dealt tile's update last among them, then the whole tiles: the sums over parts are
// hidden behind the whole tiles where there are any.
//
// Measured back to back: 1 row of 4096 x 4096, rank 16: 13.2 us (19.5 with the general GEMM and the same update); 48 rows of 8192
// x 28672, 30 adapters of rank 16: 91 us, 5.6 TB/s (101); 1 row of 8192 x 28672: 75 us, 0.96 of the copy rate; n-contiguous
// weights within 4 %. A unit of its own for the updates instead of the last parts, and parts written only once the first launch
// is through, took 15.0 us for 1 row of 4096 x 4096 and 37 instead of 33 for 64 rows of 4096 x 8192 with 64 adapters.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common_host.h"
#include "low_rank.cuh"
#include "ptx.cuh"
#include "token_ops.cuh"

namespace tb {

namespace {

constexpr int kThreads = 7 * 32;  // four epilogue warps, weight loader, MMA issuer, token loader
constexpr int kWarpWeights = 4, kWarpMma = 5, kWarpTokens = 6;
constexpr int kMaxStages = 10;    // 160 KB of weights ahead
constexpr int kRowBytes = 128;
constexpr int kStageK = 64;       // K of a stage: one 128-byte row of 16-bit elements
constexpr int kTile = 128;        // features of a tile
constexpr int kMaxTokens = 64;
constexpr int kPieceStages = 4;   // of an update, at least
constexpr uint32_t kWeightBytes = kTile * kRowBytes;  // of a stage

struct DecodeParams {
  int tokens, n;
  int cols;             // MMA columns, and rows of a v block: tokens rounded up to 16
  int stages, stage_bytes;
  int acc_stride, tmem_cols;
  int nkb;              // stages per tile
  int w_mn;             // 1: W is stored with its output features contiguous
  int full_tiles, dealt_tiles, deal_ctas;
  // low-rank update
  const int* list;      // number of adapters, then their indices
  int max_slots, pack, kblocks, rank;
  const LowRankRows* rows;
  int pieces;           // a dealt tile's update is cut into at most this many
  float* parts;         // [2 * grid][tokens][kTile], and [grid] more when there are pieces
  unsigned* arrived;    // [dealt_tiles][4], cleared by the first launch
  const void* bias;
  long long bias_stride;
  int bias_dtype;
  void* out;
  long long out_m, out_n;
  int out_vec;          // four consecutive outputs stand on an 8-byte boundary
  uint32_t idesc;
  int* status;
  unsigned long long timeout_ns;
};

// The dealt tiles' stages [0, dealt_tiles * nkb) in equal runs, one for each of the first deal_ctas CTAs.
struct Deal {
  int base, rem, ctas;
  __device__ Deal(const DecodeParams& p) : ctas(p.deal_ctas) {
    const int total = p.dealt_tiles * p.nkb;
    base = total / max(ctas, 1);
    rem = total - base * ctas;
  }
  __device__ int begin(int cta) const { return min(cta, ctas) * base + min(cta, rem); }
  __device__ int cta_of(int stage) const {
    const int wide = rem * (base + 1);
    return stage < wide ? stage / (base + 1) : rem + (stage - wide) / max(base, 1);
  }
};

// What a CTA works on, in order; every role walks the same sequence. Its run of dealt stages is at most one tile long, so it has
// at most two parts: the end of a tile's K range, or a piece of it, and the beginning of the next one's. The beginning comes
// first: the part that holds a tile's last stage also takes the tile's update, which needs the first launch to be through. Of a
// long update it takes the first piece, the others go to one CTA each, from the last one down.
struct Unit {
  // 0 none, 1 part of a dealt tile, 2 whole tile with its update, 3 last part of a dealt tile with its update or the first piece of
  // it, 4 another piece
  int kind;
  int tile, kb0, kb1;
  int slot;       // of the part in the workspace
  int piece;
};
template <bool PIECES>
struct Units {
  const DecodeParams& p;
  int at, split, end, first_tile, next_full, turn;
  __device__ Units(const DecodeParams& p_, const Deal& d) : p(p_), next_full(blockIdx.x), turn(0) {
    at = d.begin(blockIdx.x);
    end = d.begin(blockIdx.x + 1);
    first_tile = at / p.nkb;
    split = min(end, (first_tile + 1) * p.nkb);
  }
  __device__ Unit next() {
    const int tile = p.full_tiles + first_tile, k0 = first_tile * p.nkb, slot = 2 * static_cast<int>(blockIdx.x);
    if (turn == 0) {
      turn = 1;
      if (split < end) return Unit{1, tile + 1, 0, end - split, slot + 1, 0};
    }
    if (turn == 1) {
      turn = 2;
      if (at < split) return Unit{split - k0 == p.nkb ? 3 : 1, tile, at - k0, split - k0, slot, 0};
    }
    if (PIECES && turn == 2) {
      turn = 3;
      const int j = static_cast<int>(gridDim.x - 1 - blockIdx.x);
      if (j < (p.pieces - 1) * p.dealt_tiles)
        return Unit{4, p.full_tiles + j % p.dealt_tiles, 0, 0, static_cast<int>(2 * gridDim.x + blockIdx.x), 1 + j / p.dealt_tiles};
    }
    if (next_full < p.full_tiles) {
      const Unit u = {2, next_full, 0, p.nkb, 0, 0};
      next_full += gridDim.x;
      return u;
    }
    return Unit{0, 0, 0, 0, 0, 0};
  }
};

__device__ __forceinline__ void tma_load_2d_hint(void* smem_dst, const CUtensorMap* tmap, uint64_t* bar, int x, int y, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(
          smem_u32(smem_dst)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "l"(policy)
      : "memory");
}
__device__ __forceinline__ unsigned add_acq_rel(unsigned* p, unsigned v) {
  unsigned old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}
__device__ __forceinline__ float bias_at(const void* bias, long long i, int dtype) {
  if (dtype == TB_DTYPE_F32) return static_cast<const float*>(bias)[i];
  if (dtype == TB_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[i]);
  return __half2float(static_cast<const __half*>(bias)[i]);
}
// PIECES: with dealt updates (the form without them is half a microsecond shorter). A quarter of an SM's registers belongs to each of
// its four warp schedulers: 136 for the two of these seven warps that meet there are what leaves room for two of the first launch's
// at 120. With 144 and 128 the kernels run one after the other (1 row of 4096 x 4096: 14.9 us, not 12.9 at the time).
template <typename T, bool PIECES>
__global__ void __maxnreg__(136)
lora_decode_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                   const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_v, const DecodeParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  __shared__ uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], tmem_full[2], tmem_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &abort_word;
  const WaitCtx wctx{abort_flag, p.status, p.timeout_ns};
  if (threadIdx.x == 0) {
    abort_word = 0;
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full_bar[s], 2);  // weight loader and token loader
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], 4);
    }
    mbar_fence_init();
    prefetch_tmap(&tmap_w);
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
  // The first launch waits for everything before it ahead of letting this one start, so x and W may be read at once; what it
  // writes itself (list, v, cleared counters) is waited for by each role before its first use.
  griddep_launch_dependents();
  const Deal deal(p);
  Units<PIECES> units(p, deal);
  // The adapter list, at most 64 entries for as many rows; every lane of the warp calls it. Whole tiles ask for it a few stages ahead
  // of their update; the part of a dealt tile only when all of its weights are on their way, since asking means waiting for the
  // first launch.
  int count = -1, entries = 0, more_entries = 0;
  auto read_list = [&]() {
    griddep_wait();
    count = __ldcg(p.list);
    entries = lane < p.max_slots ? __ldcg(p.list + 1 + lane) : 0;
    more_entries = 32 + lane < p.max_slots ? __ldcg(p.list + 33 + lane) : 0;
  };
  // Adapters per piece of a dealt tile's update: whole stages, at least four of them; the list's length says how many pieces there are.
  auto piece_length = [&]() {
    if (!PIECES) return kMaxTokens;
    const int groups = (count + p.pack - 1) / p.pack;
    return max((groups + p.pieces - 1) / p.pieces, (kPieceStages + p.kblocks - 1) / p.kblocks) * p.pack;
  };
  // The adapters [x, y) of the list that a unit's update takes.
  auto update_range = [&](const Unit& u) {
    if (!PIECES || u.kind == 2) return make_int2(0, count);
    const int length = piece_length();
    return make_int2(min(u.piece * length, count), min((u.piece + 1) * length, count));
  };
  // An update's stage: the rows of B of `pack` adapters (`width` ranks of each) fill the weights' part, both halves of v for them the
  // tokens' part, which has room for two columns' worth for that. (A stage of half as many ranks, within the room that the product
  // itself needs, halves the bytes of B in flight, and with them the rate: 64 rows of 4096 x 8192, 64 adapters of rank 128: 152 us.)
  const int width = kStageK / p.pack;
  const int part_w = kWeightBytes / p.pack, part_v = 2 * p.cols * kRowBytes / p.pack;  // bytes of one adapter's share of a stage

  if (warp == kWarpWeights) {
    // -------------------------------------------------------------- weights and lora_b
    const uint64_t policy = evict_first_policy();
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (Unit u = units.next(); u.kind != 0 && ok; u = units.next()) {
      const int ask = max(u.kb0, u.kb1 - 6);
      for (int kb = u.kb0; kb < u.kb1; ++kb) {
        if (u.kind == 2 && kb == ask && count < 0) read_list();
        ok = wait_warp(&empty_bar[s], ph ^ 1, wctx, TB_DEV_TIMEOUT_SMEM_EMPTY);
        if (!ok) break;
        if (elect_one()) {
          uint8_t* dst = ring + static_cast<size_t>(s) * p.stage_bytes;
          mbar_arrive_expect_tx(&full_bar[s], kWeightBytes);
          if (p.w_mn) {  // 64 features x 64 K rows per copy, one 128-byte row per K
            tma_load_2d_hint(dst, &tmap_w, &full_bar[s], u.tile * kTile, kb * kStageK, policy);
            tma_load_2d_hint(dst + kWeightBytes / 2, &tmap_w, &full_bar[s], u.tile * kTile + 64, kb * kStageK, policy);
          } else {
            tma_load_2d_hint(dst, &tmap_w, &full_bar[s], kb * kStageK, u.tile * kTile, policy);
          }
        }
        __syncwarp();
        if (++s == p.stages) {
          s = 0;
          ph ^= 1;
        }
      }
      if (!ok || u.kind == 1) continue;
      if (count < 0) read_list();
      const int2 range = update_range(u);
      for (int i = range.x; i < range.y && ok; i += p.pack) {
        const int filled = min(p.pack, count - i);
        int adapter[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) adapter[j] = __shfl_sync(0xffffffffu, i < 32 ? entries : more_entries, (i + j) & 31);
        for (int kb = 0; kb < p.kblocks; ++kb) {
          ok = wait_warp(&empty_bar[s], ph ^ 1, wctx, TB_DEV_TIMEOUT_SMEM_EMPTY);
          if (!ok) break;
          if (elect_one()) {
            uint8_t* dst = ring + static_cast<size_t>(s) * p.stage_bytes;
            mbar_arrive_expect_tx(&full_bar[s], static_cast<uint32_t>(filled * part_w));
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (j < filled) tma_load_3d(dst + j * part_w, &tmap_b, &full_bar[s], kb * kStageK, u.tile * kTile, adapter[j]);
          }
          __syncwarp();
          if (++s == p.stages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
    }
  } else if (warp == kWarpTokens) {
    // -------------------------------------------------------------- x and v
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (Unit u = units.next(); u.kind != 0 && ok; u = units.next()) {
      const int ask = max(u.kb0, u.kb1 - 6);
      for (int kb = u.kb0; kb < u.kb1; ++kb) {
        if (u.kind == 2 && kb == ask && count < 0) read_list();
        ok = wait_warp(&empty_bar[s], ph ^ 1, wctx, TB_DEV_TIMEOUT_SMEM_EMPTY);
        if (!ok) break;
        if (elect_one()) {
          // rows behind the last token keep an earlier stage's values: columns of the product that nobody reads
          uint8_t* dst = ring + static_cast<size_t>(s) * p.stage_bytes + kWeightBytes;
          mbar_arrive_expect_tx(&full_bar[s], static_cast<uint32_t>(p.tokens * kRowBytes));
          tma_load_2d(dst, &tmap_x, &full_bar[s], kb * kStageK, 0);
        }
        __syncwarp();
        if (++s == p.stages) {
          s = 0;
          ph ^= 1;
        }
      }
      if (!ok || u.kind == 1) continue;
      if (count < 0) read_list();
      const int2 range = update_range(u);
      for (int i = range.x; i < range.y && ok; i += p.pack) {
        const int filled = min(p.pack, count - i);
        for (int kb = 0; kb < p.kblocks; ++kb) {
          ok = wait_warp(&empty_bar[s], ph ^ 1, wctx, TB_DEV_TIMEOUT_SMEM_EMPTY);
          if (!ok) break;
          if (elect_one()) {
            uint8_t* dst = ring + static_cast<size_t>(s) * p.stage_bytes + kWeightBytes;
            mbar_arrive_expect_tx(&full_bar[s], static_cast<uint32_t>(filled * part_v));
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (j < filled) tma_load_2d(dst + j * part_v, &tmap_v, &full_bar[s], kb * 2 * width, (i + j) * p.cols);
            // rows of 2 * width elements, or 128 bytes of them at a time
            if (p.pack == 1) tma_load_2d(dst + part_v / 2, &tmap_v, &full_bar[s], (2 * kb + 1) * width, i * p.cols);
          }
          __syncwarp();
          if (++s == p.stages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
    }
  } else if (warp == kWarpMma) {
    // -------------------------------------------------------------- MMA issuer
    int s = 0, acc = 0;
    uint32_t ph = 0, acc_parity = 0;
    bool ok = true;
    const uint32_t ring_addr = smem_u32(ring);
    // W: K-contiguous rows of 128 bytes, or 64-feature columns of 64 K rows, 8 KB apart; a step of 16 K is 32 bytes or 16 rows on
    const uint64_t w0 = make_smem_desc(ring_addr, p.w_mn ? kWeightBytes / 2 : 16u, 1024);
    const uint64_t x0 = make_smem_desc(ring_addr + kWeightBytes, 16, 1024);
    const uint64_t w_step = p.w_mn ? 16 * kRowBytes >> 4 : 2;
    const uint32_t idesc = p.idesc | (p.w_mn ? 1u << 15 : 0u);
    // an update's operands: rows of 128, 64 or 32 bytes of B, twice that of v but no more than 128
    const uint64_t xa0 = make_smem_desc(ring_addr, 16, 1024u / p.pack, p.pack == 1 ? 2u : (p.pack == 2 ? 4u : 6u));
    const uint64_t xb0 = make_smem_desc(ring_addr + kWeightBytes, 16, p.pack == 4 ? 512u : 1024u, p.pack == 4 ? 4u : 2u);
    const uint64_t v_low = static_cast<uint64_t>(p.pack == 1 ? part_v / 2 : width * 2) >> 4;
    for (Unit u = units.next(); u.kind != 0 && ok; u = units.next()) {
      if (PIECES && u.kind == 4) {
        if (count < 0) read_list();
        const int2 range = update_range(u);
        if (range.x >= range.y) continue;  // a shorter list: the other roles know it too
      }
      const uint32_t d = tmem_base + static_cast<uint32_t>(acc * p.acc_stride);
      ok = wait_warp(&tmem_empty[acc], ((acc_parity >> acc) & 1u) ^ 1u, wctx, TB_DEV_TIMEOUT_TMEM_EMPTY);
      if (!ok) break;
      tc_fence_after();
      const int ask = max(u.kb0, u.kb1 - 6);
      for (int kb = u.kb0; kb < u.kb1; ++kb) {
        if (u.kind == 2 && kb == ask && count < 0) read_list();
        ok = wait_warp(&full_bar[s], ph, wctx, TB_DEV_TIMEOUT_SMEM_FULL);
        if (!ok) break;
        if (elect_one()) {
          const uint64_t soff = static_cast<uint64_t>((s * p.stage_bytes) >> 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) umma<0, 1>(d, w0 + soff + k * w_step, x0 + soff + 2 * k, idesc, (k > 0 || kb > u.kb0) ? 1u : 0u);
          umma_commit(&empty_bar[s]);
          if (u.kind == 1 && kb + 1 == u.kb1) umma_commit(&tmem_full[acc]);
        }
        __syncwarp();
        if (++s == p.stages) {
          s = 0;
          ph ^= 1;
        }
      }
      if (!ok) break;
      if (u.kind != 1) {
        if (count < 0) read_list();
        const int2 range = update_range(u);
        for (int i = range.x, kb = 0; i < range.y;) {
          ok = wait_warp(&full_bar[s], ph, wctx, TB_DEV_TIMEOUT_SMEM_FULL);
          if (!ok) break;
          if (elect_one()) {
            const uint64_t soff = static_cast<uint64_t>((s * p.stage_bytes) >> 4);
            const int filled = min(p.pack, count - i);
            const int steps = min(4 / p.pack, (p.rank - kb * kStageK + 15) >> 4);  // columns behind the rank are zeros
            for (int j = 0; j < filled; ++j)
              for (int k = 0; k < 2 * steps; ++k)  // high and low half in turn
                umma<0, 1>(d, xa0 + soff + ((j * part_w) >> 4) + (k & ~1), xb0 + soff + ((j * part_v) >> 4) + (k & 1) * v_low + (k & ~1), p.idesc,
                           (PIECES && u.kind == 4 && i == range.x && kb == 0 && j == 0 && k == 0) ? 0u : 1u);
            umma_commit(&empty_bar[s]);
          }
          __syncwarp();
          if (++kb == p.kblocks) {
            kb = 0;
            i += p.pack;
          }
          if (++s == p.stages) {
            s = 0;
            ph ^= 1;
          }
        }
        if (!ok) break;
        if (elect_one()) umma_commit(&tmem_full[acc]);
        __syncwarp();
      }
      acc_parity ^= 1u << acc;
      acc ^= 1;
    }
  } else {
    // -------------------------------------------------------------- epilogue (warps 0-3, one per TMEM lane quarter)
    int acc = 0;
    uint32_t parity = 0;
    bool ok = true;
    T* out = static_cast<T*>(p.out);
    for (Unit u = units.next(); u.kind != 0 && ok; u = units.next()) {
      const int n = u.tile * kTile + warp * 32 + lane;  // this lane's feature
      const bool mine = n < p.n;
      const float bias = u.kind == 2 && mine && p.bias != nullptr ? bias_at(p.bias, n * p.bias_stride, p.bias_dtype) : 0.0f;
      if (PIECES && u.kind == 4) {
        if (count < 0) read_list();
        const int2 range = update_range(u);
        if (range.x >= range.y) continue;
      }
      float* part = p.parts + static_cast<size_t>(u.slot) * p.tokens * kTile + warp * 32 + lane;
      ok = __all_sync(0xffffffffu, mbar_wait(&tmem_full[acc], (parity >> acc) & 1u, wctx, TB_DEV_TIMEOUT_TMEM_FULL));
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(warp * 32) << 16) + static_cast<uint32_t>(acc * p.acc_stride);
      float zero = 0.0f;  // stays so as long as every sum is finite
      for (int c0 = 0; c0 < p.tokens; c0 += 32) {
        uint32_t r[32];
        tmem_ld_32x32(t_row + c0, r);
        tmem_ld_wait(r);
        if (c0 + 32 >= p.tokens) {  // the last columns sit in registers
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tmem_empty[acc]);
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const int t = c0 + j;
          if (t < p.tokens) {
            const float v = __uint_as_float(r[j]);
            if (u.kind != 2) __stcg(part + static_cast<size_t>(t) * kTile, v);
            else if (mine) out[t * p.out_m + n * p.out_n] = cast16<T>(v + bias);
            zero = fmaf(v, 0.0f, zero);
          }
        }
      }
      parity ^= 1u << acc;
      acc ^= 1;
      const int n_first = u.tile * kTile + warp * 32, n_last = min(n_first + 32, p.n);
      if (u.kind == 2) {
        if (__any_sync(0xffffffffu, !(zero == 0.0f))) low_rank::redo(p.rows, 0, p.tokens, n_first, n_last);
        continue;
      }
      // count this warp's quarter in; the last of its tile's parts adds them up
      const int dealt = u.tile - p.full_tiles;
      const int c_first = deal.cta_of(dealt * p.nkb), c_last = deal.cta_of((dealt + 1) * p.nkb - 1);
      griddep_wait();  // the counters are clear
      int extra = 0;  // pieces behind the first one
      if (PIECES) {
        if (count < 0) read_list();
        const int length = piece_length();
        extra = max((count + length - 1) / length, 1) - 1;
      }
      __syncwarp();
      unsigned old = 0;
      if (lane == 0) old = add_acq_rel(p.arrived + dealt * 4 + warp, 1u);
      old = __shfl_sync(0xffffffffu, old, 0);
      if (old != static_cast<unsigned>(c_last - c_first + extra)) continue;
      __syncwarp();
      // Four features per lane, four tokens per load instruction; four of those and four parts at a time, or two and eight where
      // there are no more tokens: sixteen 16-byte loads are in flight before the first sum, since each round is a round trip to L2.
      const int n4 = u.tile * kTile + warp * 32 + (lane & 7) * 4;
      const float* lane_parts = p.parts + warp * 32 + (lane & 7) * 4;
      const size_t slot_stride = static_cast<size_t>(p.tokens) * kTile;
      // only the first of the tile's CTAs can have begun inside an earlier tile
      const size_t first_slot = 2 * c_first + dealt - deal.begin(c_first) / p.nkb;
      float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (p.bias != nullptr && n4 + i < p.n) b[i] = bias_at(p.bias, (n4 + i) * p.bias_stride, p.bias_dtype);
      zero = 0.0f;
      auto add_up = [&](auto parts_at_once, auto tokens_at_once) {
        constexpr int kQ = decltype(parts_at_once)::value, kT = decltype(tokens_at_once)::value;
        for (int t0 = lane >> 3; t0 < p.tokens; t0 += 4 * kT) {
          float4 sum[kT];
#pragma unroll
          for (int j = 0; j < kT; ++j) sum[j] = make_float4(b[0], b[1], b[2], b[3]);
          auto add = [&](int n, auto slot_of) {
            for (int q0 = 0; q0 < n; q0 += kQ) {
              float4 v[kQ][kT];
#pragma unroll
              for (int q = 0; q < kQ; ++q) {
                const float* src = lane_parts + slot_of(q0 + q) * slot_stride;
#pragma unroll
                for (int j = 0; j < kT; ++j)
                  v[q][j] = q0 + q < n && t0 + 4 * j < p.tokens
                                ? __ldcg(reinterpret_cast<const float4*>(src + static_cast<size_t>(t0 + 4 * j) * kTile))
                                : make_float4(0.f, 0.f, 0.f, 0.f);
              }
#pragma unroll
              for (int q = 0; q < kQ; ++q)
#pragma unroll
                for (int j = 0; j < kT; ++j) {
                  sum[j].x += v[q][j].x;
                  sum[j].y += v[q][j].y;
                  sum[j].z += v[q][j].z;
                  sum[j].w += v[q][j].w;
                }
            }
          };
          add(c_last - c_first + 1, [&](int q) { return q == 0 ? first_slot : 2 * static_cast<size_t>(c_first + q); });
          if (PIECES && extra > 0) add(extra, [&](int q) { return static_cast<size_t>(3 * gridDim.x - 1 - (q * p.dealt_tiles + dealt)); });
#pragma unroll
          for (int j = 0; j < kT; ++j) {
            const int t = t0 + 4 * j;
            if (t >= p.tokens) break;
            zero = fmaf(sum[j].x, 0.0f, fmaf(sum[j].y, 0.0f, fmaf(sum[j].z, 0.0f, fmaf(sum[j].w, 0.0f, zero))));
            T* o = out + t * p.out_m + n4 * p.out_n;
            if (p.out_vec && n4 + 3 < p.n) {
              alignas(8) const T quad[4] = {cast16<T>(sum[j].x), cast16<T>(sum[j].y), cast16<T>(sum[j].z), cast16<T>(sum[j].w)};
              *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(quad);
              continue;
            }
            if (n4 < p.n) o[0] = cast16<T>(sum[j].x);
            if (n4 + 1 < p.n) o[p.out_n] = cast16<T>(sum[j].y);
            if (n4 + 2 < p.n) o[2 * p.out_n] = cast16<T>(sum[j].z);
            if (n4 + 3 < p.n) o[3 * p.out_n] = cast16<T>(sum[j].w);
          }
        }
      };
      if (p.tokens <= 8) add_up(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
      else add_up(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
      __syncwarp();
      if (__any_sync(0xffffffffu, !(zero == 0.0f))) low_rank::redo(p.rows, 0, p.tokens, n_first, n_last);
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

template <typename T, bool PIECES>
int decode_launch(const CUtensorMap& w, const CUtensorMap& x, const CUtensorMap& b, const CUtensorMap& v, const DecodeParams& p, int grid,
                  int smem_bytes, int device, cudaStream_t stream) {
  auto kernel = lora_decode_kernel<T, PIECES>;
  static SmemOptIn configured;
  const int rc = opt_in_smem(kernel, smem_bytes, device, configured, "cudaFuncSetAttribute(lora_decode)");
  if (rc != TB_OK) return rc;
  return launch_token_kernel(kernel, dim3(static_cast<unsigned>(grid)), kThreads, smem_bytes, 0, stream, "lora_decode_kernel launch", w, x, b, v, p);
}

}  // namespace

// Whole rounds of tiles go to one CTA each, the rest is dealt. (64-row tiles measured 1 us better up to eight tokens at 8192 x
// 28672 and 4-15 % worse everywhere else, so there are none.)
// A dealt tile has at most as many parts as make its reading and the sum over them about equally long: a stage takes a quarter of a
// microsecond, as does a part of up to 16 tokens in the sum, or two parts of up to 8.
// Its update, up to update_stages long, is cut into pieces of four stages or more as long as every CTA gets at most one of them, and
// where a quarter of the CTAs' number of tiles or fewer is dealt (64 rows of 1024 x 256, 64 adapters of rank 128: 69 -> 38 us; of
// 4096 x 8192, rank 16, with two pieces for each of 64 tiles: 35 -> 42, so not there).
LoraDecodeShape lora_decode_shape(int tokens, int n, int k, int update_stages, int grid) {
  LoraDecodeShape s;
  s.cols = (tokens + 15) / 16 * 16;
  s.grid = grid;
  const int tiles = (n + kTile - 1) / kTile;
  s.full_tiles = tiles / grid * grid;
  s.dealt_tiles = tiles - s.full_tiles;
  const int ratio = (k + kStageK - 1) / kStageK * (tokens <= 8 ? 2 : 1) / ((tokens + 15) / 16);
  int parts = 1;
  while ((parts + 1) * (parts + 1) <= ratio && parts < grid) ++parts;
  s.deal_ctas = s.dealt_tiles * parts < grid ? s.dealt_tiles * parts : grid;
  s.pieces = 1;
  if (s.dealt_tiles > 0) {
    const int by_grid = grid / s.dealt_tiles, by_stages = (update_stages - 1) / kPieceStages;
    if (by_grid >= 4) s.pieces += by_grid < by_stages ? by_grid : by_stages;
  }
  s.part_bytes = s.dealt_tiles > 0 ? 4ll * (s.pieces > 1 ? 3 : 2) * grid * tokens * kTile : 0;
  return s;
}

int lora_decode(const tb_lora_args& a, const LoraDecodeShape& s, const LowRank& lr, void* parts, void* arrived, int device,
                int smem_optin, int* status, cudaStream_t stream) {
  DecodeParams p = {};
  p.tokens = a.m;
  p.n = a.n;
  p.cols = s.cols;
  p.stage_bytes = static_cast<int>(kWeightBytes) + 2 * s.cols * kRowBytes;  // twice the tokens' part: both halves of an update's v
  // beside the ring: the barriers, the ring's alignment, and a block of the first launch, which runs at the same time
  p.stages = (smem_optin - 28 * 1024) / p.stage_bytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  p.acc_stride = s.cols <= 32 ? 32 : 64;
  p.tmem_cols = 2 * p.acc_stride;
  p.nkb = (a.k + kStageK - 1) / kStageK;
  p.full_tiles = s.full_tiles;
  p.dealt_tiles = s.dealt_tiles;
  p.deal_ctas = s.deal_ctas;
  p.pieces = s.pieces;
  p.list = lr.list;
  p.max_slots = lr.list_stride - 1;
  p.pack = lr.pack;
  p.kblocks = lr.kblocks;
  p.rank = a.rank;
  p.rows = lr.rows;
  p.parts = static_cast<float*>(parts);
  p.arrived = static_cast<unsigned*>(arrived);
  p.bias = a.bias;
  p.bias_stride = a.bias_stride;
  p.bias_dtype = a.bias_dtype;
  p.out = a.out;
  p.out_m = a.out_stride_m;
  p.out_n = a.out_stride_n;
  p.out_vec = a.out_stride_n == 1 && reinterpret_cast<uintptr_t>(a.out) % 8 == 0 && (a.m == 1 || a.out_stride_m % 4 == 0) ? 1 : 0;
  p.status = status;
  p.timeout_ns = a.wait_timeout_ms > 0 ? static_cast<unsigned long long>(a.wait_timeout_ms) * 1000000ull : 2000000000ull;
  const uint32_t fmt = a.dtype == TB_DTYPE_BF16 ? 1u : 0u;
  p.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(s.cols >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);

  CUtensorMap tw, tx, tb_, tv;
  p.w_mn = a.w_stride_k == 1 ? 0 : 1;
  int rc = p.w_mn ? encode_2d(&tw, a.dtype, a.w, a.n, a.k, static_cast<uint64_t>(a.w_stride_k) * 2, 64, kStageK, 1)
                  : encode_2d(&tw, a.dtype, a.w, a.k, a.n, static_cast<uint64_t>(a.n > 1 ? a.w_stride_n : a.k) * 2, kStageK, kTile, 1);
  if (rc != TB_OK) return rc;
  rc = encode_2d(&tx, a.dtype, a.x, a.k, a.m, static_cast<uint64_t>(a.m > 1 ? a.x_row_stride : a.k) * 2, kStageK, a.m, 1);
  if (rc != TB_OK) return rc;
  const uint32_t inner = static_cast<uint32_t>(kStageK / lr.pack);
  const uint64_t v_cols = 2ull * lr.kblocks * inner;  // both halves
  const uint64_t v_dims[2] = {v_cols, static_cast<uint64_t>(lr.v_rows)}, v_strides[1] = {v_cols * 2};
  const uint32_t v_box[2] = {lr.pack == 1 ? inner : 2 * inner, static_cast<uint32_t>(s.cols)};
  if ((rc = encode_nd(&tv, a.dtype, lr.v, 2, v_dims, v_strides, v_box)) != TB_OK) return rc;
  const uint64_t dims[3] = {static_cast<uint64_t>(lr.rank), static_cast<uint64_t>(lr.n), static_cast<uint64_t>(lr.num_adapters)};
  const uint64_t row = static_cast<uint64_t>(lr.b_row_stride) * 2;
  const uint64_t strides[2] = {row, lr.num_adapters > 1 ? static_cast<uint64_t>(lr.b_adapter_stride) * 2 : row * lr.n};
  const uint32_t box[3] = {inner, kTile, 1};
  if ((rc = encode_nd(&tb_, a.dtype, lr.b, 3, dims, strides, box)) != TB_OK) return rc;
  const int smem_bytes = p.stages * p.stage_bytes + 1024;
  auto launch = p.pieces > 1 ? (fmt ? decode_launch<__nv_bfloat16, true> : decode_launch<__half, true>)
                             : (fmt ? decode_launch<__nv_bfloat16, false> : decode_launch<__half, false>);
  return launch(tw, tx, tb_, tv, p, s.grid, smem_bytes, device, stream);
}

}  // namespace tb
