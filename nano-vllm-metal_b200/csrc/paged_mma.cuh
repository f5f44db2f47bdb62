// paged_mma.cuh -- tensor-core paged attention for decode, multi-token verify and
// chunked prefill (and dense attention viewed as one page per sequence).
//
// Replaces the reference's Metal kernels paged_attention_decode_split_kv
// (paged_attention.metal:276-408), paged_attention_kv (:6-128) and
// paged_attention_int8_decode_kv (:417-525), with the dispatch of
// paged_attention.cpp:413-642.  Same results, different decomposition:
//
//  * One CTA owns one (sequence b, kv head h, row block, key chunk).  The rows are
//    the g*L query rows that share kv head h (g = Hq/Hkv q heads x L tokens), packed
//    into 16-row m-tiles, so every K/V byte is read from HBM once per kv head instead
//    of once per q head as in the reference (grid = B*Hq there).
//  * Keys are processed in 16-token tiles.  A producer warp (on the n8 tile, each
//    consumer warp for the stages it consumes) streams each tile's K and V rows
//    ([16][D] contiguous inside one page) with plain tile-mode TMA tensor loads
//    (128-byte swizzle) into an NSTAGE-deep shared-memory ring guarded by mbarriers; page ids
//    come from the block table, holes are skipped.
//  * Consumer warps run the FA2-style online softmax on mma.sync m16n8k16 (fp32
//    accumulate): S = Q K^T from ldmatrix'd K, P kept in registers as the A operand
//    of O += P V with ldmatrix.trans'd V.  int8 pages are converted to f16 in
//    registers (exact), the per-token key scale multiplies S and the value scale
//    multiplies V, i.e. dequantisation happens in-kernel for every L.
//  * Split-K: long contexts are cut into chunks of `chunk_tiles` tiles handled by
//    separate CTAs; each writes (O, m, l) to the workspace and the last CTA of the
//    unit (atomic ticket) merges them with log-sum-exp weights and resets the ticket.
//  * kExt instances (paged_mma_window.cu) also take a sliding window with sinks: a row at
//    position pos sees key s only if s < sinks or s > pos - window.  The key tiles between
//    the sinks and the row block's windows are jumped over by renumbering: virtual tile v is
//    tile v below the sinks' last tile and tile v + skip past it, so chunks, rings and merges
//    run on virtual tiles unchanged.  They can leave every row's log-sum-exp.  Their keys are
//    counted in 32 bits.  On the n8 tile they can keep every score in the workspace and, where
//    units merge in a cluster or not at all, add the keys' weights to a buffer of the caller's
//    once the log-sum-exps are known.  A tile is named by one row of the pool seen as [P * Hkv *
//    page_size, D], worked out with the page ids, so that the warp that copies a tile between
//    two of its own spends few instructions on it.
//  * Every mbarrier wait is bounded (nvm::mbar_wait); on expiry the kernel records an
//    error code, each issuing warp drains what it issued, and the CTA returns.
#pragma once

#include <cooperative_groups.h>
#include <type_traits>

#include <cstdio>
#include <cstdlib>
#include <atomic>
#include <mutex>

#include "nvm_common.cuh"
#include "nvm_internal.h"

namespace nvm {
namespace {

constexpr int kMaxChunkTiles = 256;
// Split-K tickets live in a fixed region at the start of the workspace that partial
// results never use, so one zero-filled workspace can serve calls of any shape.
constexpr size_t kCounterBytes = kTicketRegionBytes;
constexpr int64_t kMaxUnits = (int64_t)(kCounterBytes / sizeof(int));

struct MmaParams {
  const void* q;
  void* out;
  const int32_t* block_table;
  const int32_t* context_lens;
  float* part_o;      // [units][n_chunks][rows_real][D]
  float2* part_ml;    // [units][n_chunks][rows_real]
  int* counters;      // [units]
  int* err;
  int q_dtype, out_dtype;
  int64_t B, Hq, Hkv, L, P, ps, mp, dense_ctx;
  int64_t g, M;       // q heads per kv head, rows per (b, h)
  int64_t n_rb, rows_real, ct, n_chunks;
  float scale_log2;   // softmax scale * log2(e)
  int causal;
  int cluster;        // the n_chunks CTAs of a unit are one cluster: merge over DSMEM
  int64_t window, sinks;  // kExt: window == 0 for none
  int out_vec;            // kExt: out is aligned for four elements at once
  int defer;              // kExt: leave the chunks' merge to the kernel over the kept scores
  int64_t nb;             // kExt: row blocks per q head (a block then never spans two), 0: over all g * L rows
  float* lse;             // kExt: log2 of every row's sum of 2^z ([B*Hq*L], +inf: no key), or null
  const void* k_scales;   // kExt: int8 pages' scales, copied by row
  const void* v_scales;
  float* scores;          // kExt, n8: keep every score ([units][n_chunks * ct * 16][rows, even]), or null
  float* mass;            // kExt, n8, with scores and no workspace merge: [b * mass_sb + h * mass_sh + key], key < mass_len
  int64_t mass_sb, mass_sh, mass_len;
};

template <typename KvT, int D, int NWM, int NWK, int NS_ = 0>
struct Cfg {
  static constexpr bool kI8 = std::is_same<KvT, int8_t>::value;
  using MmaT = typename std::conditional<kI8, __half, KvT>::type;
  static constexpr bool kSplitP = std::is_same<KvT, __nv_bfloat16>::value;
  // NWM == 0 selects the n8 tile: keys are the mma's M (16 per tile) and up to eight
  // query rows its N, so S^T = K Q^T and O^T = V^T P^T take half the mma.sync of the
  // 16-row tile when a kv head has at most eight query rows.
  static constexpr bool kN8 = NWM == 0;
  static constexpr int kCons = (kN8 ? 1 : NWM) * NWK;
  // The n8 tile has no producer warp: each consumer warp refills the ring
  // stages it consumes (stage s belongs to warp s % NWK), so a CTA is 64 threads and more
  // CTAs fit on an SM (the kernel is latency-bound there).
  static constexpr bool kSelfFeed = kN8;
  static constexpr int kThreads = (kCons + (kSelfFeed ? 0 : 1)) * 32;
  static constexpr int kRB = kN8 ? 8 : 16 * NWM;
  static constexpr int kTileBytes = 16 * D * (int)sizeof(KvT);
  // K scales at +0, V scales at +128 past the two tiles: TMA destinations are 128-byte aligned.
  static constexpr int kScaleBytes = kI8 ? 256 : 0;
  static constexpr int kStageBytes = ((2 * kTileBytes + kScaleBytes + 1023) / 1024) * 1024;
  static constexpr int kStages = NS_ > 0 ? NS_ : (kI8 ? 12 : 8);
  static constexpr int kBoxElems = 128 / (int)sizeof(KvT);  // 128-byte inner box (swizzle span)
  static constexpr int kBoxes = D / kBoxElems;
  static constexpr int kEpiBytes = NWK * kRB * D * 4 + 2 * NWK * kRB * 4;
  static constexpr int kRingBytes = kStages * kStageBytes;
  // cluster merge (n8 tile): this CTA's combined partial rows [kRB][D], their (m, l) and
  // the chunk weights [8][kRB] + sums [kRB], placed after the epilogue staging area
  static constexpr int kClusterOff = ((kEpiBytes + 15) / 16) * 16;
  static constexpr int kClusterBytes = kRB * D * 4 + kRB * 8 + 8 * kRB * 4 + kRB * 4;
  // only self-feeding CTAs (every warp is a consumer and reaches the cluster barriers)
  static constexpr bool kClusterFits = kN8 && kSelfFeed;
  static constexpr int kEpiAll = kClusterFits ? kClusterOff + kClusterBytes : kEpiBytes;
  static constexpr int kMainBytes = kRingBytes > kEpiAll ? kRingBytes : kEpiAll;
  static constexpr int kSmemBytes = 1024 + kMainBytes + kStages * 16 + kStages * 4 + kMaxChunkTiles * 4 + 16;
  static_assert(kStages % NWK == 0, "stage ring must be a multiple of the k-split");
  static_assert(D % 64 == 0, "head dim must be 64 or 128");
  static_assert(!kI8 || D == 128, "int8 path needs D == 128");
};

// 8x8 b16 matrix held in the mma accumulator layout (row lane/4, columns 2(lane%4), +1),
// transposed across the warp (PTX movmatrix)
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float ex2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// bf16 pair of the rounding residuals (a - hi.x, b - hi.y) of a packed bf16 pair.
__device__ __forceinline__ uint32_t pack_residual(float a, float b, uint32_t hi) {
  const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&hi);
  return pack2<__nv_bfloat16>(a - __low2float(h), b - __high2float(h));
}

// Address of 16-byte chunk `q` of token row `tok` inside a TMA tile written with
// 128-byte swizzle: boxes of 128 bytes x 16 rows, 2048 bytes each, chunk index XOR row.
__device__ __forceinline__ uint32_t swz(uint32_t tile, int tok, int q) {
  return tile + (uint32_t)((q >> 3) * 2048 + tok * 128 + (((q & 7) ^ (tok & 7)) << 4));
}

constexpr int64_t kExtLimit = int64_t(1) << 30;  // keys of a kExt call; larger windows and sinks count as this

// Untiled bulk copy of `bytes` (a multiple of 16, both addresses 16-byte aligned) into this CTA's
// shared memory, completing on an mbarrier.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <typename KvT, typename ScaleT, int D, int NWM, int NWK, int NS_, bool kExt>
__global__ void __launch_bounds__(Cfg<KvT, D, NWM, NWK, NS_>::kThreads)
    paged_mma_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ CUtensorMap tm_ks, const __grid_constant__ CUtensorMap tm_vs,
                     const MmaParams p) {
  using C = Cfg<KvT, D, NWM, NWK, NS_>;
  using MmaT = typename C::MmaT;
  using Tok = typename std::conditional<kExt, int, int64_t>::type;  // key positions
  constexpr int NS = C::kStages;
  constexpr int NKS = D / 16;  // k-steps of Q K^T
  constexpr int NDT = D / 8;   // n8 tiles of the output

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kMainBytes);
  uint64_t* empty = full + NS;
  int* stage_valid = reinterpret_cast<int*>(empty + NS);
  int* tile_pid = stage_valid + NS;
  int* s_flag = tile_pid + kMaxChunkTiles;

  if (kExt && p.lse != nullptr && p.scores == nullptr) pdl_trigger();  // the key scores' kernel follows
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // 32-bit index arithmetic (the plan bounds units, rows and tiles below 2^31): a 64-bit
  // division costs about a hundred instructions, and these sit in front of the first
  // page copies.
  const int64_t unit = blockIdx.x;
  const uint32_t u32 = blockIdx.x, nrb = (uint32_t)p.n_rb, hkv = (uint32_t)p.Hkv;
  const uint32_t bh32 = u32 / nrb;
  const int64_t rb = u32 - bh32 * nrb;
  const uint32_t b32 = bh32 / hkv;
  const int64_t h = bh32 - b32 * hkv, b = b32;
  // paged: 16-token tiles per page (page_size is a multiple of 16)
  const uint32_t tpp = (uint32_t)(p.ps >> 4);
  const int64_t c = blockIdx.y;

  const int64_t ctx = p.context_lens ? (int64_t)p.context_lens[b] : p.dense_ctx;
  const int64_t cap = p.mp * p.ps;
  const int64_t ctx_limit = ctx < cap ? ctx : cap;
  int64_t row0 = rb * C::kRB, row_end = p.M;
  if constexpr (kExt) {
    if (p.nb > 0) {
      const uint32_t head = (uint32_t)rb / (uint32_t)p.nb, j = (uint32_t)rb - head * (uint32_t)p.nb;
      row0 = (int64_t)head * p.L + (int64_t)j * C::kRB;
      row_end = ((int64_t)head + 1) * p.L;
    }
  }
  const int64_t rows_here = (row_end - row0) < C::kRB ? (row_end - row0) : C::kRB;
  const int64_t t_begin = c * p.ct;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], C::kN8 ? 1 : NWM);
    }
    fence_mbar_init();
  }
  // Consumers load their Q fragments while the producer reads the block table: one
  // round of independent vector loads (pairs of elements), dtype dispatch outside.
  constexpr int kWM = C::kN8 ? 1 : NWM;
  const int wm = warp % kWM, wk = warp / kWM;
  const int r = lane >> 2, cq = lane & 3;
  const int64_t q_row0 = (b * p.Hq + h * p.g) * p.L;  // flat row of (b, h, m = 0)
  // this thread's two softmax rows (unit-relative): m16 tile rows r, r + 8; n8 tile
  // columns 2 cq, 2 cq + 1.  The n8 tile's Q operand is row r (loaded as "row A").
  const int64_t mA = C::kN8 ? row0 + r : row0 + wm * 16 + r, mB = C::kN8 ? row_end : mA + 8;
  const bool vA = mA < row_end, vB = mB < row_end;
  const int64_t sA = C::kN8 ? row0 + 2 * cq : mA, sB = C::kN8 ? sA + 1 : mB;
  uint32_t qa[NKS][4];
  if (warp < C::kCons) {
    const int64_t offA = (q_row0 + mA) * D, offB = (q_row0 + mB) * D;
    auto load_q = [&](auto tag) {
      using QT = decltype(tag);
      float2 va[NKS][2], vb[NKS][2];
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        int d0, d1;  // first d of the low / high k pair of this thread in k-step ks
        if (C::kI8) {
          d0 = 32 * cq + 4 * ks;
          d1 = d0 + 2;
        } else {
          d0 = 16 * ks + 2 * cq;
          d1 = d0 + 8;
        }
        va[ks][0] = vA ? load_pair<QT>(p.q, offA + d0) : make_float2(0.f, 0.f);
        va[ks][1] = vA ? load_pair<QT>(p.q, offA + d1) : make_float2(0.f, 0.f);
        vb[ks][0] = vB ? load_pair<QT>(p.q, offB + d0) : make_float2(0.f, 0.f);
        vb[ks][1] = vB ? load_pair<QT>(p.q, offB + d1) : make_float2(0.f, 0.f);
      }
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        qa[ks][0] = pack2<MmaT>(va[ks][0].x, va[ks][0].y);
        qa[ks][1] = pack2<MmaT>(vb[ks][0].x, vb[ks][0].y);
        qa[ks][2] = pack2<MmaT>(va[ks][1].x, va[ks][1].y);
        qa[ks][3] = pack2<MmaT>(vb[ks][1].x, vb[ks][1].y);
      }
    };
    if (p.q_dtype == NVM_F32)
      load_q(float{});
    else if (p.q_dtype == NVM_F16)
      load_q(__half{});
    else
      load_q(__nv_bfloat16{});
  }
  // n8 tile, int8 pages: K enters the mma as int8 + 1152 (the byte-permute alone, exact in
  // f16), so every score carries 1152 * sum_d q[row][d] too; this lane's two rows'
  // corrections (rows 2cq, 2cq+1), from the f16 q values the mma multiplies.
  float kbias0 = 0.f, kbias1 = 0.f;
  if constexpr (C::kN8 && C::kI8) {
    float qs = 0.f;  // this lane's share of row r: d = 32 cq + 4 ks + {0..3}
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&qa[ks][0]));
      const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&qa[ks][2]));
      qs += (a.x + a.y) + (b.x + b.y);
    }
    qs += __shfl_xor_sync(0xffffffffu, qs, 1);
    qs += __shfl_xor_sync(0xffffffffu, qs, 2);  // row r's sum on all four lanes of row r
    kbias0 = 1152.f * __shfl_sync(0xffffffffu, qs, 4 * (2 * cq));
    kbias1 = 1152.f * __shfl_sync(0xffffffffu, qs, 4 * (2 * cq + 1));
  }
  // kExt: the row block's tiles, renumbered without the ones no row sees
  int x_tiles = 0, x_sink_tiles = 0, x_skip = 0;
  int x_first = 0, x_end = 0, x_sinks = 0;  // keys in [x_sinks, x_first) and from x_end on: seen by no row
  if constexpr (kExt) {
    const bool spans = rows_here >= p.L || (int64_t)((uint32_t)row0 % (uint32_t)p.L) + rows_here > p.L;
    int64_t end = ctx_limit;
    if (p.causal) {
      const int64_t lmax = spans ? p.L - 1 : (int64_t)((uint32_t)(row0 + rows_here - 1) % (uint32_t)p.L);
      const int64_t lim = lmax + ctx - p.L + 1;
      if (lim < end) end = lim;
    }
    x_end = ctx <= 0 || end < 0 ? 0 : (int)end;
    x_tiles = (x_end + 15) >> 4;
    x_sink_tiles = x_tiles;
    if (p.window > 0) {
      const int64_t lmin = spans ? 0 : (int64_t)((uint32_t)row0 % (uint32_t)p.L);
      const int64_t first = lmin + ctx - p.L - p.window + 1;  // no row's window reaches below this key
      x_first = first > 0 ? (int)first : 0;
      x_sinks = (int)(p.sinks < kExtLimit ? p.sinks : kExtLimit);
      const int st = (x_sinks + 15) >> 4;
      if ((x_first >> 4) > st && st < x_tiles) {
        x_sink_tiles = st;
        x_skip = (x_first >> 4) - st;
        x_tiles = x_tiles - x_skip > st ? x_tiles - x_skip : st;
      }
    }
  }
  auto tile_of = [&](int v) -> int { return v >= x_sink_tiles ? v + x_skip : v; };  // kExt
  if constexpr (kExt) {  // a chunk past the unit's keys ends here, before any barrier
    const int chunks = x_tiles > 0 ? (int)((uint32_t)(x_tiles + p.ct - 1) / (uint32_t)p.ct) : 1;
    if (c >= chunks && !(C::kClusterFits && p.cluster)) return;
  }
  const int t0 = (int)t_begin;
  if (warp == (C::kSelfFeed ? 0 : C::kCons) && !(kExt && p.block_table == nullptr)) {
    // The chunk's block-table entries, read together with (not after) the context
    // length: the row holds mp entries, so entries past the context are in bounds and
    // simply never used.  All loads are issued before any is consumed.
    int64_t n_tab = (cap + 15) / 16 - t_begin;
    if constexpr (kExt) n_tab = x_tiles - t0;
    if (n_tab > p.ct) n_tab = p.ct;
    constexpr int kPer = kMaxChunkTiles / 32;
    int64_t pv[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = lane + 32 * j;
      pv[j] = -1;
      if (i < n_tab) {
        const uint32_t tile = kExt ? (uint32_t)tile_of(t0 + i) : (uint32_t)(t_begin + i);
        pv[j] = p.block_table ? (int64_t)__ldg(&p.block_table[b * p.mp + (tpp == 1 ? tile : tile / tpp)]) : b;
      }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = lane + 32 * j;
      if constexpr (kExt) {  // the tile's first row in the pool seen as rows
        const uint32_t tile = (uint32_t)tile_of(t0 + i), slot = tpp == 1 ? 0 : (tile % tpp) * 16;
        if (i < n_tab)
          tile_pid[i] = (pv[j] >= 0 && pv[j] < p.P) ? ((int)pv[j] * (int)hkv + (int)h) * (int)p.ps + (int)slot : -1;
      } else {
        if (i < n_tab) tile_pid[i] = (pv[j] >= 0 && pv[j] < p.P) ? (int)pv[j] : -1;
      }
    }
  }
  __syncthreads();

  int64_t need_keys = ctx_limit;
  if (p.causal) {
    const bool spans = rows_here >= p.L || (int64_t)((uint32_t)row0 % (uint32_t)p.L) + rows_here > p.L;
    const int64_t lmax = spans ? p.L - 1 : (int64_t)((uint32_t)(row0 + rows_here - 1) % (uint32_t)p.L);
    const int64_t lim = lmax + ctx - p.L + 1;
    if (lim < need_keys) need_keys = lim;
  }
  if (ctx <= 0 || need_keys < 0) need_keys = 0;
  const int64_t n_tiles = kExt ? x_tiles : (need_keys + 15) / 16;
  const int64_t n_chunks = n_tiles > 0 ? (int64_t)((uint32_t)(n_tiles + p.ct - 1) / (uint32_t)p.ct) : 1;
  // A chunk past this unit's keys has nothing to do; inside a cluster it still takes
  // part in the cluster barriers of the merge (with no tiles), so it does not return.
  if (c >= n_chunks && !(C::kClusterFits && p.cluster)) return;
  int64_t n_left = n_tiles - t_begin;
  if (n_left > p.ct) n_left = p.ct;
  const int n_my = n_left > 0 ? (int)n_left : 0;

  // One ring stage's loads (tile i of the chunk into stage i % NS), by one thread.
  auto issue_tile = [&](int i) {
    const int s = i % NS;
    if constexpr (kExt) {
      const int row = p.block_table == nullptr ? ((int)b * (int)hkv + (int)h) * (int)p.ps + tile_of(t0 + i) * 16 : tile_pid[i];
      stage_valid[s] = row >= 0 ? 1 : 0;
      if (row >= 0) {
        uint8_t* st = smem + s * C::kStageBytes;
        mbar_arrive_expect_tx(&full[s], 2 * C::kTileBytes + (C::kI8 ? 64 : 0));
#pragma unroll
        for (int hb = 0; hb < C::kBoxes; ++hb) {
          tma_load_2d(st + hb * 2048, &tm_k, hb * C::kBoxElems, row, &full[s]);
          tma_load_2d(st + C::kTileBytes + hb * 2048, &tm_v, hb * C::kBoxElems, row, &full[s]);
        }
        if (C::kI8) {
          bulk_load(st + 2 * C::kTileBytes, static_cast<const ScaleT*>(p.k_scales) + row, 32, &full[s]);
          bulk_load(st + 2 * C::kTileBytes + 128, static_cast<const ScaleT*>(p.v_scales) + row, 32, &full[s]);
        }
      } else {
        mbar_arrive(&full[s]);
      }
      return;
    }
    const int pid = tile_pid[i];
    stage_valid[s] = pid >= 0 ? 1 : 0;
    if (pid >= 0) {
      const uint32_t tile = (uint32_t)(t_begin + i);
      const int slot0 = p.block_table ? (tpp == 1 ? 0 : (int)((tile % tpp) * 16)) : (int)(((t_begin + i) * 16) % p.ps);
      uint8_t* st = smem + s * C::kStageBytes;
      mbar_arrive_expect_tx(&full[s], 2 * C::kTileBytes + (C::kI8 ? 64 : 0));
#pragma unroll
      for (int hb = 0; hb < C::kBoxes; ++hb) {
        tma_load_4d(st + hb * 2048, &tm_k, hb * C::kBoxElems, slot0, (int)h, pid, &full[s]);
        tma_load_4d(st + C::kTileBytes + hb * 2048, &tm_v, hb * C::kBoxElems, slot0, (int)h, pid, &full[s]);
      }
      if (C::kI8) {
        tma_load_3d(st + 2 * C::kTileBytes, &tm_ks, slot0, (int)h, pid, &full[s]);
        tma_load_3d(st + 2 * C::kTileBytes + 128, &tm_vs, slot0, (int)h, pid, &full[s]);
      }
    } else {
      mbar_arrive(&full[s]);
    }
  };

  // ------------------------------------------------------------------ producer
  if constexpr (!C::kSelfFeed) {
    if (warp == C::kCons) {
      if (lane == 0) {
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
        if (C::kI8) {
          prefetch_tmap(&tm_ks);
          prefetch_tmap(&tm_vs);
        }
        int issued = 0;
        for (int i = 0; i < n_my; ++i) {
          const int s = i % NS;
          if (i >= NS && !mbar_wait(&empty[s], ((i / NS) & 1) ^ 1)) {
            record_error(p.err, kDevErrEmptyWait);
            break;
          }
          issue_tile(i);
          issued = i + 1;
        }
        // Drain: the last use of every stage must have landed before the CTA can exit.
        for (int s = 0; s < NS && s < issued; ++s) {
          const int last = s + ((issued - 1 - s) / NS) * NS;
          if (!mbar_wait(&full[s], (last / NS) & 1)) record_error(p.err, kDevErrDrainWait);
        }
      }
      return;
    }
  }
  int last_issued = -1;  // self-feed: the highest tile this warp has issued (lane 0)
  if constexpr (C::kSelfFeed) {
    // each consumer warp fills its own first stages
    if (lane == 0) {
      if (warp == 0) {
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
        prefetch_tmap(&tm_ks);
        prefetch_tmap(&tm_vs);
      }
      for (int i = warp; i < n_my && i < NS; i += NWK) {
        issue_tile(i);
        last_issued = i;
      }
    }
    __syncwarp();
  }

  // ------------------------------------------------------------------ consumers

  // Inclusive last visible key of each row (rows past M never mask anything).
  const Tok BIG = kExt ? (Tok)kExtLimit : (Tok)(INT64_MAX / 4);
  Tok limA = BIG, limB = BIG;
  if (p.causal) {
    if (sA < row_end) limA = (Tok)((int64_t)((uint32_t)sA % (uint32_t)p.L) + ctx - p.L);
    if (sB < row_end) limB = (Tok)((int64_t)((uint32_t)sB % (uint32_t)p.L) + ctx - p.L);
    if constexpr (kExt) {  // a context length past the table's end may be as large as an int
      limA = limA < BIG ? limA : BIG;
      limB = limB < BIG ? limB : BIG;
    }
  }
  // kExt: the first key of each row's window (the sinks aside), and the last of these
  int loA = 0, loB = 0, lo_max = 0;
  if constexpr (kExt) {
    if (p.window > 0) {
      const int64_t base = ctx - p.L - p.window + 1;
      const int64_t a = sA < row_end ? (int64_t)((uint32_t)sA % (uint32_t)p.L) + base : 0;
      const int64_t b2 = sB < row_end ? (int64_t)((uint32_t)sB % (uint32_t)p.L) + base : 0;
      loA = a > 0 ? (int)a : 0;
      loB = b2 > 0 ? (int)b2 : 0;
      lo_max = loA > loB ? loA : loB;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_xor_sync(0xffffffffu, lo_max, o);
        lo_max = x > lo_max ? x : lo_max;
      }
    }
  }
  // Keys below `clean` are visible to every real row of this warp: no masking there.
  const Tok ctx_end = (Tok)ctx_limit;
  Tok clean = ctx_end;
  {
    Tok mn = limA < limB ? limA : limB;
    mn = mn + 1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const Tok x = __shfl_xor_sync(0xffffffffu, mn, o);
      mn = x < mn ? x : mn;
    }
    if (mn < clean) clean = mn;
  }

  float mrA = -INFINITY, mrB = -INFINITY, lA = 0.f, lB = 0.f;
  float o[NDT][4];
#pragma unroll
  for (int i = 0; i < NDT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  // kExt: V of the keys that no row of the block sees becomes zero in the stage (their weight is
  // zero, but 0 times a NaN or an infinity is not): 16-bit pages the row, int8 pages the scale.
  // Only tiles at an edge of a window or of the context come here.  The warps that share a
  // stage all write the same zeros, each before it reads.
  auto hide_unseen = [&](uint8_t* st, int tok0) {
    const int t = lane >> 1, tok = tok0 + t;
    if (tok >= x_end || (tok >= x_sinks && tok < x_first)) {
      if constexpr (C::kI8) {
        if ((lane & 1) == 0) reinterpret_cast<uint16_t*>(st + 2 * C::kTileBytes + 128)[t] = 0;
      } else {
#pragma unroll
        for (int hb = 0; hb < C::kBoxes; ++hb) {
          uint4* d = reinterpret_cast<uint4*>(st + C::kTileBytes + hb * 2048 + t * 128 + (lane & 1) * 64);
#pragma unroll
          for (int x = 0; x < 4; ++x) d[x] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
    }
    __syncwarp();
    // the stage's next TMA load must not be overtaken by these stores
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  };

  // kExt, n8: this lane's two rows' scores of keys r and r + 8 of the chunk's tile i
  float* score_row = nullptr;
  const int rows_pad = (int)((p.M + 1) & ~int64_t(1));
  if constexpr (kExt && C::kN8) {
    if (p.scores != nullptr && 2 * cq < rows_pad)
      score_row = p.scores + ((unit * p.n_chunks * p.ct + t_begin) * 16 + r) * rows_pad + 2 * cq;
  }
  auto keep_scores = [&](int i, float2 a, float2 b2) {
    float2* d = reinterpret_cast<float2*>(score_row + (int64_t)i * 16 * rows_pad);
    d[0] = a;
    d[4 * rows_pad] = b2;  // 8 keys on
  };

  bool timed_out = false;
  for (int i = wk; i < n_my; i += NWK) {
    const int s = i % NS;
    if (!mbar_wait(&full[s], (i / NS) & 1)) {
      record_error(p.err, kDevErrFullWait);
      timed_out = true;
      break;
    }
    if (stage_valid[s]) {
      if constexpr (C::kN8) {
      const Tok tok0 = kExt ? (Tok)(tile_of(t0 + i) * 16) : (Tok)((t_begin + i) * 16);
      const uint32_t kt = smem_u32(smem + s * C::kStageBytes);
      const uint32_t vt = kt + C::kTileBytes;
      // S^T = K Q^T (16 keys x 8 rows).  16-bit pages: the k-steps go round-robin into
      // four independent accumulator chains (the mma.sync result latency, not issue,
      // bounds a warp walking its tiles); int8 pages (issue-bound): two chains.
      constexpr int kQc = C::kI8 ? 2 : 4;
      float sacc[kQc][4];
#pragma unroll
      for (int q2 = 0; q2 < kQc; ++q2) sacc[q2][0] = sacc[q2][1] = sacc[q2][2] = sacc[q2][3] = 0.f;
      if constexpr (!C::kI8) {
        const int mi = lane >> 3;
        const int ktok = (mi >> 1) * 8 + (lane & 7);
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          uint32_t k0, k1, k2, k3;
          ldsm_x4(swz(kt, ktok, 2 * ks + (mi & 1)), k0, k1, k2, k3);
          const uint32_t a[4] = {k0, k2, k1, k3};
          mma16816<MmaT>(sacc[ks % kQc], a, qa[ks][0], qa[ks][2]);
        }
      } else {
        // keys r and r + 8, bytes [32 cq, 32 cq + 32) of each (the k dimension is
        // permuted identically in Q: k pair (2cq, 2cq+1) <-> d 32cq + 4ks + {0,1},
        // k pair (2cq+8, 2cq+9) <-> d 32cq + 4ks + {2,3})
        uint32_t kw[2][8];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int tok = hf * 8 + r;
          lds128(swz(kt, tok, 2 * cq), kw[hf][0], kw[hf][1], kw[hf][2], kw[hf][3]);
          lds128(swz(kt, tok, 2 * cq + 1), kw[hf][4], kw[hf][5], kw[hf][6], kw[hf][7]);
        }
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          const uint32_t x0 = kw[0][ks] ^ 0x80808080u, x1 = kw[1][ks] ^ 0x80808080u;
          // f16 value 1024 + (byte ^ 0x80) = int8 + 1152 (the bias is removed below)
          const uint32_t a[4] = {prmt(x0, 0x64646464u, 0x4140u), prmt(x1, 0x64646464u, 0x4140u),
                                 prmt(x0, 0x64646464u, 0x4342u), prmt(x1, 0x64646464u, 0x4342u)};
          mma16816<MmaT>(sacc[ks & 1], a, qa[ks][0], qa[ks][2]);
        }
      }
      // sv[0] = (key r, row 2cq), [1] = (key r, row 2cq+1), [2] = (key r+8, row 2cq), [3] = (key r+8, row 2cq+1)
      float sv[4];
      if constexpr (C::kI8) {
        // the +1152 bias of K removed per row, then each key's scale
        const ScaleT* ksp = reinterpret_cast<const ScaleT*>(smem + s * C::kStageBytes + 2 * C::kTileBytes);
        const float k0 = to_f32(ksp[r]), k1 = to_f32(ksp[r + 8]);
        sv[0] = ((sacc[0][0] + sacc[1][0]) - kbias0) * k0;
        sv[1] = ((sacc[0][1] + sacc[1][1]) - kbias1) * k0;
        sv[2] = ((sacc[0][2] + sacc[1][2]) - kbias0) * k1;
        sv[3] = ((sacc[0][3] + sacc[1][3]) - kbias1) * k1;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (kQc == 4)
            sv[e] = (sacc[0][e] + sacc[1][e]) + (sacc[2][e] + sacc[3][e]);
          else
            sv[e] = sacc[0][e] + sacc[1][e];
        }
      }
      const bool need_mask = tok0 + 16 > clean || (kExt && tok0 < lo_max && tok0 + 16 > x_sinks);
      if constexpr (kExt) {
        if (need_mask) hide_unseen(smem + s * C::kStageBytes, (int)tok0);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = sv[e] * p.scale_log2;
        if (need_mask) {
          const Tok tok = tok0 + r + 8 * (e >> 1);
          const Tok lim = (e & 1) ? limB : limA;
          if (tok >= ctx_end || tok > lim) v = -INFINITY;
          if constexpr (kExt) {
            if (tok >= x_sinks && tok < ((e & 1) ? loB : loA)) v = -INFINITY;
          }
        }
        sv[e] = v;
      }
      if constexpr (kExt) {
        if (score_row != nullptr) keep_scores(i, make_float2(sv[0], sv[1]), make_float2(sv[2], sv[3]));
      }
      // row max over the 16 keys: two in the thread, the rest across r (lanes xor 4, 8, 16)
      float mxA = fmaxf(sv[0], sv[2]), mxB = fmaxf(sv[1], sv[3]);
#pragma unroll
      for (int o2 = 4; o2 < 32; o2 <<= 1) {
        mxA = fmaxf(mxA, __shfl_xor_sync(0xffffffffu, mxA, o2));
        mxB = fmaxf(mxB, __shfl_xor_sync(0xffffffffu, mxB, o2));
      }
      const float mnA = fmaxf(mrA, mxA), mnB = fmaxf(mrB, mxB);
      const float muA = mnA == -INFINITY ? 0.f : mnA, muB = mnB == -INFINITY ? 0.f : mnB;
      const float alA = ex2_ftz(mrA - muA), alB = ex2_ftz(mrB - muB);
      const bool moved = mrA != mnA || mrB != mnB;
      mrA = mnA;
      mrB = mnB;
      sv[0] = ex2_ftz(sv[0] - muA);
      sv[1] = ex2_ftz(sv[1] - muB);
      sv[2] = ex2_ftz(sv[2] - muA);
      sv[3] = ex2_ftz(sv[3] - muB);
      lA = lA * alA + (sv[0] + sv[2]);
      lB = lB * alB + (sv[1] + sv[3]);
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          o[j][0] *= alA;
          o[j][1] *= alB;
          o[j][2] *= alA;
          o[j][3] *= alB;
        }
      }
      // P^T as the B operand (keys x rows): each 8 x 8 quadrant of P^T's accumulator
      // layout transposed in registers.  int8 pages: each key's value scale multiplies its
      // P entries here (keys r and r + 8 of this lane), so V enters the mma unscaled.
      if constexpr (C::kI8) {
        const ScaleT* vsp = reinterpret_cast<const ScaleT*>(smem + s * C::kStageBytes + 2 * C::kTileBytes + 128);
        const float v0 = to_f32(vsp[r]), v1 = to_f32(vsp[r + 8]);
        sv[0] *= v0;
        sv[1] *= v0;
        sv[2] *= v1;
        sv[3] *= v1;
      }
      uint32_t pb[2], pbl[2];
      pb[0] = movmatrix_t(pack2<MmaT>(sv[0], sv[1]));
      pb[1] = movmatrix_t(pack2<MmaT>(sv[2], sv[3]));
      if constexpr (C::kSplitP) {
        const uint32_t h0 = pack2<MmaT>(sv[0], sv[1]), h1 = pack2<MmaT>(sv[2], sv[3]);
        pbl[0] = movmatrix_t(pack_residual(sv[0], sv[1], h0));
        pbl[1] = movmatrix_t(pack_residual(sv[2], sv[3], h1));
      }
      // O^T += V^T P^T, one m16 tile of d per mma
      if constexpr (!C::kI8) {
        const int mi = lane >> 3;
        const int vtok = (mi & 1) * 8 + (lane & 7);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t v0, v1, v2, v3;
          ldsm_x4_t(swz(vt, vtok, 2 * j + (mi >> 1)), v0, v1, v2, v3);
          const uint32_t a[4] = {v0, v2, v1, v3};
          mma16816<MmaT>(o[j], a, pb[0], pb[1]);
          if constexpr (C::kSplitP) mma16816<MmaT>(o[j], a, pbl[0], pbl[1]);
        }
      } else {
        // V rows 2cq, 2cq+1, 2cq+8, 2cq+9, bytes [16 r, 16 r + 16): tile j row r <-> d 16r + 2j,
        // row r + 8 <-> d 16r + 2j + 1
        uint32_t vw[4][4];
#pragma unroll
        for (int t4 = 0; t4 < 4; ++t4) {
          const int tok = 2 * cq + (t4 & 1) + (t4 >> 1) * 8;
          lds128(swz(vt, tok, r), vw[t4][0], vw[t4][1], vw[t4][2], vw[t4][3]);
        }
        // V enters unscaled (exact int8 -> f16); the value scales were folded into P^T
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t y01 = prmt(vw[0][w], vw[1][w], 0x5140u) ^ 0x80808080u;
          const uint32_t y23 = prmt(vw[0][w], vw[1][w], 0x7362u) ^ 0x80808080u;
          const uint32_t z01 = prmt(vw[2][w], vw[3][w], 0x5140u) ^ 0x80808080u;
          const uint32_t z23 = prmt(vw[2][w], vw[3][w], 0x7362u) ^ 0x80808080u;
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {
            const uint32_t y = jj ? y23 : y01, z = jj ? z23 : z01;
            const uint32_t a[4] = {i8pair_to_f16x2(y, 0x4140u), i8pair_to_f16x2(y, 0x4342u),
                                   i8pair_to_f16x2(z, 0x4140u), i8pair_to_f16x2(z, 0x4342u)};
            mma16816<MmaT>(o[2 * w + jj], a, pb[0], pb[1]);
          }
        }
      }
      } else {
      const Tok tok0 = kExt ? (Tok)(tile_of(t0 + i) * 16) : (Tok)((t_begin + i) * 16);
      const uint32_t kt = smem_u32(smem + s * C::kStageBytes);
      const uint32_t vt = kt + C::kTileBytes;
      float sc[2][4];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;

      if constexpr (!C::kI8) {
        // two accumulator sets (even / odd k-steps) halve the dependent mma chain
        float sd[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) sd[nt][0] = sd[nt][1] = sd[nt][2] = sd[nt][3] = 0.f;
        const int mi = lane >> 3;
        const int ktok = (mi >> 1) * 8 + (lane & 7);
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
          uint32_t b0, b1, b2, b3;
          ldsm_x4(swz(kt, ktok, 2 * ks + (mi & 1)), b0, b1, b2, b3);
          if (ks & 1) {
            mma16816<MmaT>(sd[0], qa[ks], b0, b1);
            mma16816<MmaT>(sd[1], qa[ks], b2, b3);
          } else {
            mma16816<MmaT>(sc[0], qa[ks], b0, b1);
            mma16816<MmaT>(sc[1], qa[ks], b2, b3);
          }
        }
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[nt][e] += sd[nt][e];
      } else {
        uint32_t kw[2][8];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const int tok = nt * 8 + r;
          lds128(swz(kt, tok, 2 * cq), kw[nt][0], kw[nt][1], kw[nt][2], kw[nt][3]);
          lds128(swz(kt, tok, 2 * cq + 1), kw[nt][4], kw[nt][5], kw[nt][6], kw[nt][7]);
        }
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            const uint32_t x = kw[nt][ks] ^ 0x80808080u;
            mma16816<MmaT>(sc[nt], qa[ks], i8pair_to_f16x2(x, 0x4140u), i8pair_to_f16x2(x, 0x4342u));
          }
        }
        const ScaleT* ksp = reinterpret_cast<const ScaleT*>(smem + s * C::kStageBytes + 2 * C::kTileBytes);
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const float k0 = to_f32(ksp[nt * 8 + 2 * cq]), k1 = to_f32(ksp[nt * 8 + 2 * cq + 1]);
          sc[nt][0] *= k0;
          sc[nt][1] *= k1;
          sc[nt][2] *= k0;
          sc[nt][3] *= k1;
        }
      }

      // scale, mask, online softmax (base 2)
      const bool need_mask = tok0 + 16 > clean || (kExt && tok0 < lo_max && tok0 + 16 > x_sinks);
      if constexpr (kExt) {
        if (need_mask) hide_unseen(smem + s * C::kStageBytes, (int)tok0);
      }
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = sc[nt][e] * p.scale_log2;
          if (need_mask) {
            const Tok tok = tok0 + nt * 8 + 2 * cq + (e & 1);
            const Tok lim = e < 2 ? limA : limB;
            if (tok >= ctx_end || tok > lim) v = -INFINITY;
            if constexpr (kExt) {
              if (tok >= x_sinks && tok < (e < 2 ? loA : loB)) v = -INFINITY;
            }
          }
          sc[nt][e] = v;
        }
      }
      float mxA = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1]));
      float mxB = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
      mxA = fmaxf(mxA, __shfl_xor_sync(0xffffffffu, mxA, 1));
      mxA = fmaxf(mxA, __shfl_xor_sync(0xffffffffu, mxA, 2));
      mxB = fmaxf(mxB, __shfl_xor_sync(0xffffffffu, mxB, 1));
      mxB = fmaxf(mxB, __shfl_xor_sync(0xffffffffu, mxB, 2));
      const float mnA = fmaxf(mrA, mxA), mnB = fmaxf(mrB, mxB);
      const float muA = mnA == -INFINITY ? 0.f : mnA, muB = mnB == -INFINITY ? 0.f : mnB;
      // 2^x on the MUFU unit (ex2.approx.ftz: 2 ulp, -inf -> +0)
      const float alA = ex2_ftz(mrA - muA), alB = ex2_ftz(mrB - muB);
      const bool moved = mrA != mnA || mrB != mnB;  // a row max changed: O needs rescaling
      mrA = mnA;
      mrB = mnB;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        sc[nt][0] = ex2_ftz(sc[nt][0] - muA);
        sc[nt][1] = ex2_ftz(sc[nt][1] - muA);
        sc[nt][2] = ex2_ftz(sc[nt][2] - muB);
        sc[nt][3] = ex2_ftz(sc[nt][3] - muB);
      }
      lA = lA * alA + (sc[0][0] + sc[0][1] + sc[1][0] + sc[1][1]);
      lB = lB * alB + (sc[0][2] + sc[0][3] + sc[1][2] + sc[1][3]);
      // alpha is exactly 1 for rows whose max did not move (and for rows without a key
      // yet, whose O is 0): skipping the multiply then changes nothing
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int i2 = 0; i2 < NDT; ++i2) {
          o[i2][0] *= alA;
          o[i2][1] *= alA;
          o[i2][2] *= alB;
          o[i2][3] *= alB;
        }
      }
      uint32_t pa[4], pl[4];
      pa[0] = pack2<MmaT>(sc[0][0], sc[0][1]);
      pa[1] = pack2<MmaT>(sc[0][2], sc[0][3]);
      pa[2] = pack2<MmaT>(sc[1][0], sc[1][1]);
      pa[3] = pack2<MmaT>(sc[1][2], sc[1][3]);
      if constexpr (C::kSplitP) {
        // bf16 keeps 8 mantissa bits; the residual p - bf16(p) is a second bf16
        // operand so P reaches the tensor core with ~16 bits.
        pl[0] = pack_residual(sc[0][0], sc[0][1], pa[0]);
        pl[1] = pack_residual(sc[0][2], sc[0][3], pa[1]);
        pl[2] = pack_residual(sc[1][0], sc[1][1], pa[2]);
        pl[3] = pack_residual(sc[1][2], sc[1][3], pa[3]);
      }

      if constexpr (!C::kI8) {
        const int mi = lane >> 3;
        const int vtok = (mi & 1) * 8 + (lane & 7);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t b0, b1, b2, b3;
          ldsm_x4_t(swz(vt, vtok, 2 * j + (mi >> 1)), b0, b1, b2, b3);
          mma16816<MmaT>(o[2 * j], pa, b0, b1);
          mma16816<MmaT>(o[2 * j + 1], pa, b2, b3);
          if constexpr (C::kSplitP) {
            mma16816<MmaT>(o[2 * j], pl, b0, b1);
            mma16816<MmaT>(o[2 * j + 1], pl, b2, b3);
          }
        }
      } else {
        uint32_t vw[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int tok = 2 * cq + (t & 1) + (t >> 1) * 8;
          lds128(swz(vt, tok, r), vw[t][0], vw[t][1], vw[t][2], vw[t][3]);
        }
        const ScaleT* vsp = reinterpret_cast<const ScaleT*>(smem + s * C::kStageBytes + 2 * C::kTileBytes + 128);
        const __half2 vlo = __floats2half2_rn(to_f32(vsp[2 * cq]), to_f32(vsp[2 * cq + 1]));
        const __half2 vhi = __floats2half2_rn(to_f32(vsp[2 * cq + 8]), to_f32(vsp[2 * cq + 9]));
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t y01 = prmt(vw[0][w], vw[1][w], 0x5140u) ^ 0x80808080u;
          const uint32_t y23 = prmt(vw[0][w], vw[1][w], 0x7362u) ^ 0x80808080u;
          const uint32_t z01 = prmt(vw[2][w], vw[3][w], 0x5140u) ^ 0x80808080u;
          const uint32_t z23 = prmt(vw[2][w], vw[3][w], 0x7362u) ^ 0x80808080u;
          const uint32_t ys[4] = {y01, y01, y23, y23};
          const uint32_t zs[4] = {z01, z01, z23, z23};
#pragma unroll
          for (int i2 = 0; i2 < 4; ++i2) {
            const uint32_t sel = (i2 & 1) ? 0x4342u : 0x4140u;
            uint32_t lo = i8pair_to_f16x2(ys[i2], sel), hi = i8pair_to_f16x2(zs[i2], sel);
            __half2 lo2 = __hmul2(*reinterpret_cast<__half2*>(&lo), vlo);
            __half2 hi2 = __hmul2(*reinterpret_cast<__half2*>(&hi), vhi);
            mma16816<MmaT>(o[4 * w + i2], pa, *reinterpret_cast<uint32_t*>(&lo2), *reinterpret_cast<uint32_t*>(&hi2));
          }
        }
      }
          }
    }
    else if constexpr (kExt && C::kN8) {  // unmapped page: no row sees its keys
      if (score_row != nullptr)
        keep_scores(i, make_float2(-INFINITY, -INFINITY), make_float2(-INFINITY, -INFINITY));
    }
    __syncwarp();
    if constexpr (C::kSelfFeed) {
      // the stage's shared-memory reads are done: refill it with the warp's next tile
      if (lane == 0 && i + NS < n_my) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        issue_tile(i + NS);
        last_issued = i + NS;
      }
    } else {
      if (lane == 0) mbar_arrive(&empty[(i % NS)]);
    }
  }
  if constexpr (C::kSelfFeed) {
    // after a timed-out wait, loads this warp issued may still be landing in its stages
    if (timed_out && lane == 0) {
      for (int s = wk; s < NS && s <= last_issued; s += NWK) {
        const int last = s + ((last_issued - s) / NS) * NS;  // last tile issued into stage s
        if (!mbar_wait(&full[s], (last / NS) & 1)) record_error(p.err, kDevErrDrainWait);
      }
    }
  }
  // A consumer that timed out still joins the epilogue barriers below (so no other
  // warp waits forever); its rows carry garbage and the error word is set.
  (void)timed_out;

  if constexpr (C::kN8) {
    // row sums: partial over this thread's keys, reduced across r
#pragma unroll
    for (int o2 = 4; o2 < 32; o2 <<= 1) {
      lA += __shfl_xor_sync(0xffffffffu, lA, o2);
      lB += __shfl_xor_sync(0xffffffffu, lB, o2);
    }
  } else {
    lA += __shfl_xor_sync(0xffffffffu, lA, 1);
    lA += __shfl_xor_sync(0xffffffffu, lA, 2);
    lB += __shfl_xor_sync(0xffffffffu, lB, 1);
    lB += __shfl_xor_sync(0xffffffffu, lB, 2);
  }

  // ------------------------------------------------------------------ epilogue
  constexpr int NCT = C::kCons * 32;
  named_barrier(1, NCT);  // every consumer is done with the ring; reuse it
  float* eo = reinterpret_cast<float*>(smem);  // [NWK][RB][D]
  float* em = eo + NWK * C::kRB * D;            // [NWK][RB]
  float* el = em + NWK * C::kRB;                // [NWK][RB]
  if constexpr (C::kN8) {
    const int rlA = 2 * cq, rlB = rlA + 1;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = C::kI8 ? 16 * r + 2 * j + (e >> 1) : 16 * j + 8 * (e >> 1) + r;
        const int rl = (e & 1) ? rlB : rlA;
        eo[(wk * C::kRB + rl) * D + d] = o[j][e];
      }
    }
    if (r == 0) {
      em[wk * C::kRB + rlA] = mrA;
      el[wk * C::kRB + rlA] = lA;
      em[wk * C::kRB + rlB] = mrB;
      el[wk * C::kRB + rlB] = lB;
    }
  } else {
    const int rlA = wm * 16 + r, rlB = rlA + 8;
#pragma unroll
    for (int nd = 0; nd < NDT; ++nd) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = C::kI8 ? (32 * cq + 16 * (e & 1) + nd) : (nd * 8 + 2 * cq + (e & 1));
        const int rl = e < 2 ? rlA : rlB;
        eo[(wk * C::kRB + rl) * D + d] = o[nd][e];
      }
    }
    if (cq == 0) {
      em[wk * C::kRB + rlA] = mrA;
      el[wk * C::kRB + rlA] = lA;
      em[wk * C::kRB + rlB] = mrB;
      el[wk * C::kRB + rlB] = lB;
    }
  }
  named_barrier(1, NCT);
  const int tid = threadIdx.x;
  // row rl's log2-sum-exp from its maximum and sum
  auto put_lse = [&](int rl, float ms, float ls) {
    if (p.lse != nullptr) p.lse[q_row0 + row0 + rl] = ls > 0.f ? ms + log2f(ls) : INFINITY;
  };
  // kExt: four elements at a time (one element a thread and step made the epilogue of a 64-row
  // block 3800 of its instructions: a chunk of 927 int8 tokens under a 3-key window took 107 us,
  // with this and row blocks inside heads 34 us).
  auto put4 = [&](int rl, int d, float4 o4, float ls) {
    const float inv = ls > 0.f ? 1.f / ls : 0.f;
    const int64_t at = (q_row0 + row0 + rl) * D + d;
    o4 = make_float4(o4.x * inv, o4.y * inv, o4.z * inv, o4.w * inv);
    if (p.out_vec == 0) {
      store_dyn(p.out, at, p.out_dtype, o4.x);
      store_dyn(p.out, at + 1, p.out_dtype, o4.y);
      store_dyn(p.out, at + 2, p.out_dtype, o4.z);
      store_dyn(p.out, at + 3, p.out_dtype, o4.w);
    } else if (p.out_dtype == NVM_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = o4;
    } else if (p.out_dtype == NVM_BF16) {
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
          make_uint2(pack2<__nv_bfloat16>(o4.x, o4.y), pack2<__nv_bfloat16>(o4.z, o4.w));
    } else {
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
          make_uint2(pack2<__half>(o4.x, o4.y), pack2<__half>(o4.z, o4.w));
    }
  };
  // kExt: this CTA's row rl, elements d .. d + 3, over its warps along the keys
  auto combine4 = [&](int rl, int d, float& ms, float& ls) -> float4 {
    ms = -INFINITY;
#pragma unroll
    for (int w = 0; w < NWK; ++w) ms = fmaxf(ms, em[w * C::kRB + rl]);
    ls = 0.f;
    float4 o4 = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < NWK; ++w) {
      const float mw = em[w * C::kRB + rl];
      if (mw != -INFINITY) {
        const float f = exp2f(mw - ms);
        const float4 v = *reinterpret_cast<const float4*>(eo + (w * C::kRB + rl) * D + d);
        ls += el[w * C::kRB + rl] * f;
        o4.x += v.x * f;
        o4.y += v.y * f;
        o4.z += v.z * f;
        o4.w += v.w * f;
      }
    }
    return o4;
  };
  // The weights of virtual keys [v0, v1), by all consumer threads, after put_lse of every row:
  // new keys (the last L positions) start at zero, the others gain.
  auto add_mass = [&](int v0, int v1) {
    named_barrier(1, NCT);
    float lse[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) lse[i] = i < (int)rows_here ? __ldcg(p.lse + q_row0 + i) : INFINITY;
    float* mrow = p.mass + b * p.mass_sb + h * p.mass_sh;
    const float* z = p.scores + unit * p.n_chunks * p.ct * 16 * rows_pad;
    const int end = (int)(p.mass_len < x_end ? p.mass_len : x_end), first_new = (int)(ctx - p.L);
    constexpr int kU = 4;  // keys in flight per thread
    for (int v = v0 + tid; v < v1; v += kU * NCT) {
      float2 x[kU][4];
      float old[kU];
      int key[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int vu = v + u * NCT;
        key[u] = vu < v1 ? tile_of(vu >> 4) * 16 + (vu & 15) : end;
        if (key[u] >= end) continue;
        old[u] = key[u] < first_new ? mrow[key[u]] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (2 * i < rows_pad) x[u][i] = __ldcg(reinterpret_cast<const float2*>(z + (int64_t)vu * rows_pad) + i);
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (key[u] >= end) continue;
        float gain = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (2 * i < (int)rows_here) gain += ex2_ftz(x[u][i].x - lse[2 * i]);
          if (2 * i + 1 < (int)rows_here) gain += ex2_ftz(x[u][i].y - lse[2 * i + 1]);
        }
        mrow[key[u]] = old[u] + gain;
      }
    }
  };
  if constexpr (C::kClusterFits) {
    if (p.cluster) {
      // Split-K inside a thread-block cluster: the unit's chunks are CTAs 0 .. n_chunks-1
      // of one cluster (cluster rank == chunk index).  Each leaves its combined partial
      // rows (O, m, l) in its own shared memory; chunk 0 merges them over distributed
      // shared memory with the same operations, in the same chunk order, as the
      // workspace merge below.  Every CTA of the cluster, with or without keys, reaches
      // both cluster barriers; the second one keeps the partials alive until read.
      namespace cg = cooperative_groups;
      cg::cluster_group cluster = cg::this_cluster();
      float* cb_o = reinterpret_cast<float*>(smem + C::kClusterOff);  // [kRB][D]
      float2* cb_ml = reinterpret_cast<float2*>(cb_o + C::kRB * D);   // [kRB]
      float* cw = reinterpret_cast<float*>(cb_ml + C::kRB);           // [8][kRB] chunk weights
      float* cwl = cw + 8 * C::kRB;                                   // [kRB]
      if constexpr (kExt) {
        for (int g4 = tid; g4 < (int)rows_here * (D / 4); g4 += NCT) {
          const int rl = g4 / (D / 4), d = (g4 % (D / 4)) * 4;
          float ms, ls;
          *reinterpret_cast<float4*>(cb_o + rl * D + d) = combine4(rl, d, ms, ls);
          if (d == 0) cb_ml[rl] = make_float2(ms, ls);
        }
      }
      for (int64_t idx = tid; !kExt && idx < rows_here * D; idx += NCT) {
        const int rl = (int)(idx / D), d = (int)(idx % D);
        float ms = -INFINITY;
#pragma unroll
        for (int w = 0; w < NWK; ++w) ms = fmaxf(ms, em[w * C::kRB + rl]);
        float ls = 0.f, os = 0.f;
#pragma unroll
        for (int w = 0; w < NWK; ++w) {
          const float mw = em[w * C::kRB + rl];
          if (mw != -INFINITY) {
            const float f = exp2f(mw - ms);
            ls += el[w * C::kRB + rl] * f;
            os += eo[(w * C::kRB + rl) * D + d] * f;
          }
        }
        cb_o[rl * D + d] = os;
        if (d == 0) cb_ml[rl] = make_float2(ms, ls);
      }
      cluster.sync();
      if (c == 0) {
        const int nc = (int)n_chunks;  // chunks of this unit that hold keys (<= cluster size)
        for (int rl = tid; rl < rows_here; rl += NCT) {
          float ms = -INFINITY;
          for (int cc = 0; cc < nc; ++cc) ms = fmaxf(ms, cluster.map_shared_rank(cb_ml, cc)[rl].x);
          float ls = 0.f;
          for (int cc = 0; cc < nc; ++cc) {
            const float2 ml = cluster.map_shared_rank(cb_ml, cc)[rl];
            float f = -1.f;
            if (ml.x != -INFINITY) {
              f = exp2f(ml.x - ms);
              ls += ml.y * f;
            }
            cw[cc * C::kRB + rl] = f;
          }
          if constexpr (kExt) put_lse(rl, ms, ls);
          cwl[rl] = ls;
        }
        named_barrier(1, NCT);
        for (int64_t g4 = tid; g4 < rows_here * (D / 4); g4 += NCT) {
          const int rl = (int)(g4 / (D / 4)), d = (int)(g4 % (D / 4)) * 4;
          float o4[4] = {0.f, 0.f, 0.f, 0.f};
          for (int cc = 0; cc < nc; ++cc) {
            const float f = cw[cc * C::kRB + rl];
            if (f >= 0.f) {
              const float4 v = *reinterpret_cast<const float4*>(cluster.map_shared_rank(cb_o + rl * D + d, cc));
              o4[0] += v.x * f;
              o4[1] += v.y * f;
              o4[2] += v.z * f;
              o4[3] += v.w * f;
            }
          }
          const float ls = cwl[rl];
          if constexpr (kExt) put4(rl, d, make_float4(o4[0], o4[1], o4[2], o4[3]), ls);
#pragma unroll
          for (int e = 0; !kExt && e < 4; ++e)
            store_dyn(p.out, (q_row0 + row0 + rl) * D + d + e, p.out_dtype, ls > 0.f ? o4[e] / ls : 0.f);
        }
      }
      cluster.sync();
      if constexpr (kExt) {
        if (p.mass != nullptr) add_mass(t0 * 16, (t0 + n_my) * 16);  // each CTA its own chunk
      }
      return;
    }
  }
  const bool single = n_chunks == 1;
  const int64_t wsrow = (unit * p.n_chunks + c) * p.rows_real;
  if constexpr (kExt) {
    for (int g4 = tid; g4 < (int)rows_here * (D / 4); g4 += NCT) {
      const int rl = g4 / (D / 4), d = (g4 % (D / 4)) * 4;
      float ms, ls;
      const float4 o4 = combine4(rl, d, ms, ls);
      if (single) {
        put4(rl, d, o4, ls);
        if (d == 0) put_lse(rl, ms, ls);
      } else {
        *reinterpret_cast<float4*>(p.part_o + (wsrow + rl) * D + d) = o4;
        if (d == 0) p.part_ml[wsrow + rl] = make_float2(ms, ls);
      }
    }
  }
  for (int64_t idx = tid; !kExt && idx < rows_here * D; idx += NCT) {
    const int rl = (int)(idx / D), d = (int)(idx % D);
    float ms = -INFINITY;
#pragma unroll
    for (int w = 0; w < NWK; ++w) ms = fmaxf(ms, em[w * C::kRB + rl]);
    float ls = 0.f, os = 0.f;
#pragma unroll
    for (int w = 0; w < NWK; ++w) {
      const float mw = em[w * C::kRB + rl];
      if (mw != -INFINITY) {
        const float f = exp2f(mw - ms);
        ls += el[w * C::kRB + rl] * f;
        os += eo[(w * C::kRB + rl) * D + d] * f;
      }
    }
    if (single) {
      store_dyn(p.out, (q_row0 + row0 + rl) * D + d, p.out_dtype, ls > 0.f ? os / ls : 0.f);
    } else {
      p.part_o[(wsrow + rl) * D + d] = os;
      if (d == 0) p.part_ml[wsrow + rl] = make_float2(ms, ls);
    }
  }
  if (single) {
    if constexpr (kExt && C::kN8) {
      if (p.mass != nullptr) add_mass(0, x_tiles * 16);
    }
    return;
  }

  if constexpr (kExt && C::kN8) {
    if (p.defer) return;
  }
  // Split-K: the last CTA of this unit merges every chunk's partial result.
  __threadfence();
  named_barrier(1, NCT);
  if (tid == 0) {
    const int prev = atomicAdd(&p.counters[unit], 1);
    *s_flag = prev == (int)n_chunks - 1;
  }
  named_barrier(1, NCT);
  if (!*s_flag) return;
  __threadfence();
  const int64_t base = unit * p.n_chunks * p.rows_real;
  if ((2 * n_chunks + 1) * rows_here * (int64_t)sizeof(float) <= C::kMainBytes) {
    // Stage every chunk's (m, l) in shared memory with one parallel round of loads, turn
    // them into the log-sum-exp weights f = 2^(m_c - max m) (-1 marks a chunk without
    // keys), then sum the partial O rows with all chunk loads independent of one another.
    // Same operations in the same chunk order as the one-thread-per-element loop below.
    float* wm = reinterpret_cast<float*>(smem);  // [n_chunks][rows_here]: m, then the weight f
    float* wlc = wm + n_chunks * rows_here;      // [n_chunks][rows_here]: l
    float* wl = wlc + n_chunks * rows_here;      // [rows_here]: sum of l * f
    for (int64_t i = tid; i < n_chunks * rows_here; i += NCT) {
      const uint32_t cc32 = (uint32_t)i / (uint32_t)rows_here;
      const int64_t cc = cc32, rl = (int64_t)((uint32_t)i - cc32 * (uint32_t)rows_here);
      const float2 ml = __ldcg(&p.part_ml[base + cc * p.rows_real + rl]);
      wm[i] = ml.x;
      wlc[i] = ml.y;
    }
    named_barrier(1, NCT);
    for (int64_t rl = tid; rl < rows_here; rl += NCT) {
      float ms = -INFINITY;
      for (int64_t cc = 0; cc < n_chunks; ++cc) ms = fmaxf(ms, wm[cc * rows_here + rl]);
      float ls = 0.f;
      for (int64_t cc = 0; cc < n_chunks; ++cc) {
        const float mc = wm[cc * rows_here + rl];
        float f = -1.f;
        if (mc != -INFINITY) {
          f = exp2f(mc - ms);
          ls += wlc[cc * rows_here + rl] * f;
        }
        wm[cc * rows_here + rl] = f;
      }
      if constexpr (kExt) put_lse(rl, ms, ls);
      wl[rl] = ls;
    }
    named_barrier(1, NCT);
    // four consecutive d per thread (16-byte loads), eight chunks' loads in flight at once
    const int64_t cstride = p.rows_real * D;
    for (int64_t g4 = tid; g4 < rows_here * (D / 4); g4 += NCT) {
      const int rl = (int)(g4 / (D / 4)), d = (int)(g4 % (D / 4)) * 4;
      const float* po = p.part_o + (base + rl) * D + d;
      float os[4] = {0.f, 0.f, 0.f, 0.f};
      for (int64_t cc = 0; cc < n_chunks; cc += 8) {
        float4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[j] = cc + j < n_chunks ? __ldcg(reinterpret_cast<const float4*>(po + (cc + j) * cstride))
                                   : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (cc + j >= n_chunks) break;
          const float f = wm[(cc + j) * rows_here + rl];
          if (f >= 0.f) {
            os[0] += v[j].x * f;
            os[1] += v[j].y * f;
            os[2] += v[j].z * f;
            os[3] += v[j].w * f;
          }
        }
      }
      const float ls = wl[rl];
      if constexpr (kExt) put4(rl, d, make_float4(os[0], os[1], os[2], os[3]), ls);
#pragma unroll
      for (int e = 0; !kExt && e < 4; ++e)
        store_dyn(p.out, (q_row0 + row0 + rl) * D + d + e, p.out_dtype, ls > 0.f ? os[e] / ls : 0.f);
    }
    if (tid == 0) p.counters[unit] = 0;
    return;
  }
  for (int64_t idx = tid; idx < rows_here * D; idx += NCT) {
    const int rl = (int)(idx / D), d = (int)(idx % D);
    float ms = -INFINITY;
    for (int64_t cc = 0; cc < n_chunks; ++cc) ms = fmaxf(ms, __ldcg(&p.part_ml[base + cc * p.rows_real + rl].x));
    float ls = 0.f, os = 0.f;
    for (int64_t cc = 0; cc < n_chunks; ++cc) {
      const float2 ml = __ldcg(&p.part_ml[base + cc * p.rows_real + rl]);
      if (ml.x != -INFINITY) {
        const float f = exp2f(ml.x - ms);
        ls += ml.y * f;
        os += __ldcg(&p.part_o[(base + cc * p.rows_real + rl) * D + d]) * f;
      }
    }
    store_dyn(p.out, (q_row0 + row0 + rl) * D + d, p.out_dtype, ls > 0.f ? os / ls : 0.f);
    if constexpr (kExt) {
      if (d == 0) put_lse(rl, ms, ls);
    }
  }
  if (tid == 0) p.counters[unit] = 0;
}

int64_t env_int(const char* name, int64_t dflt) {
  const char* v = env_get(name);
  if (v == nullptr || v[0] == '\0') return dflt;
  return std::atoll(v);
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Opts one kernel instance into its dynamic shared memory, once per device.
template <typename KvT, typename ScaleT, int D, int NWM, int NWK, int NS_, bool kExt>
int ensure_smem_attr() {
  using C = Cfg<KvT, D, NWM, NWK, NS_>;
  static std::mutex mu;
  static uint64_t done_mask = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  if (dev < 64 && !(done_mask & (1ull << dev))) {
    int st = check_cuda(cudaFuncSetAttribute(paged_mma_kernel<KvT, ScaleT, D, NWM, NWK, NS_, kExt>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes),
                        "paged_attention: cudaFuncSetAttribute");
    if (st != NVM_OK) return st;
    done_mask |= 1ull << dev;
  }
  return NVM_OK;
}

template <typename KvT, typename ScaleT, int D, int NWM, int NWK, int NS_ = 0, bool kExt = false>
int launch_cfg(const PagedArgs& a, const MmaPlan& plan, void* ws, cudaStream_t s) {
  using C = Cfg<KvT, D, NWM, NWK, NS_>;
  auto kern = paged_mma_kernel<KvT, ScaleT, D, NWM, NWK, NS_, kExt>;
  {
    const int st = ensure_smem_attr<KvT, ScaleT, D, NWM, NWK, NS_, kExt>();
    if (st != NVM_OK) return st;
  }
  // Tensor maps: pools [P, Hkv, ps, D] -> dims (D, ps, Hkv, P); scales [P, Hkv, ps] -> (ps, Hkv, P).
  const CUtensorMapDataType dt = C::kI8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                        : (std::is_same<KvT, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                            : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
  const uint64_t e = sizeof(KvT);
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)a.page_size, (uint64_t)a.Hkv, (uint64_t)a.P};
  const uint64_t strides[3] = {D * e, (uint64_t)a.page_size * D * e, (uint64_t)(a.Hkv * a.page_size) * D * e};
  const uint32_t box[4] = {(uint32_t)C::kBoxElems, 16u, 1u, 1u};
  CUtensorMap tk, tv, tks, tvs;
  const uint64_t rdims[2] = {(uint64_t)D, (uint64_t)(a.P * a.Hkv * a.page_size)};  // kExt: the pool as rows
  int st = kExt ? encode_tmap(&tk, dt, 2, a.k_pages, rdims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)
                : encode_tmap(&tk, dt, 4, a.k_pages, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != NVM_OK) return st;
  st = kExt ? encode_tmap(&tv, dt, 2, a.v_pages, rdims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)
            : encode_tmap(&tv, dt, 4, a.v_pages, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != NVM_OK) return st;
  if (C::kI8 && !kExt) {
    const CUtensorMapDataType sdt =
        std::is_same<ScaleT, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const uint64_t sdims[3] = {(uint64_t)a.page_size, (uint64_t)a.Hkv, (uint64_t)a.P};
    const uint64_t sstr[2] = {(uint64_t)a.page_size * 2, (uint64_t)(a.Hkv * a.page_size) * 2};
    const uint32_t sbox[3] = {16u, 1u, 1u};
    st = encode_tmap(&tks, sdt, 3, a.k_scales, sdims, sstr, sbox, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (st != NVM_OK) return st;
    st = encode_tmap(&tvs, sdt, 3, a.v_scales, sdims, sstr, sbox, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (st != NVM_OK) return st;
  } else {
    tks = tk;
    tvs = tv;
  }
  MmaParams p{};
  p.q = a.q; p.out = a.out; p.block_table = a.block_table; p.context_lens = a.context_lens;
  if (plan.ws_bytes > 0) {
    char* w = static_cast<char*>(ws);
    p.counters = reinterpret_cast<int*>(w);
    w += kCounterBytes;
    p.part_ml = reinterpret_cast<float2*>(w);
    w += align256(plan.n_units * plan.n_chunks * plan.rows_real * sizeof(float2));
    p.part_o = reinterpret_cast<float*>(w);
  }
  p.err = device_error_word();
  p.q_dtype = a.q_dtype; p.out_dtype = a.out_dtype;
  p.B = a.B; p.Hq = a.Hq; p.Hkv = a.Hkv; p.L = a.L; p.P = a.P; p.ps = a.page_size; p.mp = a.max_pages;
  p.dense_ctx = a.dense_ctx;
  p.g = a.Hq / a.Hkv; p.M = p.g * a.L;
  p.n_rb = plan.n_row_blocks; p.rows_real = plan.rows_real; p.ct = plan.chunk_tiles; p.n_chunks = plan.n_chunks;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.causal = a.is_causal;
  p.cluster = 0;
  const uintptr_t out_align = a.out_dtype == NVM_F32 ? 15 : 7;
  p.out_vec = (reinterpret_cast<uintptr_t>(a.out) & out_align) == 0 ? 1 : 0;
  p.nb = plan.head_blocks;
  p.defer = a.defer;
  p.window = a.window; p.sinks = a.sinks; p.lse = a.lse; p.scores = a.scores;
  p.mass = a.mass; p.mass_sb = a.mass_sb; p.mass_sh = a.mass_sh; p.mass_len = a.mass_len;
  p.k_scales = a.k_scales; p.v_scales = a.v_scales;
  const dim3 grid((unsigned)plan.n_units, (unsigned)plan.n_chunks);
  if (plan.cluster && C::kClusterFits && plan.n_chunks > 1 && plan.n_chunks <= 8) {
    p.cluster = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = (unsigned)plan.n_chunks;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return check_cuda(cudaLaunchKernelEx(&cfg, kern, tk, tv, tks, tvs, p),
                      "paged_attention: tensor-core kernel launch (cluster)");
  }
  if (plan.cluster) return fail(NVM_ERR_UNSUPPORTED, "paged_attention: cluster plan for a kernel without it");
  kern<<<grid, C::kThreads, C::kSmemBytes, s>>>(tk, tv, tks, tvs, p);
  return check_cuda(cudaGetLastError(), "paged_attention: tensor-core kernel launch");
}

}  // namespace
}  // namespace nvm
